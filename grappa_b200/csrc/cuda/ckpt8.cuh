// Rows in 8 bits: the device side of the form that kernels.h (Rows8) describes.
//
// A group of 32 columns holds codes c = round-half-even(x 2^-E), |c| <= 127, and the
// byte E + 127, with E the smallest integer >= -126 such that max|x| <= 127 * 2^E.  So
// |c 2^E - x| <= 2^E / 2 <= max|x| / 127 (max|x| > 63.5 * 2^E unless E = -126).  The
// scale is a power of two, not max|x| / 127, because then c 2^E needs 7 bits and a
// bfloat16 holds it exactly: a tensor-core product of the rows that the codes stand for
// has no rounding of its operand.  It costs up to one of the eight bits (half a bit on
// average).  A group that holds a NaN or an infinity gets the byte 255 and codes 0: all
// of it reads back as NaN.  The byte 0 (a cleared buffer) stands for zeros.
#pragma once
#include "common.cuh"

namespace grappa {
namespace dev {

constexpr int kGroup8 = 32;

// Exponent byte of a group from the largest |x| bit pattern in it (integer order of the
// patterns of non-negative floats is their order, with infinities and NaN above all).
__device__ __forceinline__ uint32_t group8_byte(uint32_t abs_bits) {
  if (abs_bits >= 0x7F800000u) return 255u;
  // |x| = m 2^k, 1 <= m < 2: 127 * 2^E >= |x| first at E = k - 6 while 64 m <= 127
  const uint32_t over = (abs_bits & 0x7FFFFFu) > 0x7E0000u ? 1u : 0u;
  const int e = static_cast<int>(abs_bits >> 23) - 6 + static_cast<int>(over);
  return static_cast<uint32_t>(max(e, 1));
}
// 2^-E for the byte (E + 127); 0 for the byte of a group that is not finite
__device__ __forceinline__ float group8_inv(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
// 2^E; infinity for the byte 255 (0 * infinity = NaN), 0 for the byte 0
__device__ __forceinline__ float group8_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// x 2^-E rounded to the nearest integer, ties to even, in the low byte.  |x 2^-E| <= 127,
// so adding 1.5 * 2^23 rounds at the unit and leaves the integer in the low mantissa bits.
__device__ __forceinline__ uint32_t code8(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)) & 0xFFu;
}
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// eight codes of one chunk (a group's columns are four consecutive chunks)
__device__ __forceinline__ uint2 codes8(const float* v, float inv) {
  if (inv == 0.f) return make_uint2(0u, 0u);
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = code8(v[i], inv);
  return make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
}
__device__ __forceinline__ uint32_t abs_max_bits8(const float* v) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
  return m;
}
// the eight values of a chunk's codes
__device__ __forceinline__ void values8(uint2 q, float scale, float* v) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = static_cast<float>(static_cast<int8_t>(q.x >> (8 * i))) * scale;
    v[4 + i] = static_cast<float>(static_cast<int8_t>(q.y >> (8 * i))) * scale;
  }
}

// Eight consecutive columns of a bf16 or fp32 row (16-byte aligned), as fp32 and back.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float* v) {
  if constexpr (sizeof(T) == 2) {
    bf16x8_to_f32(*reinterpret_cast<const uint4*>(p), v);
  } else {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
    v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  if constexpr (sizeof(T) == 2) {
    *reinterpret_cast<uint4*>(p) = f32_to_bf16x8(v);
  } else {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
  }
}
// the columns of chunk c at or past dim are zero
__device__ __forceinline__ void mask8(float* v, int c, int dim) {
  if (c * 8 + 8 <= dim) return;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c * 8 + i >= dim) v[i] = 0.f;
}

__device__ __forceinline__ int live_rows(const int32_t* n_ptr, int cap) {
  return n_ptr ? max(0, min(*n_ptr, cap)) : cap;
}

// out[c] (+)= sum over the parts of part[p][c], in a fixed order (column sums of the
// row kernels: every CTA writes its own part, so no atomics and the same bits each time)
void launch_sum_parts(const float* part, int parts, int64_t ld, int cols, float* out, bool accumulate,
                      cudaStream_t stream);

}  // namespace dev
}  // namespace grappa
