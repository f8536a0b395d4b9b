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
#include "f32x2.cuh"

namespace grappa {
namespace dev {

constexpr int kGroup8 = 32;

// Exponent byte of a group from its largest |x| (NaN if it holds one).
__device__ __forceinline__ uint32_t group8_byte(float top) {
  const uint32_t abs_bits = __float_as_uint(top);
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

// x 2^-E rounded to the nearest integer, ties to even, in the low byte.  |x 2^-E| <= 127 and
// the product is exact, so adding 1.5 * 2^23 in the same operation rounds at the unit and
// leaves the integer in the low mantissa bits.
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// eight codes of one chunk (a group's columns are four consecutive chunks); inv = 0, of a
// group that is not finite, makes codes 0 of its finite values, and the others are masked
__device__ __forceinline__ uint32_t codes4(const float* v, float inv) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    float a, b;
    unpack(fma2(f2(v[i], v[i + 1]), both(inv), both(12582912.f)), a, b);
    c[i] = __float_as_uint(a), c[i + 1] = __float_as_uint(b);
  }
  return inv == 0.f ? 0u : pack4(c[0], c[1], c[2], c[3]);
}
__device__ __forceinline__ uint2 codes8(const float* v, float inv) {
  return make_uint2(codes4(v, inv), codes4(v + 4, inv));
}
// max(|a|, |b|, |c|), NaN if one of them is
__device__ __forceinline__ float abs_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(fabsf(a)), "f"(fabsf(b)), "f"(fabsf(c)));
  return d;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ float abs_max8(const float* v) {
  return max_nan(abs_max3(abs_max3(v[0], v[1], v[2]), v[3], v[4]), abs_max3(v[5], v[6], v[7]));
}
// the four values of a word's codes: a code c + 128 in the low byte of 2^23 is the float
// 8388736 + c (a byte permutation instead of the quarter-rate integer conversion)
__device__ __forceinline__ void values4(uint32_t q, float scale, float* v) {
  q ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const F2 c = f2(__uint_as_float(__byte_perm(q, 0x4B000000u, 0x7540 + i)),
                    __uint_as_float(__byte_perm(q, 0x4B000000u, 0x7541 + i)));
    unpack(mul2(add2(c, both(-8388736.f)), both(scale)), v[i], v[i + 1]);
  }
}
// the eight values of a chunk's codes
__device__ __forceinline__ void values8(uint2 q, float scale, float* v) {
  values4(q.x, scale, v);
  values4(q.y, scale, v + 4);
}
// The same as four bf16 pairs, without passing through fp32: with x = c + 128 = 128 h + m (m of
// seven bits), c = (128 + m) - (256 - 128 h); both terms are bf16 patterns made by one logic
// operation a pair (0x4300 | m, and 0x4380 with the bit h cleared from its exponent), their
// difference and its product with the power of two are exact.
__device__ __forceinline__ uint32_t pair_bf16(uint32_t x, uint32_t sel, __nv_bfloat162 scale) {
  const uint32_t p = __byte_perm(x, 0u, sel);
  const uint32_t a = (p & 0x007F007Fu) | 0x43004300u, b = (p & 0x00800080u) ^ 0x43804380u;
  const __nv_bfloat162 d = __hmul2(__hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                           *reinterpret_cast<const __nv_bfloat162*>(&b)), scale);
  return *reinterpret_cast<const uint32_t*>(&d);
}
__device__ __forceinline__ uint4 values8_bf16(uint32_t qx, uint32_t qy, __nv_bfloat162 scale) {
  qx ^= 0x80808080u;
  qy ^= 0x80808080u;
  return make_uint4(pair_bf16(qx, 0x4140, scale), pair_bf16(qx, 0x4342, scale), pair_bf16(qy, 0x4140, scale),
                    pair_bf16(qy, 0x4342, scale));
}
// 2^E as a bf16 pair (the byte is the exponent field)
__device__ __forceinline__ __nv_bfloat162 group8_scale_bf16(uint32_t byte) {
  const uint32_t s = byte * 0x00800080u;
  return *reinterpret_cast<const __nv_bfloat162*>(&s);
}

// Eight consecutive columns into a bf16 or fp32 row (16-byte aligned).
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

// the first n columns of 16 bytes, zeros after them
template <typename T = __nv_bfloat16>
__device__ __forceinline__ uint4 first_columns(uint4 o, int n) {
  if constexpr (sizeof(T) == 4) return make_uint4(n > 0 ? o.x : 0u, n > 1 ? o.y : 0u, n > 2 ? o.z : 0u, n > 3 ? o.w : 0u);
  auto keep = [](uint32_t w, int k) { return k >= 2 ? w : (k == 1 ? w & 0xFFFFu : 0u); };
  return make_uint4(keep(o.x, n), keep(o.y, n - 2), keep(o.z, n - 4), keep(o.w, n - 6));
}

__device__ __forceinline__ int live_rows(const int32_t* n_ptr, int cap) {
  return n_ptr ? max(0, min(*n_ptr, cap)) : cap;
}

// out[c] (+)= sum over the parts of part[p][c], in a fixed order (column sums of the
// row kernels: every CTA writes its own part, so no atomics and the same bits each time)
void launch_sum_parts(const float* part, int parts, int64_t ld, int cols, float* out, bool accumulate,
                      cudaStream_t stream);

// Up to this many passes of a row kernel's CTA are left to one cluster (four rounds of it).
constexpr int kClusterPasses = 32;

// out[c] (+)= sum over the cluster's CTAs, in order, of cols[c] in their shared memory; the CTAs
// share the columns.  Called by all threads of all CTAs; cols was written by this CTA.
__device__ __forceinline__ void cluster_column_sums(const float* cols, int n, float* out, bool accumulate) {
  uint32_t ctas;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  __syncthreads();
  cluster_sync();
  const int first = static_cast<int>(cluster_rank() * blockDim.x + threadIdx.x);
  for (int c = first; c < n; c += static_cast<int>(ctas * blockDim.x)) {
    float s = 0.f;
    for (uint32_t r = 0; r < ctas; ++r) s += ld_cluster(cluster_addr(cols + c, r));
    out[c] = (accumulate ? out[c] : 0.f) + s;
  }
  cluster_sync();  // the others may still read this CTA's sums
}

}  // namespace dev
}  // namespace grappa
