// Activations of the linear layer and their slopes.
//
//   SiLU  z p,            p = 1 / (1 + exp(-z)),   slope p + z p (1 - p)
//   GELU  z p,            p = 1 / (1 + exp(-2u)),  u = sqrt(2/pi) (z + 0.044715 z^3),
//         slope p + z p (1 - p) 2 u'
// The GELU is its tanh form: (1 + tanh u) / 2 = 1 / (1 + exp(-2u)).  Written through p, the
// negative tail keeps its relative accuracy (1 + tanh u would cancel there).  One fast
// exponential and one fast reciprocal an element: about 1e-6 relative, far below the half
// step of bf16 (2^-9 of the value), so that their error does not show in bf16 outputs and
// stays at fp32 level in the fp32 column sums.
#pragma once
#include "f32x2.cuh"

namespace grappa {
namespace dev {

// 2 sqrt(2/pi) and that times 0.044715; with log2(e) for the power of two of the exponential
constexpr float kGelu2C = 1.5957691216057308f;
constexpr float kGelu2C3 = 0.07135481627260025f;
constexpr float kLog2e = 1.4426950408889634f;

// 1 / (1 + 2^x) for a pair
__device__ __forceinline__ F2 logistic2(F2 x) {
  float a, b;
  unpack(x, a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  unpack(add2(f2(a, b), both(1.f)), a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return f2(a, b);
}

// v[0], v[1] become their activations.  One reciprocal serves the pair (1 / a = b / (a b):
// exponentials and reciprocals run at an eighth of the FMA rate and bound the epilogue of a
// layer), so a and b stay below 2^60: z is cut off below at the point where p is 2^-60 and
// z p is less than 1e-16 in magnitude.  The exponents take the cut-off for a NaN (fmaxf), or
// the pair's reciprocal would carry it into the other value; the factor z keeps it.
__device__ __forceinline__ float above(float z, float least) {  // a NaN stays
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(z), "f"(least));
  return r;
}
__device__ __forceinline__ F2 factor2(const float* v, float least) { return f2(above(v[0], least), above(v[1], least)); }
__device__ __forceinline__ F2 argument2(const float* v, float least) { return f2(fmaxf(v[0], least), fmaxf(v[1], least)); }
__device__ __forceinline__ void times_logistic2(F2 z, F2 x, float* v) {
  float a, b, r;
  unpack(x, a, b);
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(b));
  unpack(add2(f2(a, b), both(1.f)), a, b);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a * b));
  unpack(mul2(z, f2(b * r, a * r)), v[0], v[1]);
}
__device__ __forceinline__ void silu2(float* v) {
  constexpr float kLeast = -41.5f;
  times_logistic2(factor2(v, kLeast), mul2(argument2(v, kLeast), both(-kLog2e)), v);
}
__device__ __forceinline__ void gelu2(float* v) {
  constexpr float kLeast = -7.4f;
  const F2 z = argument2(v, kLeast);
  const F2 u = fma2(mul2(z, z), both(-kGelu2C3 * kLog2e), both(-kGelu2C * kLog2e));
  times_logistic2(factor2(v, kLeast), mul2(z, u), v);
}

// g[0], g[1] times the slopes at z[0], z[1].  p (1 - p) is 0 for large |z|, where the other
// factor may be infinite: the slope is p there.
__device__ __forceinline__ void scale_by_slope(F2 p, F2 rest, float* g) {
  const F2 t = mul2(p, fma2(p, both(-1.f), both(1.f)));
  const F2 s = fma2(rest, t, p);
  float t0, t1, p0, p1, s0, s1;
  unpack(t, t0, t1);
  unpack(p, p0, p1);
  unpack(s, s0, s1);
  unpack(mul2(f2(g[0], g[1]), f2(t0 == 0.f ? p0 : s0, t1 == 0.f ? p1 : s1)), g[0], g[1]);
}
__device__ __forceinline__ void silu_slope2(const float* v, float* g) {
  const F2 z = f2(v[0], v[1]);
  scale_by_slope(logistic2(mul2(z, both(-kLog2e))), z, g);
}
__device__ __forceinline__ void gelu_slope2(const float* v, float* g) {
  const F2 z = f2(v[0], v[1]), zz = mul2(z, z);
  const F2 u = fma2(zz, both(-kGelu2C3 * kLog2e), both(-kGelu2C * kLog2e));
  scale_by_slope(logistic2(mul2(z, u)), mul2(z, fma2(zz, both(3.f * kGelu2C3), both(kGelu2C))), g);
}

}  // namespace dev
}  // namespace grappa
