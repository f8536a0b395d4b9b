// Activations of the linear layer and their slopes.
//
//   SiLU  z p,            p = 1 / (1 + exp(-z)),   slope p + z p (1 - p)
//   GELU  z p,            p = 1 / (1 + exp(-2u)),  u = sqrt(2/pi) (z + 0.044715 z^3),
//         slope p + z p (1 - p) 2 u'
// The GELU is its tanh form: (1 + tanh u) / 2 = 1 / (1 + exp(-2u)).  Written through p, the
// negative tail keeps its relative accuracy (1 + tanh u would cancel there).  One fast
// exponential and one fast division an element: about 1e-6 relative, far below the half
// step of bf16 (2^-9 of the value), so that their error does not show in bf16 outputs and
// stays at fp32 level in the fp32 column sums.
#pragma once
#include <cuda_runtime.h>

namespace grappa {
namespace dev {

constexpr float kGelu2C = 1.5957691216057308f;       // 2 sqrt(2 / pi)
constexpr float kGelu2C3 = 0.07135481627260025f;     // that times 0.044715

__device__ __forceinline__ float logistic(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }

__device__ __forceinline__ float silu(float z) { return z * logistic(z); }
__device__ __forceinline__ float gelu(float z) { return z * logistic(z * fmaf(kGelu2C3, z * z, kGelu2C)); }

// p (1 - p) is 0 for large |z|, where the other factor may be infinite
__device__ __forceinline__ float silu_slope(float z) {
  const float p = logistic(z), t = p * (1.f - p);
  return t == 0.f ? p : fmaf(z, t, p);
}
__device__ __forceinline__ float gelu_slope(float z) {
  const float z2 = z * z;
  const float p = logistic(z * fmaf(kGelu2C3, z2, kGelu2C)), t = p * (1.f - p);
  return t == 0.f ? p : fmaf(z * t, fmaf(3.f * kGelu2C3, z2, kGelu2C), p);
}

}  // namespace dev
}  // namespace grappa
