// Exponentials and sigmoids of the gated kernels.
#pragma once

#include "common.cuh"

namespace fo {

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// s = sigmoid(z) and c = 1 - sigmoid(z), neither with cancellation: from t = e^{-|z|} <= 1,
// 1 / (1 + t) and t / (1 + t).  Exact 0 and 1 at -inf and +inf; NaN stays NaN.
__device__ __forceinline__ void sigmoid2(float z, float& s, float& c) {
  const float t = ex2(-fabsf(z) * kLog2e), hi = rcp(1.f + t), lo = t * hi;
  s = z < 0.f ? lo : hi;
  c = z < 0.f ? hi : lo;
}

}  // namespace fo
