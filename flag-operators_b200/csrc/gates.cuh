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

// ---------------------------------------------------------------------------
// One or two fp32 values handled alike: float, or float2 with the packed instructions (two
// results per issue slot).
// ---------------------------------------------------------------------------
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ float mul_(float a, float b) { return a * b; }
__device__ __forceinline__ float add_(float a, float b) { return a + b; }
__device__ __forceinline__ float2 fma_(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)),
        "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul_(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add_(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
// A pair of T, as it is in memory, to and from fp32
template <typename T> __device__ __forceinline__ float2 unpack2(uint32_t w);
template <> __device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float2 f);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float2 f) {
  const __nv_bfloat162 h = __float22bfloat162_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float2 f) {
  const __half2 h = __float22half2_rn(f);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename F> __device__ __forceinline__ F all_(float x);
template <> __device__ __forceinline__ float all_<float>(float x) { return x; }
template <> __device__ __forceinline__ float2 all_<float2>(float x) { return make_float2(x, x); }
// f on every value
template <typename Fn> __device__ __forceinline__ float map_(Fn f, float a) { return f(a); }
template <typename Fn> __device__ __forceinline__ float2 map_(Fn f, float2 a) {
  return make_float2(f(a.x), f(a.y));
}
template <typename Fn> __device__ __forceinline__ float map_(Fn f, float a, float b) {
  return f(a, b);
}
template <typename Fn> __device__ __forceinline__ float2 map_(Fn f, float2 a, float2 b) {
  return make_float2(f(a.x, b.x), f(a.y, b.y));
}
template <typename Fn> __device__ __forceinline__ float map_(Fn f, float a, float b, float c) {
  return f(a, b, c);
}
template <typename Fn>
__device__ __forceinline__ float2 map_(Fn f, float2 a, float2 b, float2 c) {
  return make_float2(f(a.x, b.x, c.x), f(a.y, b.y, c.y));
}

// sigmoid(z) and 1 - sigmoid(z), neither with cancellation: e = e^-z, s = 1 / (1 + e), c = e s, which
// is 1 (fmin passes over the NaN of inf * 0) where e is infinite.  For e of 2^126 and more (z below
// -87.3) the reciprocal flushes s to 0, and c is 0 with it until e is infinite (z below -88.7): only
// for callers that take c times s, or times what has s as a factor, as all here do.
template <typename F> __device__ __forceinline__ void sigmoid_pair(F z, F& s, F& c) {
  const F e = map_(ex2, mul_(z, all_<F>(-kLog2e)));
  s = map_(rcp, add_(e, all_<F>(1.f)));
  c = map_([](float v) { return fminf(v, 1.f); }, mul_(e, s));
}

}  // namespace fo
