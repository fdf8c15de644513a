// Gated linear recurrence for sm_100a: forward, single-token step, backward.
//
//   h_t = a_t h_{t-1} + b_t, independently for every channel of [B, L, C]
//   gates as values (decay == NULL):  a_t = g_t,  b_t = beta_t x_t
//   gates as logits:  u_t = -scale softplus(decay) sigmoid(g_t),  a_t = e^{u_t},
//                     b_t = m_t i_t x_t,  m_t = sqrt(1 - a_t^2),  i_t = sigmoid(beta_t)
//   reset[b, t] != 0 takes a_t as 0 (so m_t as 1): the state starts again at step t.
//
// Backward, with D_t = dL/dh_t in total: D_t = dh_t + a_{t+1} D_{t+1} (D_{L-1} += dL/dh_T),
//   values:  dg = D h_{t-1},  dbeta = D x,  dx = D beta
//   logits:  du = D (a h_{t-1} - a^2 / m * i x),  dg = du u (1 - sigmoid(g)),
//            ddecay = -scale sigmoid(decay) sum du sigmoid(g),
//            dx = D m i,  dbeta = D m x i (1 - i)
//   and dg = du = 0 at a reset step; dh0 = a_0 D_0.
// The states h_{t-1} are recomputed in fp32 from the state the forward keeps in front of every
// FO_GLR_CHECKPOINT-th step: recomputing costs no traffic beyond x, g and beta, which the
// backward reads anyway, and gradients do not see the output's rounding to 16 bits.
//
// All of it is held in fp32; h and the gradients are rounded once when they are written.
#include "gates.cuh"

namespace fo {
namespace {

constexpr int kCkpt = FO_GLR_CHECKPOINT;

struct Strides {
  int64_t xb, xl, gb, gl, bb, bl;  // batch and step strides of x, g, beta, in elements
};

// 1 - e^{-w} for w >= 0.  Below 0.5 by its series to w^8 (next term / first term < 4e-9 there),
// since 1 - e^{-w} loses 1/w in relative precision; above, the subtraction loses at most 2.5x.
__device__ __forceinline__ float one_minus_exp(float w, float e) {
  float p = fmaf(w, -1.f / 40320.f, 1.f / 5040.f);
  p = fmaf(w, -p, 1.f / 720.f);
  p = fmaf(w, -p, 1.f / 120.f);
  p = fmaf(w, -p, 1.f / 24.f);
  p = fmaf(w, -p, 1.f / 6.f);
  p = fmaf(w, -p, 0.5f);
  p = fmaf(w, -p, 1.f);
  return w < 0.5f ? w * p : 1.f - e;
}

// Per-channel -scale * softplus(decay) (the log decay of a fully open gate).
__device__ __forceinline__ float log_decay(float decay, float scale) {
  return -scale * (decay > 20.f ? decay : log1pf(expf(decay)));
}

struct Gate {
  float a, b;        // h_t = a h_{t-1} + b
  float u, s, c;     // log a, sigmoid(g), 1 - sigmoid(g)
  float m, i, ci;    // sqrt(1 - a^2), sigmoid(beta), 1 - sigmoid(beta)
};

template <bool LOGITS>
__device__ __forceinline__ Gate gate_of(float x, float g, float beta, float rate, bool reset) {
  Gate q;
  if (!LOGITS) {
    q.a = reset ? 0.f : g;
    q.b = beta * x;
    return q;
  }
  sigmoid2(g, q.s, q.c);
  sigmoid2(beta, q.i, q.ci);
  q.u = rate * q.s;
  q.a = ex2(q.u * kLog2e);
  q.m = sqrtf(one_minus_exp(-2.f * q.u, q.a * q.a));
  if (reset) {
    q.a = 0.f;
    q.m = 1.f;
  }
  q.b = q.m * q.i * x;
  return q;
}

template <typename T, typename G, bool LOGITS>
__global__ void __launch_bounds__(128)
glr_fwd_kernel(const T* __restrict__ x, const G* __restrict__ g, const G* __restrict__ beta,
               const float* __restrict__ decay, const float* __restrict__ h0,
               const uint8_t* __restrict__ reset, T* __restrict__ h, float* __restrict__ hT,
               float* __restrict__ ckpt, int64_t L, int64_t C, Strides st, float scale) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
  if (c >= C) return;
  const float rate = LOGITS ? log_decay(decay[c], scale) : 0.f;
  const int64_t nck = (L + kCkpt - 1) / kCkpt;
  float s = h0 ? h0[b * C + c] : 0.f;
  for (int64_t t = 0; t < L; ++t) {
    if (ckpt && t % kCkpt == 0) ckpt[(b * nck + t / kCkpt) * C + c] = s;
    const Gate q = gate_of<LOGITS>(to_f<T>(x[b * st.xb + t * st.xl + c]),
                                   to_f<G>(g[b * st.gb + t * st.gl + c]),
                                   to_f<G>(beta[b * st.bb + t * st.bl + c]), rate,
                                   reset && reset[b * L + t]);
    s = q.a == 0.f ? q.b : fmaf(q.a, s, q.b);
    h[(b * L + t) * C + c] = from_f<T>(s);
  }
  if (hT) hT[b * C + c] = s;
}

template <typename T, typename G, bool LOGITS>
__global__ void __launch_bounds__(128)
glr_bwd_kernel(const T* __restrict__ x, const G* __restrict__ g, const G* __restrict__ beta,
               const float* __restrict__ decay, const uint8_t* __restrict__ reset,
               const float* __restrict__ ckpt, const T* __restrict__ dh,
               const float* __restrict__ dhT, T* __restrict__ dx, G* __restrict__ dg,
               G* __restrict__ dbeta, float* __restrict__ dh0, float* __restrict__ ddecay_part,
               int64_t L, int64_t C, Strides st, float scale) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x, b = blockIdx.y;
  if (c >= C) return;
  const float rate = LOGITS ? log_decay(decay[c], scale) : 0.f;
  const int64_t nck = (L + kCkpt - 1) / kCkpt;
  float d = dhT ? dhT[b * C + c] : 0.f, sum = 0.f;
  for (int64_t j = nck - 1; j >= 0; --j) {
    float before[kCkpt];
    float s = ckpt[(b * nck + j) * C + c];
    const int64_t t0 = j * kCkpt;
    const int n = (int)(L - t0 < kCkpt ? L - t0 : kCkpt);
    auto gate = [&](int64_t t) {
      return gate_of<LOGITS>(to_f<T>(x[b * st.xb + t * st.xl + c]),
                             to_f<G>(g[b * st.gb + t * st.gl + c]),
                             to_f<G>(beta[b * st.bb + t * st.bl + c]), rate,
                             reset && reset[b * L + t]);
    };
    for (int k = 0; k < n; ++k) {
      before[k] = s;
      const Gate q = gate(t0 + k);
      s = q.a == 0.f ? q.b : fmaf(q.a, s, q.b);
    }
    for (int k = n - 1; k >= 0; --k) {
      const int64_t t = t0 + k, o = (b * L + t) * C + c;
      const Gate q = gate(t);
      const bool rs = reset && reset[b * L + t];
      const float xv = to_f<T>(x[b * st.xb + t * st.xl + c]);
      d += to_f<T>(dh[o]);
      if (!LOGITS) {
        dx[o] = from_f<T>(d * to_f<G>(beta[b * st.bb + t * st.bl + c]));
        dg[o] = from_f<G>(rs ? 0.f : d * before[k]);
        dbeta[o] = from_f<G>(d * xv);
      } else {
        // a^2 / m -> the gradient's limit is 0 where a == 1 (m == 0)
        const float am = q.m > 0.f ? q.a / q.m : 0.f;
        const float du = rs ? 0.f : d * q.a * (before[k] - am * q.i * xv);
        sum = fmaf(du, q.s, sum);
        dg[o] = from_f<G>(du * q.u * q.c);
        const float dm = d * q.m;
        dx[o] = from_f<T>(dm * q.i);
        dbeta[o] = from_f<G>(dm * xv * q.i * q.ci);
      }
      d = q.a == 0.f ? 0.f : q.a * d;
    }
  }
  if (dh0) dh0[b * C + c] = d;
  if (ddecay_part) ddecay_part[b * C + c] = sum;
}

// ddecay[c] = -scale sigmoid(decay[c]) * the sum of the partial rows, in their order.
__global__ void __launch_bounds__(128)
glr_ddecay_kernel(const float* __restrict__ part, int64_t rows, const float* __restrict__ decay,
                  float* __restrict__ ddecay, int64_t C, float scale) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= C) return;
  float t = 0.f;
  for (int64_t r = 0; r < rows; ++r) t += part[r * C + c];
  float s, cs;
  sigmoid2(decay[c], s, cs);
  ddecay[c] = -scale * s * t;
}

template <typename T, typename G, bool LOGITS>
__global__ void __launch_bounds__(128)
glr_step_kernel(const T* __restrict__ x, const G* __restrict__ g, const G* __restrict__ beta,
                const float* __restrict__ decay, float* __restrict__ state, T* __restrict__ h,
                int64_t B, int64_t C, Strides st, float scale) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= C) return;
  const float rate = LOGITS ? log_decay(decay[c], scale) : 0.f;
  for (int64_t b = blockIdx.y; b < B; b += gridDim.y) {
    const Gate q = gate_of<LOGITS>(to_f<T>(x[b * st.xb + c]), to_f<G>(g[b * st.gb + c]),
                                   to_f<G>(beta[b * st.bb + c]), rate, false);
    const float s = q.a == 0.f ? q.b : fmaf(q.a, state[b * C + c], q.b);
    state[b * C + c] = s;
    h[b * C + c] = from_f<T>(s);
  }
}

// Calls f with values of the two element types of (dtype, gate_dtype): x's, and the gates',
// which are x's or fp32.
template <typename F>
int with_types(int dtype, int gate_dtype, F&& f) {
  if (gate_dtype != dtype && gate_dtype != FO_F32) {
    set_error("gated recurrence: gates of dtype code %d with x of %d (x's or fp32 wanted)",
              gate_dtype, dtype);
    return FO_EDTYPE;
  }
  switch (dtype) {
    case FO_F32: return f(float{}, float{});
    case FO_F16: return gate_dtype == FO_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
    case FO_BF16:
      return gate_dtype == FO_F32 ? f(__nv_bfloat16{}, float{})
                                  : f(__nv_bfloat16{}, __nv_bfloat16{});
  }
  set_error("gated recurrence: unsupported dtype code %d", dtype);
  return FO_EDTYPE;
}

int check_sizes(const char* what, int64_t B, int64_t L, int64_t C, int64_t most_b = 65535) {
  FO_CHECK_ARG(B >= 0 && L >= 0 && C >= 0, "%s: negative size B=%lld L=%lld C=%lld", what,
               (long long)B, (long long)L, (long long)C);
  FO_CHECK_ARG(B <= most_b, "%s: B=%lld is over 65535", what, (long long)B);
  FO_CHECK_ARG(C <= (int64_t)1 << 31, "%s: C=%lld is over 2^31", what, (long long)C);
  return FO_OK;
}

}  // namespace
}  // namespace fo

using namespace fo;

extern "C" int fo_glr_fwd(const void* x, const void* g, const void* beta, const float* decay,
                          const float* h0, const uint8_t* reset, void* h, float* hT, float* ckpt,
                          int64_t B, int64_t L, int64_t C, const int64_t* strides, float scale,
                          int dtype, int gate_dtype, void* stream) {
  clear_error();
  if (int rc = check_sizes("gated recurrence", B, L, C)) return rc;
  if (B == 0 || C == 0) return FO_OK;
  FO_CHECK_ARG(L == 0 || (x && g && beta && h && strides), "gated recurrence: null pointer");
  const Strides s = strides ? Strides{strides[0], strides[1], strides[2], strides[3], strides[4],
                                      strides[5]}
                            : Strides{};
  return with_types(dtype, gate_dtype, [&](auto t, auto gt) {
    using T = decltype(t);
    using G = decltype(gt);
    auto run = [&](auto k) {
      k<<<dim3((unsigned)((C + 127) / 128), (unsigned)B), 128, 0, as_stream(stream)>>>(
          (const T*)x, (const G*)g, (const G*)beta, decay, h0, reset, (T*)h, hT, ckpt, L, C, s,
          scale);
      return check_launch("glr_fwd_kernel");
    };
    return decay ? run(glr_fwd_kernel<T, G, true>) : run(glr_fwd_kernel<T, G, false>);
  });
}

extern "C" int fo_glr_step(const void* x, const void* g, const void* beta, const float* decay,
                           float* state, void* h, int64_t B, int64_t C, const int64_t* strides,
                           float scale, int dtype, int gate_dtype, void* stream) {
  clear_error();
  if (int rc = check_sizes("gated recurrence step", B, 1, C, INT64_MAX)) return rc;
  if (B == 0 || C == 0) return FO_OK;
  FO_CHECK_ARG(x && g && beta && state && h && strides, "gated recurrence step: null pointer");
  const Strides s{strides[0], 0, strides[1], 0, strides[2], 0};
  return with_types(dtype, gate_dtype, [&](auto t, auto gt) {
    using T = decltype(t);
    using G = decltype(gt);
    auto run = [&](auto k) {
      k<<<dim3((unsigned)((C + 127) / 128), (unsigned)(B < 65535 ? B : 65535)), 128, 0, as_stream(stream)>>>(
          (const T*)x, (const G*)g, (const G*)beta, decay, state, (T*)h, B, C, s, scale);
      return check_launch("glr_step_kernel");
    };
    return decay ? run(glr_step_kernel<T, G, true>) : run(glr_step_kernel<T, G, false>);
  });
}

extern "C" int fo_glr_bwd_workspace_bytes(int64_t B, int64_t L, int64_t C, int64_t* bytes) {
  clear_error();
  FO_CHECK_ARG(bytes, "gated recurrence backward: null pointer");
  if (int rc = check_sizes("gated recurrence backward", B, L, C)) return rc;
  *bytes = B * C * 4;
  return FO_OK;
}

extern "C" int fo_glr_bwd(const void* x, const void* g, const void* beta, const float* decay,
                          const uint8_t* reset, const float* ckpt, const void* dh,
                          const float* dhT, void* dx, void* dg, void* dbeta, float* dh0,
                          float* ddecay, int64_t B, int64_t L, int64_t C, const int64_t* strides,
                          float scale, int dtype, int gate_dtype, void* workspace,
                          int64_t ws_bytes, void* stream) {
  clear_error();
  if (int rc = check_sizes("gated recurrence backward", B, L, C)) return rc;
  FO_CHECK_ARG(!ddecay || decay, "gated recurrence backward: ddecay without decay");
  cudaStream_t q = as_stream(stream);
  if (C == 0) return FO_OK;
  if (B == 0) {
    if (ddecay) cudaMemsetAsync(ddecay, 0, (size_t)C * 4, q);
    return check_launch("gated recurrence backward (empty)");
  }
  FO_CHECK_ARG(L == 0 || (x && g && beta && ckpt && dh && dx && dg && dbeta && strides),
               "gated recurrence backward: null pointer");
  int64_t need = 0;
  if (ddecay) fo_glr_bwd_workspace_bytes(B, L, C, &need);
  if (need && (!workspace || ws_bytes < need)) {
    set_error("gated recurrence backward: workspace of %lld bytes required", (long long)need);
    return FO_EWORKSPACE;
  }
  const Strides s = strides ? Strides{strides[0], strides[1], strides[2], strides[3], strides[4],
                                      strides[5]}
                            : Strides{};
  float* part = ddecay ? (float*)workspace : nullptr;
  return with_types(dtype, gate_dtype, [&](auto t, auto gt) {
    using T = decltype(t);
    using G = decltype(gt);
    auto run = [&](auto k) {
      k<<<dim3((unsigned)((C + 127) / 128), (unsigned)B), 128, 0, q>>>(
          (const T*)x, (const G*)g, (const G*)beta, decay, reset, ckpt, (const T*)dh, dhT, (T*)dx,
          (G*)dg, (G*)dbeta, dh0, part, L, C, s, scale);
      return check_launch("glr_bwd_kernel");
    };
    int rc = decay ? run(glr_bwd_kernel<T, G, true>) : run(glr_bwd_kernel<T, G, false>);
    if (rc || !ddecay) return rc;
    glr_ddecay_kernel<<<(unsigned)((C + 127) / 128), 128, 0, q>>>(part, B, decay, ddecay, C,
                                                                  scale);
    return check_launch("glr_ddecay_kernel");
  });
}
