// Residual update and RMS norms around a block, fused, for sm_100a: forward and backward.
//
//   p = y * inv1 * w_post    inv1 = 1/sqrt(mean(y^2) + eps)      (p = y without w_post)
//   u = act(gate) * p        act: silu, sigmoid or none
//   r' = r + s * u           s: a vector [N], a number, or 1
//   out = r' * inv2 * w      inv2 = 1/sqrt(mean(r'^2) + eps)     (from r' before it is rounded)
//
// Backward from d = dL/dout and dr' = dL/dr', with e = d * w:
//   D  = dr' + inv2 e - r' inv2^3 mean(e r')        (all that reaches r')
//   dr = D,  ds = sum D u,  dw = sum d r' inv2
//   dgate = s D p act'(gate),  dp = s D act(gate)
//   dw_post = sum dp y inv1,  k = dp w_post,  dy = inv1 k - y inv1^3 mean(k y)
// r' is recomputed from y, gate, r and the forward's inv1, inv2 in fp32, so gradients do not see
// the rounding of the stored r'.  mean(k y) needs D, which needs mean(e r'); writing
//   sum k y = sum q y (dr' + inv2 e) - c2 sum q y r',  q = s act w_post, c2 = inv2^3 mean(e r')
// gets all three sums of a row from one pass and one block reduction.
#include "gates.cuh"

namespace fo {
namespace {

constexpr int kChunks = 64;  // row chunks of the column sums

struct Fwd {
  const void *y, *r, *w, *wp, *gate, *sv;
  void *out, *res;
  float *inv1, *inv2;
  int64_t M, N, y_ld, r_ld, g_ld;
  float s, eps;
  int act;
};

struct Bwd {
  const void *dout, *dres, *y, *r, *w, *wp, *gate, *sv;
  const float *inv1, *inv2;
  void *dy, *dr, *dgate, *dw, *dwp, *ds;
  float *c2, *part;
  int64_t M, N, y_ld, r_ld, g_ld;
  float s;
  int act;
};

__device__ __forceinline__ float act_of(int act, float z) {
  if (act == FO_ACT_NONE) return 1.f;
  float s, c;
  sigmoid2(z, s, c);
  return act == FO_ACT_SILU ? z * s : s;
}
// act(z) and its derivative
__device__ __forceinline__ void act_grad(int act, float z, float& a, float& da) {
  if (act == FO_ACT_NONE) {
    a = 1.f;
    da = 0.f;
    return;
  }
  float s, c;
  sigmoid2(z, s, c);
  a = act == FO_ACT_SILU ? z * s : s;
  da = act == FO_ACT_SILU ? s * fmaf(z, c, 1.f) : s * c;
}

// Any width and alignment: a CTA per row, three passes over it (the later ones from L1 / L2).
template <typename T, typename W>
__global__ void __launch_bounds__(256) rrn_fwd_generic_kernel(Fwd a) {
  __shared__ float red[32];
  const W *w = (const W*)a.w, *wp = (const W*)a.wp, *sv = (const W*)a.sv;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* y = (const T*)a.y + row * a.y_ld;
    const T* r = (const T*)a.r + row * a.r_ld;
    const T* z = a.gate ? (const T*)a.gate + row * a.g_ld : nullptr;
    float inv1 = 1.f;
    if (wp) {
      float ss = 0.f;
      for (int64_t j = threadIdx.x; j < a.N; j += blockDim.x) {
        const float f = to_f<T>(y[j]);
        ss = fmaf(f, f, ss);
      }
      inv1 = 1.f / sqrtf(block_sum(ss, red) / (float)a.N + a.eps);
    }
    auto updated = [&](int64_t j) {
      float u = to_f<T>(y[j]) * inv1;
      if (wp) u *= to_f<W>(wp[j]);
      if (z) u *= act_of(a.act, to_f<T>(z[j]));
      return fmaf(sv ? to_f<W>(sv[j]) : a.s, u, to_f<T>(r[j]));
    };
    float ss = 0.f;
    for (int64_t j = threadIdx.x; j < a.N; j += blockDim.x) {
      const float f = updated(j);
      ss = fmaf(f, f, ss);
    }
    const float inv2 = 1.f / sqrtf(block_sum(ss, red) / (float)a.N + a.eps);
    if (threadIdx.x == 0) {
      if (a.inv1) a.inv1[row] = inv1;
      if (a.inv2) a.inv2[row] = inv2;
    }
    for (int64_t j = threadIdx.x; j < a.N; j += blockDim.x) {
      const float f = updated(j);
      ((T*)a.res)[row * a.N + j] = from_f<T>(f);
      ((T*)a.out)[row * a.N + j] = from_f<T>(f * inv2 * to_f<W>(w[j]));
    }
  }
}

// dy, dr, dgate for any width and alignment; leaves c2 = inv2^3 mean(e r') of each row for the
// column sums.
template <typename T, typename W>
__global__ void __launch_bounds__(256) rrn_bwd_generic_kernel(Bwd a) {
  __shared__ float red[32];
  const W *w = (const W*)a.w, *wp = (const W*)a.wp, *sv = (const W*)a.sv;
  for (int64_t row = blockIdx.x; row < a.M; row += gridDim.x) {
    const T* y = (const T*)a.y + row * a.y_ld;
    const T* r = (const T*)a.r + row * a.r_ld;
    const T* z = a.gate ? (const T*)a.gate + row * a.g_ld : nullptr;
    const T* d = a.dout ? (const T*)a.dout + row * a.N : nullptr;
    const T* dres = a.dres ? (const T*)a.dres + row * a.N : nullptr;
    const float inv1 = wp ? a.inv1[row] : 1.f, inv2 = a.inv2[row];
    float s1 = 0.f, s2 = 0.f, s3 = 0.f;
    for (int64_t j = threadIdx.x; j < a.N; j += blockDim.x) {
      const float yv = to_f<T>(y[j]), wpv = wp ? to_f<W>(wp[j]) : 1.f;
      const float sj = sv ? to_f<W>(sv[j]) : a.s;
      const float qy = sj * (z ? act_of(a.act, to_f<T>(z[j])) : 1.f) * wpv * yv;
      const float r2 = fmaf(inv1, qy, to_f<T>(r[j]));
      const float e = d ? to_f<T>(d[j]) * to_f<W>(w[j]) : 0.f;
      s1 = fmaf(e, r2, s1);
      if (wp) {
        s2 = fmaf(qy, fmaf(inv2, e, dres ? to_f<T>(dres[j]) : 0.f), s2);
        s3 = fmaf(qy, r2, s3);
      }
    }
    s1 = block_sum(s1, red);
    const float c2 = inv2 * inv2 * inv2 * s1 / (float)a.N;
    float c1 = 0.f;
    if (wp) {
      s2 = block_sum(s2, red);
      s3 = block_sum(s3, red);
      c1 = inv1 * inv1 * inv1 * fmaf(-c2, s3, s2) / (float)a.N;
    }
    if (threadIdx.x == 0) a.c2[row] = c2;
    for (int64_t j = threadIdx.x; j < a.N; j += blockDim.x) {
      const float yv = to_f<T>(y[j]), wpv = wp ? to_f<W>(wp[j]) : 1.f;
      const float sj = sv ? to_f<W>(sv[j]) : a.s;
      float av = 1.f, da = 0.f;
      if (z) act_grad(a.act, to_f<T>(z[j]), av, da);
      const float p = yv * inv1 * wpv;
      const float r2 = fmaf(sj * av, p, to_f<T>(r[j]));
      const float e = d ? to_f<T>(d[j]) * to_f<W>(w[j]) : 0.f;
      const float D = fmaf(inv2, e, fmaf(-c2, r2, dres ? to_f<T>(dres[j]) : 0.f));
      ((T*)a.dr)[row * a.N + j] = from_f<T>(D);
      if (z) ((T*)a.dgate)[row * a.N + j] = from_f<T>(sj * D * p * da);
      ((T*)a.dy)[row * a.N + j] = from_f<T>(fmaf(inv1, sj * D * av * wpv, -c1 * yv));
    }
  }
}

// Partial sums of dw, ds, dw_post over a chunk of rows: a column per thread, part[3][chunks][N].
template <typename T, typename W>
__global__ void __launch_bounds__(256) rrn_cols_kernel(Bwd a) {
  const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= a.N) return;
  const W *wp = (const W*)a.wp, *sv = (const W*)a.sv;
  const int64_t rows = (a.M + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * rows, r1 = r0 + rows < a.M ? r0 + rows : a.M;
  const float wj = to_f<W>(((const W*)a.w)[j]), wpv = wp ? to_f<W>(wp[j]) : 1.f;
  const float sj = sv ? to_f<W>(sv[j]) : a.s;
  float dw = 0.f, ds = 0.f, dwp = 0.f;
  for (int64_t row = r0; row < r1; ++row) {
    const float inv1 = wp ? a.inv1[row] : 1.f, inv2 = a.inv2[row];
    const float n = to_f<T>(((const T*)a.y)[row * a.y_ld + j]) * inv1;
    const float av = a.gate ? act_of(a.act, to_f<T>(((const T*)a.gate)[row * a.g_ld + j])) : 1.f;
    const float r2 = fmaf(sj * av, n * wpv, to_f<T>(((const T*)a.r)[row * a.r_ld + j]));
    const float d = a.dout ? to_f<T>(((const T*)a.dout)[row * a.N + j]) : 0.f;
    const float D = fmaf(inv2, d * wj, fmaf(-a.c2[row], r2,
                         a.dres ? to_f<T>(((const T*)a.dres)[row * a.N + j]) : 0.f));
    dw = fmaf(d * r2, inv2, dw);
    ds = fmaf(D, av * n * wpv, ds);
    dwp = fmaf(sj * D * av, n, dwp);
  }
  float* part = a.part + (int64_t)blockIdx.y * a.N + j;
  const int64_t step = (int64_t)gridDim.y * a.N;
  part[0] = dw;
  part[step] = ds;
  part[2 * step] = dwp;
}

// dw, ds, dw_post from the partial rows, added in their order.
template <typename W>
__global__ void __launch_bounds__(128) rrn_reduce_kernel(Bwd a, int G) {
  const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  W* to = (W*)(blockIdx.y == 0 ? a.dw : blockIdx.y == 1 ? a.ds : a.dwp);
  if (j >= a.N || !to) return;
  const float* p = a.part + blockIdx.y * (int64_t)G * a.N + j;
  float t = 0.f;
  for (int k = 0; k < G; ++k) t += p[(int64_t)k * a.N];
  to[j] = from_f<W>(t);
}

unsigned row_grid(int64_t M) {
  const int64_t g = (int64_t)num_sms() * 8;
  return (unsigned)(g < M ? g : M);
}

int chunks_of(int64_t M) { return (int)(M < kChunks ? (M > 0 ? M : 1) : kChunks); }

template <typename T, typename W>
int run_fwd(const Fwd& a, cudaStream_t st) {
  rrn_fwd_generic_kernel<T, W><<<row_grid(a.M), 256, 0, st>>>(a);
  return check_launch("rrn_fwd_generic_kernel");
}

template <typename T, typename W>
int run_bwd(const Bwd& a, cudaStream_t st) {
  rrn_bwd_generic_kernel<T, W><<<row_grid(a.M), 256, 0, st>>>(a);
  if (int rc = check_launch("rrn_bwd_generic_kernel")) return rc;
  const int G = chunks_of(a.M);
  rrn_cols_kernel<T, W><<<dim3((unsigned)((a.N + 255) / 256), G), 256, 0, st>>>(a);
  if (int rc = check_launch("rrn_cols_kernel")) return rc;
  rrn_reduce_kernel<W><<<dim3((unsigned)((a.N + 127) / 128), 3), 128, 0, st>>>(a, G);
  return check_launch("rrn_reduce_kernel");
}

// Calls f with values of the row and weight element types: weights are of the rows' type or fp32.
template <typename F>
int with_types(int dtype, int w_dtype, F&& f) {
  if (w_dtype != dtype && w_dtype != FO_F32) {
    set_error("residual_rms_norm: weights of dtype code %d with rows of %d (the rows' or fp32 wanted)",
              w_dtype, dtype);
    return FO_EDTYPE;
  }
  switch (dtype) {
    case FO_F32: return f(float{}, float{});
    case FO_F16: return w_dtype == FO_F32 ? f(__half{}, float{}) : f(__half{}, __half{});
    case FO_BF16:
      return w_dtype == FO_F32 ? f(__nv_bfloat16{}, float{})
                               : f(__nv_bfloat16{}, __nv_bfloat16{});
  }
  set_error("residual_rms_norm: unsupported dtype code %d", dtype);
  return FO_EDTYPE;
}

int check_common(int64_t M, int64_t N, int act, const void* gate) {
  FO_CHECK_ARG(M >= 0 && N > 0, "residual_rms_norm: bad size M=%lld N=%lld", (long long)M,
               (long long)N);
  FO_CHECK_ARG(N <= (int64_t)1 << 31, "residual_rms_norm: N=%lld is over 2^31", (long long)N);
  FO_CHECK_ARG(act == FO_ACT_NONE || act == FO_ACT_SILU || act == FO_ACT_SIGMOID,
               "residual_rms_norm: bad activation code %d", act);
  FO_CHECK_ARG(!gate == (act == FO_ACT_NONE),
               "residual_rms_norm: a gate needs an activation, and an activation a gate");
  return FO_OK;
}

}  // namespace
}  // namespace fo

using namespace fo;

extern "C" int fo_residual_rms_norm_fwd(
    const void* y, const void* residual, const void* weight, const void* post_weight,
    const void* gate, const void* scale_vec, float scale, void* out, void* res_out, float* inv1,
    float* inv2, int64_t M, int64_t N, int64_t y_ld, int64_t r_ld, int64_t g_ld, float eps, int act,
    int dtype, int w_dtype, void* stream) {
  clear_error();
  if (int rc = check_common(M, N, act, gate)) return rc;
  if (M == 0) return FO_OK;
  FO_CHECK_ARG(y && residual && weight && out && res_out, "residual_rms_norm: null pointer");
  const Fwd a{y, residual, weight, post_weight, gate, scale_vec, out, res_out, inv1, inv2,
              M, N, y_ld, r_ld, g_ld, scale, eps, act};
  return with_types(dtype, w_dtype, [&](auto t, auto w) {
    return run_fwd<decltype(t), decltype(w)>(a, as_stream(stream));
  });
}

extern "C" int fo_residual_rms_norm_bwd_workspace_bytes(int64_t M, int64_t N, int64_t* bytes) {
  clear_error();
  FO_CHECK_ARG(bytes && M >= 0 && N > 0, "fo_residual_rms_norm_bwd_workspace_bytes: bad argument");
  *bytes = (M + (int64_t)3 * chunks_of(M) * N) * 4;
  return FO_OK;
}

extern "C" int fo_residual_rms_norm_bwd(
    const void* dout, const void* dres, const void* y, const void* residual, const void* weight,
    const void* post_weight, const void* gate, const void* scale_vec, float scale,
    const float* inv1, const float* inv2, void* dy, void* dr, void* dgate, void* dw, void* dwp,
    void* ds, int64_t M, int64_t N, int64_t y_ld, int64_t r_ld, int64_t g_ld, int act, int dtype,
    int w_dtype, void* workspace, int64_t ws_bytes, void* stream) {
  clear_error();
  if (int rc = check_common(M, N, act, gate)) return rc;
  cudaStream_t st = as_stream(stream);
  if (M == 0) {  // no rows: the weights' gradients are zero
    const size_t b = (size_t)N * dtype_size(w_dtype);
    for (void* p : {dw, dwp, ds})
      if (p) cudaMemsetAsync(p, 0, b, st);
    return check_launch("residual_rms_norm backward (empty)");
  }
  FO_CHECK_ARG(y && residual && weight && inv2 && dy && dr && dw && (!gate || dgate) &&
                   (!post_weight || (inv1 && dwp)) && (!scale_vec || ds),
               "residual_rms_norm backward: null pointer");
  int64_t need = 0;
  fo_residual_rms_norm_bwd_workspace_bytes(M, N, &need);
  if (!workspace || ws_bytes < need) {
    set_error("residual_rms_norm backward: workspace of %lld bytes required", (long long)need);
    return FO_EWORKSPACE;
  }
  FO_CHECK_ARG(aligned16(workspace), "residual_rms_norm backward: workspace must be 16-byte aligned");
  float* ws = (float*)workspace;
  const Bwd a{dout, dres, y, residual, weight, post_weight, gate, scale_vec, inv1, inv2, dy, dr,
              dgate, dw, post_weight ? dwp : nullptr, scale_vec ? ds : nullptr,
              ws, ws + M, M, N, y_ld, r_ld, g_ld, scale, act};
  return with_types(dtype, w_dtype, [&](auto t, auto w) {
    return run_bwd<decltype(t), decltype(w)>(a, st);
  });
}
