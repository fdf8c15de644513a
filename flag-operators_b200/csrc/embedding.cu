// Embedding lookup with a scale, and its gradient, for sm_100a.
//
//   out[t] = scale * W[ids[t]],   dW[v] = scale * sum of dout[t] over the t with ids[t] == v
//
// Sums are in fp32 and in a fixed order, so the gradient does not change from run to run.
#include "common.cuh"

namespace fo {
namespace {

template <typename T, typename I>
__global__ void __launch_bounds__(256)
emb_fwd_kernel(const I* __restrict__ ids, const T* __restrict__ w, T* __restrict__ out, int64_t T_,
               int64_t V, int64_t N, int64_t ld, float scale) {
  for (int64_t t = blockIdx.x; t < T_; t += gridDim.x) {
    const int64_t v = ids[t];
    const bool ok = v >= 0 && v < V;
    for (int64_t j = threadIdx.x; j < N; j += blockDim.x)
      out[t * N + j] = from_f<T>(ok ? scale * to_f<T>(w[v * ld + j]) : 0.f);
  }
}

// A CTA per row of W: every id is looked at, the matching rows of dout are added in order.
template <typename T, typename I>
__global__ void __launch_bounds__(256)
emb_bwd_kernel(const T* __restrict__ dout, const I* __restrict__ ids, T* __restrict__ dw,
               int64_t T_, int64_t V, int64_t N, int64_t padding_idx, float scale) {
  __shared__ int64_t hit[256];
  __shared__ int n_hit;
  __shared__ unsigned mask[8];
  for (int64_t v = blockIdx.x; v < V; v += gridDim.x) {
    for (int64_t j0 = 0; j0 < N; j0 += 1024) {
      float acc[4] = {0.f, 0.f, 0.f, 0.f};
      for (int64_t t0 = 0; t0 < T_; t0 += 256) {
        const int64_t t = t0 + threadIdx.x;
        const bool m = t < T_ && v != padding_idx && (int64_t)ids[t] == v;
        const unsigned bal = __ballot_sync(0xffffffffu, m);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) mask[threadIdx.x >> 5] = bal;
        __syncthreads();
        int at = __popc(bal & ((1u << (threadIdx.x & 31)) - 1)), all = 0;
        for (int k = 0; k < 8; ++k) {
          if (k < (int)(threadIdx.x >> 5)) at += __popc(mask[k]);
          all += __popc(mask[k]);
        }
        if (m) hit[at] = t;
        if (threadIdx.x == 0) n_hit = all;
        __syncthreads();
        for (int k = 0; k < n_hit; ++k)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int64_t j = j0 + threadIdx.x + 256 * i;
            if (j < N) acc[i] += to_f<T>(dout[hit[k] * N + j]);
          }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t j = j0 + threadIdx.x + 256 * i;
        if (j < N) dw[v * N + j] = from_f<T>(scale * acc[i]);
      }
    }
  }
}

template <typename F>
int with_types(int dtype, int index_dtype, F&& f) {
  FO_CHECK_ARG(index_dtype == FO_I64 || index_dtype == FO_I32,
               "embedding: ids must be int64 or int32");
  const bool l = index_dtype == FO_I64;
  switch (dtype) {
    case FO_F32: return l ? f(float{}, int64_t{}) : f(float{}, int32_t{});
    case FO_F16: return l ? f(__half{}, int64_t{}) : f(__half{}, int32_t{});
    case FO_BF16: return l ? f(__nv_bfloat16{}, int64_t{}) : f(__nv_bfloat16{}, int32_t{});
  }
  set_error("embedding: unsupported dtype code %d", dtype);
  return FO_EDTYPE;
}

int check_sizes(int64_t T, int64_t V, int64_t N) {
  FO_CHECK_ARG(T >= 0 && V >= 0 && N >= 0, "embedding: negative size T=%lld V=%lld N=%lld",
               (long long)T, (long long)V, (long long)N);
  FO_CHECK_ARG(T < (int64_t)1 << 31 && V < (int64_t)1 << 31 && N < (int64_t)1 << 31,
               "embedding: T=%lld, V=%lld and N=%lld must be below 2^31", (long long)T,
               (long long)V, (long long)N);
  return FO_OK;
}

unsigned row_grid(int64_t rows) {
  const int64_t g = (int64_t)num_sms() * 8;
  return (unsigned)(g < rows ? g : rows);
}

}  // namespace
}  // namespace fo

using namespace fo;

extern "C" int fo_embedding_fwd(const void* ids, const void* weight, void* out, int64_t T,
                                int64_t V, int64_t N, int64_t ld, float scale, int dtype,
                                int index_dtype, void* stream) {
  clear_error();
  if (int rc = check_sizes(T, V, N)) return rc;
  if (T == 0 || N == 0) return FO_OK;
  FO_CHECK_ARG(ids && out && (weight || V == 0), "embedding: null pointer");
  return with_types(dtype, index_dtype, [&](auto t, auto i) {
    using E = decltype(t);
    using I = decltype(i);
    emb_fwd_kernel<E, I><<<row_grid(T), 256, 0, as_stream(stream)>>>(
        (const I*)ids, (const E*)weight, (E*)out, T, V, N, ld, scale);
    return check_launch("emb_fwd_kernel");
  });
}

extern "C" int fo_embedding_bwd_workspace_bytes(int64_t T, int64_t V, int64_t N, int64_t* bytes) {
  clear_error();
  FO_CHECK_ARG(bytes, "embedding backward: null pointer");
  if (int rc = check_sizes(T, V, N)) return rc;
  *bytes = 0;
  return FO_OK;
}

extern "C" int fo_embedding_bwd(const void* dout, const void* ids, void* dw, int64_t T, int64_t V,
                                int64_t N, int64_t padding_idx, float scale, int dtype,
                                int index_dtype, void* workspace, int64_t ws_bytes, void* stream) {
  clear_error();
  if (int rc = check_sizes(T, V, N)) return rc;
  if (V == 0 || N == 0) return FO_OK;
  FO_CHECK_ARG(dw && (T == 0 || (dout && ids)), "embedding backward: null pointer");
  int64_t need = 0;
  fo_embedding_bwd_workspace_bytes(T, V, N, &need);
  if (need && (!workspace || ws_bytes < need)) {
    set_error("embedding backward: workspace of %lld bytes required", (long long)need);
    return FO_EWORKSPACE;
  }
  return with_types(dtype, index_dtype, [&](auto t, auto i) {
    using E = decltype(t);
    using I = decltype(i);
    emb_bwd_kernel<E, I><<<row_grid(V), 256, 0, as_stream(stream)>>>(
        (const E*)dout, (const I*)ids, (E*)dw, T, V, N, padding_idx, scale);
    return check_launch("emb_bwd_kernel");
  });
}
