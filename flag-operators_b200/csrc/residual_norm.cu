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
//
// Both are bound by memory.  Where rows are 16-byte aligned and fit, TPR threads own a row, VPT
// 16-byte vectors each, and CTAs walk over the rows: every input is read once, by cp.async into a
// ring of two rows in shared memory (the next row is on its way while this one is reduced and
// written), and a thread only ever reads the slots that it filled, so the ring needs no barrier.
// The backward keeps its threads' column sums in registers over all rows of the CTA, writes them
// as one partial row a CTA, and a column kernel adds those up in their order.  Other widths take
// the generic kernels: several passes over the row, through L1 and L2.
#include <type_traits>

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

// ---------------------------------------------------------------------------
// Rows in a shared-memory ring
// ---------------------------------------------------------------------------
template <int TPR> struct Shape {
  static constexpr int kThreads = TPR > 256 ? TPR : TPR > 32 ? TPR : 256;
  static constexpr int kRows = kThreads / TPR;  // rows side by side in a CTA
};

// Streams [S] of rows in two stages; slot(s, k, i): vector i of stream k in stage s, of this thread.
template <int S, int VPT, int THREADS> struct Ring {
  uint4 v[2][S][VPT][THREADS];
  __device__ __forceinline__ uint4& slot(int s, int k, int i) { return v[s][k][i][threadIdx.x]; }
  __device__ __forceinline__ void fetch(int s, int k, int i, const void* p) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                     (uint32_t)__cvta_generic_to_shared(&slot(s, k, i))),
                 "l"(p)
                 : "memory");
  }
};
__device__ __forceinline__ void ring_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void ring_wait_one() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// Sums of K values over the TPR threads of a row, in every one of them.  `red`: [K][warps], not
// used by the reduction before this one.
template <int TPR, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float (*red)[32]) {
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if (lane == 0)
#pragma unroll
      for (int k = 0; k < K; ++k) red[k][w] = v[k];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = red[k][lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// f *= the weights' vector v (f *= number where there is none)
template <typename W, int E>
__device__ __forceinline__ void times(float (&f)[E], const W* w, int v, float number) {
  if (w) {
    float t[E];
    constexpr int kPer = Vec16<W>::E;  // fp32 weights of 16-bit rows: two loads a vector
#pragma unroll
    for (int e = 0; e < E; e += kPer) unpack16<W>(ld_global_nc_v4(w + (int64_t)v * E + e), t + e);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] *= t[e];
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] *= number;
  }
}

template <typename T, typename W, int TPR, int VPT>
__global__ void __launch_bounds__(Shape<TPR>::kThreads, 1024 / Shape<TPR>::kThreads)
rrn_fwd_kernel(Fwd a) {
  using S = Shape<TPR>;
  constexpr int E = Vec16<T>::E;
  extern __shared__ __align__(16) uint8_t smem[];
  auto& ring = *reinterpret_cast<Ring<3, VPT, S::kThreads>*>(smem);
  __shared__ float red[4][32];
  const W *w = (const W*)a.w, *wp = (const W*)a.wp, *sv = (const W*)a.sv;
  const int nvec = (int)(a.N / E), v0 = threadIdx.x % TPR;
  const float n = (float)a.N;
  const int64_t step = (int64_t)gridDim.x * S::kRows, mine = threadIdx.x / TPR;
  auto fetch = [&](int64_t base, int s) {
    const int64_t row = base + mine;
    if (row < a.M) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = v0 + i * TPR;
        if (v < nvec) {
          ring.fetch(s, 0, i, (const T*)a.y + row * a.y_ld + v * E);
          ring.fetch(s, 1, i, (const T*)a.r + row * a.r_ld + v * E);
          if (a.gate) ring.fetch(s, 2, i, (const T*)a.gate + row * a.g_ld + v * E);
        }
      }
    }
    ring_commit();
  };
  int64_t base = (int64_t)blockIdx.x * S::kRows;
  fetch(base, 0);
  for (int it = 0; base < a.M; base += step, ++it) {
    const int s = it & 1;
    fetch(base + step, s ^ 1);
    ring_wait_one();
    const int64_t row = base + mine;
    const bool on = row < a.M;
    float inv1 = 1.f;
    if (wp) {
      float ss[1] = {0.f};
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (on && v0 + i * TPR < nvec) {
          float f[E];
          unpack16<T>(ring.slot(s, 0, i), f);
#pragma unroll
          for (int e = 0; e < E; ++e) ss[0] = fmaf(f[e], f[e], ss[0]);
        }
      row_sum<TPR>(ss, red + s);
      inv1 = 1.f / sqrtf(ss[0] / n + a.eps);
    }
    float r2[VPT][E], ss[1] = {0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * TPR;
      if (on && v < nvec) {
        float u[E];
        unpack16<T>(ring.slot(s, 0, i), u);
#pragma unroll
        for (int e = 0; e < E; ++e) u[e] *= inv1;
        if (wp) times<W>(u, wp, v, 1.f);
        if (a.gate) {
          float z[E];
          unpack16<T>(ring.slot(s, 2, i), z);
#pragma unroll
          for (int e = 0; e < E; ++e) u[e] *= act_of(a.act, z[e]);
        }
        times<W>(u, sv, v, a.s);
        float r[E];
        unpack16<T>(ring.slot(s, 1, i), r);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          r2[i][e] = r[e] + u[e];
          ss[0] = fmaf(r2[i][e], r2[i][e], ss[0]);
        }
      }
    }
    row_sum<TPR>(ss, red + 2 + s);
    const float inv2 = 1.f / sqrtf(ss[0] / n + a.eps);
    if (on && v0 == 0) {
      if (a.inv1) a.inv1[row] = inv1;
      if (a.inv2) a.inv2[row] = inv2;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * TPR;
      if (on && v < nvec) {
        st_global_stream_v4((T*)a.res + row * a.N + v * E, pack16<T>(r2[i]));
#pragma unroll
        for (int e = 0; e < E; ++e) r2[i][e] *= inv2;
        times<W>(r2[i], w, v, 1.f);
        st_global_stream_v4((T*)a.out + row * a.N + v * E, pack16<T>(r2[i]));
      }
    }
  }
}

template <typename T, typename W, int TPR, int VPT>
__global__ void __launch_bounds__(Shape<TPR>::kThreads, 512 / Shape<TPR>::kThreads)
rrn_bwd_kernel(Bwd a) {
  using S = Shape<TPR>;
  constexpr int E = Vec16<T>::E;
  extern __shared__ __align__(16) uint8_t smem[];
  auto& ring = *reinterpret_cast<Ring<5, VPT, S::kThreads>*>(smem);
  __shared__ float red[6][32];
  const W *w = (const W*)a.w, *wp = (const W*)a.wp, *sv = (const W*)a.sv;
  const int nvec = (int)(a.N / E), v0 = threadIdx.x % TPR;
  const int64_t step = (int64_t)gridDim.x * S::kRows, mine = threadIdx.x / TPR;
  auto fetch = [&](int64_t base, int s) {
    const int64_t row = base + mine;
    if (row < a.M) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int v = v0 + i * TPR;
        if (v < nvec) {
          ring.fetch(s, 0, i, (const T*)a.y + row * a.y_ld + v * E);
          ring.fetch(s, 1, i, (const T*)a.r + row * a.r_ld + v * E);
          if (a.gate) ring.fetch(s, 2, i, (const T*)a.gate + row * a.g_ld + v * E);
          if (a.dout) ring.fetch(s, 3, i, (const T*)a.dout + row * a.N + v * E);
          if (a.dres) ring.fetch(s, 4, i, (const T*)a.dres + row * a.N + v * E);
        }
      }
    }
    ring_commit();
  };
  // Of a vector: y, p / inv1 = y w_post, act and act', s, r', d, e, dr'
  struct Part {
    float y[E], q[E], av[E], da[E], sj[E], r2[E], d[E], e[E], dr[E];
  };
  auto load = [&](int s, int i, int v, float inv1, Part& p) {
    unpack16<T>(ring.slot(s, 0, i), p.y);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      p.q[e] = p.y[e];
      p.sj[e] = 1.f;
      p.av[e] = 1.f;
      p.da[e] = 0.f;
      p.d[e] = p.dr[e] = 0.f;
    }
    if (wp) times<W>(p.q, wp, v, 1.f);
    times<W>(p.sj, sv, v, a.s);
    if (a.gate) {
      float z[E];
      unpack16<T>(ring.slot(s, 2, i), z);
#pragma unroll
      for (int e = 0; e < E; ++e) act_grad(a.act, z[e], p.av[e], p.da[e]);
    }
    unpack16<T>(ring.slot(s, 1, i), p.r2);
#pragma unroll
    for (int e = 0; e < E; ++e) p.r2[e] = fmaf(p.sj[e] * p.av[e], inv1 * p.q[e], p.r2[e]);
    if (a.dout) unpack16<T>(ring.slot(s, 3, i), p.d);
#pragma unroll
    for (int e = 0; e < E; ++e) p.e[e] = p.d[e];
    times<W>(p.e, w, v, 1.f);
    if (a.dres) unpack16<T>(ring.slot(s, 4, i), p.dr);
  };
  float dw[VPT][E], ds[VPT][E], dwp[VPT][E];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) dw[i][e] = ds[i][e] = dwp[i][e] = 0.f;
  int64_t base = (int64_t)blockIdx.x * S::kRows;
  fetch(base, 0);
  for (int it = 0; base < a.M; base += step, ++it) {
    const int s = it & 1;
    fetch(base + step, s ^ 1);
    const int64_t row = base + mine;
    const bool on = row < a.M;
    const float inv1 = wp && on ? a.inv1[row] : 1.f, inv2 = on ? a.inv2[row] : 1.f;
    ring_wait_one();
    float sum[3] = {0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * TPR;
      if (on && v < nvec) {
        Part p;
        load(s, i, v, inv1, p);
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float qy = p.sj[e] * p.av[e] * p.q[e];
          sum[0] = fmaf(p.e[e], p.r2[e], sum[0]);
          sum[1] = fmaf(qy, fmaf(inv2, p.e[e], p.dr[e]), sum[1]);
          sum[2] = fmaf(qy, p.r2[e], sum[2]);
        }
      }
    }
    row_sum<TPR>(sum, red + 3 * s);
    const float c2 = inv2 * inv2 * inv2 * sum[0] / (float)a.N;
    const float c1 = wp ? inv1 * inv1 * inv1 * fmaf(-c2, sum[2], sum[1]) / (float)a.N : 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * TPR;
      if (on && v < nvec) {
        Part p;
        load(s, i, v, inv1, p);
        float dr[E], dy[E], dg[E], k[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const float D = fmaf(inv2, p.e[e], fmaf(-c2, p.r2[e], p.dr[e]));
          const float pe = p.q[e] * inv1, sD = p.sj[e] * D;
          dr[e] = D;
          dg[e] = sD * pe * p.da[e];
          k[e] = sD * p.av[e];
          dw[i][e] = fmaf(p.d[e] * p.r2[e], inv2, dw[i][e]);
          ds[i][e] = fmaf(D, p.av[e] * pe, ds[i][e]);
          dwp[i][e] = fmaf(k[e], p.y[e] * inv1, dwp[i][e]);
        }
        if (wp) times<W>(k, wp, v, 1.f);
#pragma unroll
        for (int e = 0; e < E; ++e) dy[e] = fmaf(inv1, k[e], -c1 * p.y[e]);
        st_global_stream_v4((T*)a.dr + row * a.N + v * E, pack16<T>(dr));
        st_global_stream_v4((T*)a.dy + row * a.N + v * E, pack16<T>(dy));
        if (a.gate) st_global_stream_v4((T*)a.dgate + row * a.N + v * E, pack16<T>(dg));
      }
    }
  }
  // part[3][gridDim.x][N]; rows side by side in the CTA are added up first
  const int64_t stride = (int64_t)gridDim.x * a.N;
  float* part = a.part + (int64_t)blockIdx.x * a.N;
  if constexpr (S::kRows == 1) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * TPR;
      if (v < nvec)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          part[v * E + e] = dw[i][e];
          part[stride + v * E + e] = ds[i][e];
          part[2 * stride + v * E + e] = dwp[i][e];
        }
    }
  } else {
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    float* sums = reinterpret_cast<float*>(smem);  // [rows][3][N], over the ring
    __syncthreads();
    const int N = (int)a.N;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = v0 + i * TPR;
      if (v < nvec)
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float* to = sums + mine * 3 * N + v * E + e;
          to[0] = dw[i][e];
          to[N] = ds[i][e];
          to[2 * N] = dwp[i][e];
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < 3 * N; j += S::kThreads) {
      float t = 0.f;
      for (int r = 0; r < S::kRows; ++r) t += sums[r * 3 * N + j];
      part[j / N * stride + j % N] = t;
    }
  }
}

// ---------------------------------------------------------------------------
// Any width and alignment
// ---------------------------------------------------------------------------
// A CTA per row, three passes over it (the later ones from L1 / L2).
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

// dw, ds, dw_post from the G partial rows.  A CTA owns 32 columns; warp q adds the rows q, q + 16,
// ..., then warp 0 the 16 warps' sums: an order that does not depend on scheduling.
constexpr int kReduceWarps = 16;
template <typename W>
__global__ void __launch_bounds__(32 * kReduceWarps) rrn_reduce_kernel(Bwd a, int G) {
  __shared__ float acc[kReduceWarps][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.x * 32 + lane;
  W* to = (W*)(blockIdx.y == 0 ? a.dw : blockIdx.y == 1 ? a.ds : a.dwp);
  if (!to) return;
  float t = 0.f;
  if (j < a.N) {
    const float* p = a.part + blockIdx.y * (int64_t)G * a.N + j;
#pragma unroll 4
    for (int k = q; k < G; k += kReduceWarps) t += p[(int64_t)k * a.N];
  }
  acc[q][lane] = t;
  __syncthreads();
  if (q == 0 && j < a.N) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < kReduceWarps; ++k) t += acc[k][lane];
    to[j] = from_f<W>(t);
  }
}

unsigned row_grid(int64_t M) {
  const int64_t g = (int64_t)num_sms() * 8;
  return (unsigned)(g < M ? g : M);
}

// Partial rows of the column sums, at most: the generic kernel's chunks, or the CTAs of the ring
// kernel (eight an SM for narrow rows, whose CTAs are small, one for wide ones).
int64_t partial_rows(int64_t M, int64_t N) {
  const int64_t per = N <= 1024 ? 8 : N <= 2048 ? 4 : N <= 4096 ? 2 : 1;
  int64_t g = per * num_sms();
  if (g < kChunks) g = kChunks;
  return g < M ? g : (M > 0 ? M : 1);
}

template <typename T, typename W> constexpr int kMostVectors = 1024;

// Calls f(TPR, VPT) with the smallest shape whose threads cover nvec vectors: a warp or less for
// the narrowest rows (no barrier), else a CTA of up to 512 threads with one or two vectors each.
template <typename F> int with_shape(int64_t nvec, F&& f) {
  auto go = [&](auto tpr, auto vpt) { return f(tpr, vpt); };
  using std::integral_constant;
  if (nvec <= 8) return go(integral_constant<int, 8>{}, integral_constant<int, 1>{});
  if (nvec <= 32) return go(integral_constant<int, 32>{}, integral_constant<int, 1>{});
  if (nvec <= 64) return go(integral_constant<int, 64>{}, integral_constant<int, 1>{});
  if (nvec <= 128) return go(integral_constant<int, 128>{}, integral_constant<int, 1>{});
  if (nvec <= 256) return go(integral_constant<int, 256>{}, integral_constant<int, 1>{});
  if (nvec <= 512) return go(integral_constant<int, 512>{}, integral_constant<int, 1>{});
  return go(integral_constant<int, 512>{}, integral_constant<int, 2>{});
}

template <typename T, typename W>
bool ring_ok(int64_t N, const void* const* rows, const int64_t* lds, int n,
             const void* const* vectors, int nv) {
  constexpr int E = Vec16<T>::E;
  bool ok = N % E == 0 && N / E <= kMostVectors<T, W>;
  for (int i = 0; i < n; ++i) ok = ok && aligned16(rows[i]) && lds[i] % E == 0;
  for (int i = 0; i < nv; ++i) ok = ok && aligned16(vectors[i]);
  return ok;
}

template <typename K, typename A>
int launch_ring(const char* what, K kernel, int64_t ctas, int threads, int smem, const A& a,
                cudaStream_t st) {
  if (smem > 40 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("%s: %s", what, cudaGetErrorString(e));
      return FO_ECUDA;
    }
  }
  kernel<<<(unsigned)ctas, threads, smem, st>>>(a);
  return check_launch(what);
}

// CTAs of an SM: by threads (with the registers that they are compiled for), and by shared memory.
int64_t resident(int threads_per_sm, int threads, int smem) {
  const int64_t a = threads_per_sm / threads, b = 227 * 1024 / (smem + 2048);
  return a < b ? a : b;
}

template <typename T, typename W>
int run_fwd(const Fwd& a, cudaStream_t st) {
  const void *rows[] = {a.y, a.r, a.gate, a.out, a.res}, *vs[] = {a.w, a.wp, a.sv};
  const int64_t lds[] = {a.y_ld, a.r_ld, a.g_ld, a.N, a.N};
  if (ring_ok<T, W>(a.N, rows, lds, 5, vs, 3))
    return with_shape(a.N / Vec16<T>::E, [&](auto tpr, auto vpt) {
      using S = Shape<tpr>;
      constexpr int smem = (int)sizeof(Ring<3, vpt, S::kThreads>);
      const int64_t most = num_sms() * resident(1024, S::kThreads, smem);
      const int64_t need = (a.M + S::kRows - 1) / S::kRows;
      return launch_ring("rrn_fwd_kernel", rrn_fwd_kernel<T, W, tpr, vpt>,
                         need < most ? need : most, S::kThreads, smem, a, st);
    });
  rrn_fwd_generic_kernel<T, W><<<row_grid(a.M), 256, 0, st>>>(a);
  return check_launch("rrn_fwd_generic_kernel");
}

template <typename T, typename W>
int run_bwd(const Bwd& a, cudaStream_t st) {
  const void *rows[] = {a.y, a.r, a.gate, a.dout, a.dres, a.dy, a.dr, a.dgate},
             *vs[] = {a.w, a.wp, a.sv};
  const int64_t lds[] = {a.y_ld, a.r_ld, a.g_ld, a.N, a.N, a.N, a.N, a.N};
  int G = 0;
  if (ring_ok<T, W>(a.N, rows, lds, 8, vs, 3)) {
    const int rc = with_shape(a.N / Vec16<T>::E, [&](auto tpr, auto vpt) {
      using S = Shape<tpr>;
      constexpr int ring = (int)sizeof(Ring<5, vpt, S::kThreads>);
      const int sums = S::kRows > 1 ? (int)(S::kRows * 3 * a.N * 4) : 0;
      const int smem = ring > sums ? ring : sums;
      int64_t ctas = num_sms() * resident(512, S::kThreads, smem);
      const int64_t need = (a.M + S::kRows - 1) / S::kRows, most = partial_rows(a.M, a.N);
      if (ctas > need) ctas = need;
      if (ctas > most) ctas = most;
      G = (int)ctas;
      return launch_ring("rrn_bwd_kernel", rrn_bwd_kernel<T, W, tpr, vpt>, ctas, S::kThreads, smem,
                         a, st);
    });
    if (rc) return rc;
  } else {
    rrn_bwd_generic_kernel<T, W><<<row_grid(a.M), 256, 0, st>>>(a);
    if (int rc = check_launch("rrn_bwd_generic_kernel")) return rc;
    G = (int)(a.M < kChunks ? a.M : kChunks);
    rrn_cols_kernel<T, W><<<dim3((unsigned)((a.N + 255) / 256), G), 256, 0, st>>>(a);
    if (int rc = check_launch("rrn_cols_kernel")) return rc;
  }
  rrn_reduce_kernel<W><<<dim3((unsigned)((a.N + 31) / 32), 3), 32 * kReduceWarps, 0, st>>>(a, G);
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
  *bytes = ((M + 3) / 4 * 4 + 3 * partial_rows(M, N) * N) * 4;  // c2 of each row, partial rows
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
              ws, ws + (M + 3) / 4 * 4, M, N, y_ld, r_ld, g_ld, scale, act};
  return with_types(dtype, w_dtype, [&](auto t, auto w) {
    return run_bwd<decltype(t), decltype(w)>(a, st);
  });
}
