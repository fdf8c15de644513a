// Residual update and RMS norms around a block, fused, for sm_100a: forward and backward.
//
//   p = y * inv1 * w_post    inv1 = 1/sqrt(mean(y^2) + eps)      (p = y without w_post)
//   u = act(gate) * p        act: silu, sigmoid or none
//   r' = r + s * u           s: a vector [N], a number, or 1
//   out = r' * inv2 * w      inv2 = 1/sqrt(mean(r'^2) + eps)     (from r' before it is rounded)
//
// Backward from d = dL/dout and dr' = dL/dr', with e = d * w:
//   D  = dr' + inv2 e - r' inv2^3 mean(e r')        (all that reaches r')
//   dr = D,  dw = sum d r' inv2,  A = sum D act(gate) y inv1,  ds = w_post A,  dw_post = s A
//   dgate = s D p act'(gate),  k = s w_post D act(gate),  dy = inv1 k - y inv1^3 mean(k y)
// r' is recomputed from y, gate, r and the forward's inv1, inv2 in fp32, so gradients do not see
// the rounding of the stored r'.  mean(k y) needs D, which needs mean(e r'); writing
//   sum k y = sum q y (dr' + inv2 e) - c2 sum q y r',  q = s act w_post, c2 = inv2^3 mean(e r')
// gets all three sums of a row from one pass and one block reduction.
//
// Both are bound by memory.  TPR threads own a row, VPT 16-byte vectors each, and CTAs walk over the
// rows: every input is read once, by cp.async into a ring of two rows in shared memory (the next row
// is on its way while this one is reduced and written), and a thread only ever reads the slots that
// it filled, so the ring needs no barrier.  Rows that 16-byte vectors do not fit are read into
// registers instead; rows wider than 1024 vectors take 1024 threads, backward two CTAs of a cluster
// that add their sums up through distributed shared memory; still wider ones the generic kernels
// (several passes over the row, through L1 and L2).
// The backward keeps its threads' column sums (of dw and A) in registers over all rows of the CTA,
// writes them as one partial row a CTA, and a column kernel adds those up in their order; s w_post
// and w are kept in shared memory in fp32.
//
// Measured (B200): 16384 x 8192 bf16 with gate and both norms 237 us forward (5 streams, 1.34 GB,
// 5.7 TB/s) and 423 us backward (8 streams, 5.1 TB/s; 59 instructions an element at half the issue
// rate, one CTA of 512 threads on an SM) and 6 for the column sums; 4096 x 4096 fp32 without a gate 49,
// 63 and 5 us; 4096 x 16384 bf16 150 and 270 us.  1024 threads with one vector each were slower (297 us
// forward), and so was the backward with 64 registers (740 us: it spills).  The generic kernels are far
// from the memory's rate: 4096 x 12288 fp32 877 us forward, 799 + 191 backward (154 and 246 at a copy's
// rate), 4096 x 5001 bf16 241 us and 281 + 81 (31 and 50).

#include <type_traits>

#include "cluster.cuh"
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
// A row in the threads that own it
// ---------------------------------------------------------------------------
template <int TPR> struct Shape {
  static constexpr int kThreads = TPR > 32 ? TPR : 256;
  static constexpr int kRows = kThreads / TPR;  // rows side by side in a CTA
};

// What a thread has of a row: VPT vectors of E elements, TPR vectors apart, as fp32 pairs.
// WIDE: vectors of 16 bytes, rows of S streams on their way in a ring of two stages in shared
// memory.  Otherwise rows that 16-byte vectors do not fit: E = 2 elements TPR apart, read where
// they are needed first into registers.
template <typename T, typename W, int TPR, int VPT, bool WIDE, int S> struct Columns;

template <typename T, typename W, int TPR, int VPT, int S>
struct Columns<T, W, TPR, VPT, true, S> {
  static constexpr int E = Vec16<T>::E, P = E / 2, kThreads = Shape<TPR>::kThreads;
  static constexpr int kRingBytes = 2 * S * VPT * kThreads * 16;
  uint4* ring;
  int v0, nvec;
  // n: the elements of the row (or of the CTA's part of it)
  __device__ __forceinline__ Columns(uint8_t* smem, int64_t n)
      : ring(reinterpret_cast<uint4*>(smem) + threadIdx.x), v0(threadIdx.x % TPR), nvec((int)(n / E)) {}
  __device__ __forceinline__ uint4* slot(int stage, int k, int i) {
    return ring + ((stage * S + k) * VPT + i) * kThreads;
  }
  __device__ __forceinline__ bool on(int i) const { return v0 + i * TPR < nvec; }
  // Bytes from a row's begin to this thread's first element
  __device__ __forceinline__ int64_t first() const { return v0 * 16; }
  // p: a row's begin plus first()
  __device__ __forceinline__ void fetch(int stage, int k, const uint8_t* p) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(slot(stage, k, 0));
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (on(i))
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + i * kThreads * 16),
                     "l"(p + i * TPR * 16)
                     : "memory");
  }
  __device__ __forceinline__ void commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
  template <int LEFT> __device__ __forceinline__ void wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
  }
  // A vector as it is in memory, pair q of it, and one filled with a number (exact in any type)
  template <typename U> struct Words { uint4 u[E * (int)sizeof(U) / 16]; };
  using Raw = Words<T>;
  using RawW = Words<W>;
  template <typename U> static __device__ __forceinline__ float2 pair(const Words<U>& r, int q) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(r.u);
    if constexpr (sizeof(U) == 2) return unpack2<U>(w[q]);
    else return make_float2(__uint_as_float(w[2 * q]), __uint_as_float(w[2 * q + 1]));
  }
  template <typename U> static __device__ __forceinline__ void set(Words<U>& r, int q, float2 f) {
    uint32_t* w = reinterpret_cast<uint32_t*>(r.u);
    if constexpr (sizeof(U) == 2) {
      w[q] = pack2<U>(f);
    } else {
      w[2 * q] = __float_as_uint(f.x);
      w[2 * q + 1] = __float_as_uint(f.y);
    }
  }
  template <typename U> static __device__ __forceinline__ Words<U> filled(float v) {
    Words<U> r;
#pragma unroll
    for (int q = 0; q < P; ++q) set<U>(r, q, all_<float2>(v));
    return r;
  }
  __device__ __forceinline__ Raw get(int stage, int k, int i) { return {{*slot(stage, k, i)}}; }
  __device__ __forceinline__ RawW weights(const W* w, int i) const {
    RawW r;
#pragma unroll
    for (int k = 0; k < E * (int)sizeof(W) / 16; ++k)
      r.u[k] = ld_global_nc_v4(w + (v0 + i * TPR) * E + k * Vec16<W>::E);
    return r;
  }
  // Pair q of fp32 weights in shared memory
  __device__ __forceinline__ float2 weight(const float* smem, int i, int q) const {
    return *reinterpret_cast<const float2*>(smem + (v0 + i * TPR) * E + 2 * q);
  }
  __device__ __forceinline__ void put(uint8_t* p, int i, const Raw& r) const {
    st_global_stream_v4(p + i * TPR * 16, r.u[0]);
  }
  __device__ __forceinline__ void put_sums(float* row, int i, const float2 (&f)[P]) const {
#pragma unroll
    for (int q = 0; q < P; ++q) *reinterpret_cast<float2*>(row + (v0 + i * TPR) * E + 2 * q) = f[q];
  }
};

template <typename T, typename W, int TPR, int VPT, int S>
struct Columns<T, W, TPR, VPT, false, S> {
  static constexpr int E = 2, P = 1, kThreads = Shape<TPR>::kThreads, kRingBytes = 0;
  T raw[S][VPT][2];
  int c0, N;
  __device__ __forceinline__ Columns(uint8_t*, int64_t N_) : c0(threadIdx.x % TPR), N((int)N_) {}
  __device__ __forceinline__ int at(int i, int e) const { return c0 + (2 * i + e) * TPR; }
  __device__ __forceinline__ bool on(int i) const { return at(i, 0) < N; }
  __device__ __forceinline__ int64_t first() const { return c0 * (int)sizeof(T); }
  __device__ __forceinline__ void fetch(int, int k, const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e)
        raw[k][i][e] = at(i, e) < N ? reinterpret_cast<const T*>(p)[(2 * i + e) * TPR] : from_f<T>(0.f);
  }
  template <typename U> struct Words { U e[2]; };
  using Raw = Words<T>;
  using RawW = Words<W>;
  template <typename U> static __device__ __forceinline__ float2 pair(const Words<U>& r, int) {
    return make_float2(to_f<U>(r.e[0]), to_f<U>(r.e[1]));
  }
  template <typename U> static __device__ __forceinline__ void set(Words<U>& r, int, float2 f) {
    r.e[0] = from_f<U>(f.x);
    r.e[1] = from_f<U>(f.y);
  }
  template <typename U> static __device__ __forceinline__ Words<U> filled(float v) {
    return {{from_f<U>(v), from_f<U>(v)}};
  }
  __device__ __forceinline__ Raw get(int, int k, int i) { return {{raw[k][i][0], raw[k][i][1]}}; }
  __device__ __forceinline__ RawW weights(const W* w, int i) const {
    return {{w[at(i, 0)], at(i, 1) < N ? w[at(i, 1)] : from_f<W>(0.f)}};
  }
  __device__ __forceinline__ float2 weight(const float* smem, int i, int) const {
    return make_float2(smem[at(i, 0)], at(i, 1) < N ? smem[at(i, 1)] : 0.f);
  }
  __device__ __forceinline__ void put(uint8_t* p, int i, const Raw& r) const {
    reinterpret_cast<T*>(p)[2 * i * TPR] = r.e[0];
    if (at(i, 1) < N) reinterpret_cast<T*>(p)[(2 * i + 1) * TPR] = r.e[1];
  }
  __device__ __forceinline__ void put_sums(float* row, int i, const float2 (&f)[1]) const {
    row[at(i, 0)] = f[0].x;
    if (at(i, 1) < N) row[at(i, 1)] = f[0].y;
  }
};

// Sums of K values over the TPR threads of a row (of CTAS CTAs each), in every one of them.  `red`:
// [K][warps], not used by the reduction before this one.
template <int TPR, int CTAS = 1, int K>
__device__ __forceinline__ void row_sum(float (&v)[K], float (*red)[32]) {
  constexpr int kWarps = (TPR + 31) / 32 * CTAS;
  static_assert(kWarps <= 32, "a lane for each warp of the row");
#pragma unroll
  for (int o = (TPR < 32 ? TPR : 32) / 2; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if constexpr (kWarps > 1) {
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
    if constexpr (CTAS > 1) {
      const int at = (int)cluster_rank() * (TPR / 32) + w;
      if (lane < CTAS)
#pragma unroll
        for (int k = 0; k < K; ++k) store_remote(&red[k][at], lane, v[k]);
      __syncwarp();
      cluster_barrier();
    } else {
      if (lane == 0)
#pragma unroll
        for (int k = 0; k < K; ++k) red[k][w] = v[k];
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = red[k][lane % kWarps];
#pragma unroll
    for (int o = kWarps / 2; o > 0; o >>= 1)
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  }
}

// 1 / sqrt(x): the approximation (2 ulp) and one Newton step, which has to be left out where x is
// infinite.
__device__ __forceinline__ float inv_sqrt(float x) {
  const float r = rsqrtf(x);
  return x < INFINITY ? r * fmaf(-0.5f * x * r, r, 1.5f) : r;
}

// inv^3 x, for an x of about 1 / inv: inv^3 alone leaves the fp32 range for rows of norm 1e13 and 1e-13.
__device__ __forceinline__ float cubed(float inv, float x) { return inv * (inv * (inv * x)); }

// Bytes of two fp32 weight vectors of N elements, each a multiple of 16.
__host__ __device__ constexpr int weight_bytes(int64_t N) { return (int)((N + 3) / 4 * 4 * 8); }

template <typename T, typename W, int TPR, int VPT, bool WIDE>
__global__ void __launch_bounds__(Shape<TPR>::kThreads, 1024 / Shape<TPR>::kThreads)
rrn_fwd_kernel(Fwd a) {
  using S = Shape<TPR>;
  using C = Columns<T, W, TPR, VPT, WIDE, 3>;
  constexpr int P = C::P;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[4][32];
  const W *w = (const W*)a.w, *wp = (const W*)a.wp, *sv = (const W*)a.sv;
  C col(smem, a.N);
  const float rn = 1.f / (float)a.N;
  const int64_t step = (int64_t)gridDim.x * S::kRows, mine = threadIdx.x / TPR;
  int64_t base = (int64_t)blockIdx.x * S::kRows;
  // what is fetched next, and what is written: the thread's first bytes of its row
  const int64_t z = sizeof(T), r0 = base + mine;
  const uint8_t *py = (const uint8_t*)a.y + r0 * a.y_ld * z + col.first(),
                *pr = (const uint8_t*)a.r + r0 * a.r_ld * z + col.first(),
                *pg = (const uint8_t*)a.gate + r0 * a.g_ld * z + col.first();
  const int64_t dy = step * a.y_ld * z, dr = step * a.r_ld * z, dg = step * a.g_ld * z;
  int64_t to = r0 * a.N * z + col.first();
  auto fetch = [&](int64_t row, int stage) {
    if (row < a.M) {
      col.fetch(stage, 0, py);
      col.fetch(stage, 1, pr);
      if (a.gate) col.fetch(stage, 2, pg);
    }
    py += dy;
    pr += dr;
    pg += dg;
  };
  if constexpr (WIDE) {
    fetch(base + mine, 0);
    col.commit();
  }
  for (int it = 0; base < a.M; base += step, to += step * a.N * z, ++it) {
    const int s = it & 1;
    const int64_t row = base + mine;
    if constexpr (WIDE) {
      fetch(row + step, s ^ 1);
      col.commit();
      col.template wait<1>();
    } else {
      fetch(row, s);
    }
    const bool on = row < a.M;
    float inv1 = 1.f;
    if (wp) {
      float2 ss = all_<float2>(0.f);
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (on && col.on(i)) {
          const auto y = col.get(s, 0, i);
#pragma unroll
          for (int q = 0; q < P; ++q) ss = fma_(C::pair(y, q), C::pair(y, q), ss);
        }
      float sum[1] = {ss.x + ss.y};
      row_sum<TPR>(sum, red + s);
      inv1 = inv_sqrt(fmaf(sum[0], rn, a.eps));
    }
    float2 r2[VPT][P], ss = all_<float2>(0.f);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (on && col.on(i)) {
        const auto y = col.get(s, 0, i), r = col.get(s, 1, i);
        float2 u[P];
#pragma unroll
        for (int q = 0; q < P; ++q) u[q] = mul_(C::pair(y, q), all_<float2>(inv1));
        if (wp) {
          const auto t = col.weights(wp, i);
#pragma unroll
          for (int q = 0; q < P; ++q) u[q] = mul_(u[q], C::pair(t, q));
        }
        if (a.gate) {
          const auto z = col.get(s, 2, i);
#pragma unroll
          for (int q = 0; q < P; ++q) {
            const float2 e = map_(ex2, mul_(C::pair(z, q), all_<float2>(-kLog2e)));
            u[q] = mul_(u[q], map_(rcp, add_(e, all_<float2>(1.f))));
            if (a.act == FO_ACT_SILU) u[q] = mul_(u[q], C::pair(z, q));
          }
        }
        if (sv) {
          const auto t = col.weights(sv, i);
#pragma unroll
          for (int q = 0; q < P; ++q) r2[i][q] = fma_(u[q], C::pair(t, q), C::pair(r, q));
        } else {
#pragma unroll
          for (int q = 0; q < P; ++q) r2[i][q] = fma_(u[q], all_<float2>(a.s), C::pair(r, q));
        }
#pragma unroll
        for (int q = 0; q < P; ++q) ss = fma_(r2[i][q], r2[i][q], ss);
      }
    }
    float sum[1] = {ss.x + ss.y};
    row_sum<TPR>(sum, red + 2 + s);
    const float inv2 = inv_sqrt(fmaf(sum[0], rn, a.eps));
    if (on && threadIdx.x % TPR == 0) {
      if (a.inv1) a.inv1[row] = inv1;
      if (a.inv2) a.inv2[row] = inv2;
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (on && col.on(i)) {
        const auto t = col.weights(w, i);
        typename C::Raw res, out;
#pragma unroll
        for (int q = 0; q < P; ++q) {
          C::set(res, q, r2[i][q]);
          C::set(out, q, mul_(mul_(r2[i][q], all_<float2>(inv2)), C::pair(t, q)));
        }
        col.put((uint8_t*)a.res + to, i, res);
        col.put((uint8_t*)a.out + to, i, out);
      }
    }
  }
}

// CTAS > 1: a row is split over the CTAs of a cluster, a multiple of 16 bytes each.
template <typename T, typename W, int TPR, int VPT, bool WIDE, int CTAS>
__global__ void __launch_bounds__(Shape<TPR>::kThreads, 512 / Shape<TPR>::kThreads)
rrn_bwd_kernel(Bwd a) {
  using S = Shape<TPR>;
  using C = Columns<T, W, TPR, VPT, WIDE, 5>;
  using Raw = typename C::Raw;
  constexpr int P = C::P;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float red[6][32];
  // the CTA's columns: N from c0 on
  const int share = CTAS > 1 ? (int)((a.N / C::E + CTAS - 1) / CTAS) * C::E : (int)a.N;
  const int c0 = CTAS > 1 ? (int)cluster_rank() * share : 0;
  const int N = a.N - c0 < share ? (int)(a.N - c0) : share;
  // w and s w_post in fp32, in front of the ring
  float *sw = reinterpret_cast<float*>(smem), *ssw = sw + (N + 3) / 4 * 4;
  C col(smem + weight_bytes(N), N);
  for (int j = threadIdx.x; j < N; j += S::kThreads) {
    sw[j] = to_f<W>(((const W*)a.w)[c0 + j]);
    ssw[j] = (a.sv ? to_f<W>(((const W*)a.sv)[c0 + j]) : a.s) *
             (a.wp ? to_f<W>(((const W*)a.wp)[c0 + j]) : 1.f);
  }
  __syncthreads();
  if constexpr (CTAS > 1) cluster_barrier();  // every CTA runs before its memory is written to
  const int64_t groups = gridDim.x / CTAS, group = blockIdx.x / CTAS;
  const int64_t step = groups * S::kRows, mine = threadIdx.x / TPR;
  int64_t base = group * S::kRows;
  const int64_t z = sizeof(T), r0 = base + mine, first = c0 * z + col.first();
  const uint8_t *py = (const uint8_t*)a.y + r0 * a.y_ld * z + first,
                *pr = (const uint8_t*)a.r + r0 * a.r_ld * z + first,
                *pg = (const uint8_t*)a.gate + r0 * a.g_ld * z + first;
  const int64_t sy = step * a.y_ld * z, sr = step * a.r_ld * z, sg = step * a.g_ld * z,
                sn = step * a.N * z;
  int64_t to = r0 * a.N * z + first;
  // ahead: the row is `ahead` bytes behind the one at `to`
  auto fetch = [&](int64_t row, int stage, int64_t ahead) {
    if (row < a.M) {
      col.fetch(stage, 0, py);
      col.fetch(stage, 1, pr);
      if (a.gate) col.fetch(stage, 2, pg);
      if (a.dout) col.fetch(stage, 3, (const uint8_t*)a.dout + to + ahead);
      if (a.dres) col.fetch(stage, 4, (const uint8_t*)a.dres + to + ahead);
    }
    py += sy;
    pr += sr;
    pg += sg;
  };
  // What is absent is filled in, so that the arithmetic has no branches: a gate with 100 (its
  // sigmoid is 1), gradients with 0.
  const bool silu = a.act == FO_ACT_SILU;
  const float rn = 1.f / (float)a.N;
  struct Part {
    Raw y, r, z, d, dr;
  };
  auto load = [&](int s, int i, Part& p) {
    p.y = col.get(s, 0, i);
    p.r = col.get(s, 1, i);
    p.z = a.gate ? col.get(s, 2, i) : C::template filled<T>(100.f);
    p.d = a.dout ? col.get(s, 3, i) : C::template filled<T>(0.f);
    p.dr = a.dres ? col.get(s, 4, i) : C::template filled<T>(0.f);
  };
  float2 dw[VPT][P], A[VPT][P];
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int q = 0; q < P; ++q) dw[i][q] = A[i][q] = all_<float2>(0.f);
  float next1 = 1.f, next2 = 1.f;  // inv1 and inv2 of the row to come
  auto invs = [&](int64_t row) {
    if (row < a.M) {
      if (a.wp) next1 = a.inv1[row];
      next2 = a.inv2[row];
    }
  };
  invs(r0);
  if constexpr (WIDE) {
    fetch(r0, 0, 0);
    col.commit();
  }
  for (int it = 0; base < a.M; base += step, to += sn, ++it) {
    const int s = it & 1;
    const int64_t row = base + mine;
    if constexpr (WIDE) {
      fetch(row + step, s ^ 1, sn);
      col.commit();
    } else {
      fetch(row, s, 0);
    }
    const bool on = row < a.M;
    const float inv1 = next1, inv2 = next2;
    invs(row + step);
    const float2 i1 = all_<float2>(inv1), i2 = all_<float2>(inv2);
    if constexpr (WIDE) col.template wait<1>();
    float2 s1 = all_<float2>(0.f), s2 = s1, s3 = s1;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (on && col.on(i)) {
        Part p;
        load(s, i, p);
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const float2 z = C::pair(p.z, q);
          const float2 ez = map_(ex2, mul_(z, all_<float2>(-kLog2e)));
          float2 av = map_(rcp, add_(ez, all_<float2>(1.f)));
          if (silu) av = mul_(av, z);
          const float2 qy = mul_(mul_(col.weight(ssw, i, q), av), C::pair(p.y, q));
          const float2 r2 = fma_(i1, qy, C::pair(p.r, q));
          const float2 e = mul_(C::pair(p.d, q), col.weight(sw, i, q));
          s1 = fma_(e, r2, s1);
          s2 = fma_(qy, fma_(i2, e, C::pair(p.dr, q)), s2);
          s3 = fma_(qy, r2, s3);
        }
      }
    }
    float sum[3] = {s1.x + s1.y, s2.x + s2.y, s3.x + s3.y};
    row_sum<TPR, CTAS>(sum, red + 3 * s);
    const float c2 = cubed(inv2, sum[0] * rn);
    const float c1 = a.wp ? cubed(inv1, fmaf(-c2, sum[2], sum[1]) * rn) : 0.f;
    const float2 m2 = all_<float2>(-c2), m1 = all_<float2>(-c1);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      if (on && col.on(i)) {
        Part p;
        load(s, i, p);
        Raw dr, dy, dg;
#pragma unroll
        for (int q = 0; q < P; ++q) {
          const float2 z = C::pair(p.z, q), y = C::pair(p.y, q), n = mul_(y, i1);
          float2 sg, c;
          sigmoid_pair(z, sg, c);
          const float2 wq = col.weight(ssw, i, q);
          const float2 av = silu ? mul_(sg, z) : sg, sa = mul_(wq, av);
          const float2 r2 = fma_(sa, n, C::pair(p.r, q));
          const float2 d = C::pair(p.d, q), e = mul_(d, col.weight(sw, i, q));
          const float2 D = fma_(i2, e, fma_(m2, r2, C::pair(p.dr, q)));
          // silu' = s (1 + z c), sigmoid' = s c
          const float2 f = silu ? fma_(z, c, all_<float2>(1.f)) : c;
          C::set(dr, q, D);
          C::set(dg, q, mul_(mul_(mul_(wq, D), n), mul_(sg, f)));
          C::set(dy, q, fma_(i1, mul_(D, sa), mul_(m1, y)));
          dw[i][q] = fma_(mul_(d, i2), r2, dw[i][q]);
          A[i][q] = fma_(D, mul_(av, n), A[i][q]);
        }
        col.put((uint8_t*)a.dr + to, i, dr);
        col.put((uint8_t*)a.dy + to, i, dy);
        if (a.gate) col.put((uint8_t*)a.dgate + to, i, dg);
      }
    }
  }
  // part[2][groups][N]; rows side by side in the CTA are added up first
  const int64_t stride = groups * a.N;
  float* part = a.part + group * a.N + c0;
  if constexpr (S::kRows == 1) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (col.on(i)) {
        col.put_sums(part, i, dw[i]);
        col.put_sums(part + stride, i, A[i]);
      }
  } else {
    if constexpr (WIDE) col.template wait<0>();
    float* sums = reinterpret_cast<float*>(smem);  // [rows][2][N], over everything
    __syncthreads();
#pragma unroll
    for (int i = 0; i < VPT; ++i)
      if (col.on(i)) {
        col.put_sums(sums + mine * 2 * N, i, dw[i]);
        col.put_sums(sums + mine * 2 * N + N, i, A[i]);
      }
    __syncthreads();
    for (int j = threadIdx.x; j < 2 * N; j += S::kThreads) {
      float t = 0.f;
      for (int r = 0; r < S::kRows; ++r) t += sums[r * 2 * N + j];
      part[j / N * stride + j % N] = t;
    }
  }
  if constexpr (CTAS > 1) cluster_barrier();  // none leaves while another writes to it
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
    const float c2 = cubed(inv2, s1 / (float)a.N);
    float c1 = 0.f;
    if (wp) {
      s2 = block_sum(s2, red);
      s3 = block_sum(s3, red);
      c1 = cubed(inv1, fmaf(-c2, s3, s2) / (float)a.N);
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

// Partial sums of dw and A over a chunk of rows: a column per thread, part[2][chunks][N].
template <typename T, typename W>
__global__ void __launch_bounds__(256) rrn_cols_kernel(Bwd a) {
  const int64_t j = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (j >= a.N) return;
  const W *wp = (const W*)a.wp, *sv = (const W*)a.sv;
  const int64_t rows = (a.M + gridDim.y - 1) / gridDim.y;
  const int64_t r0 = blockIdx.y * rows, r1 = r0 + rows < a.M ? r0 + rows : a.M;
  const float wj = to_f<W>(((const W*)a.w)[j]);
  const float sj = (sv ? to_f<W>(sv[j]) : a.s) * (wp ? to_f<W>(wp[j]) : 1.f);
  float dw = 0.f, A = 0.f;
  for (int64_t row = r0; row < r1; ++row) {
    const float inv1 = wp ? a.inv1[row] : 1.f, inv2 = a.inv2[row];
    const float n = to_f<T>(((const T*)a.y)[row * a.y_ld + j]) * inv1;
    const float av = a.gate ? act_of(a.act, to_f<T>(((const T*)a.gate)[row * a.g_ld + j])) : 1.f;
    const float r2 = fmaf(sj * av, n, to_f<T>(((const T*)a.r)[row * a.r_ld + j]));
    const float d = a.dout ? to_f<T>(((const T*)a.dout)[row * a.N + j]) : 0.f;
    const float D = fmaf(inv2, d * wj, fmaf(-a.c2[row], r2,
                         a.dres ? to_f<T>(((const T*)a.dres)[row * a.N + j]) : 0.f));
    dw = fmaf(d * r2, inv2, dw);
    A = fmaf(D, av * n, A);
  }
  float* part = a.part + (int64_t)blockIdx.y * a.N + j;
  part[0] = dw;
  part[(int64_t)gridDim.y * a.N] = A;
}

// dw, or ds = w_post A and dw_post = s A, from the G partial rows.  A CTA owns 32 columns; warp q adds the rows q, q + 16,
// ..., then warp 0 the 16 warps' sums: an order that does not depend on scheduling.
constexpr int kReduceWarps = 16;
template <typename W>
__global__ void __launch_bounds__(32 * kReduceWarps) rrn_reduce_kernel(Bwd a, int G) {
  __shared__ float acc[kReduceWarps][33];
  const int lane = threadIdx.x & 31, q = threadIdx.x >> 5;
  const int64_t j = (int64_t)blockIdx.x * 32 + lane;
  if (blockIdx.y == 1 && !a.ds && !a.dwp) return;
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
    const W *wp = (const W*)a.wp, *sv = (const W*)a.sv;
    if (blockIdx.y == 0) {
      ((W*)a.dw)[j] = from_f<W>(t);
    } else {
      if (a.ds) ((W*)a.ds)[j] = from_f<W>(wp ? t * to_f<W>(wp[j]) : t);
      if (a.dwp) ((W*)a.dwp)[j] = from_f<W>(t * (sv ? to_f<W>(sv[j]) : a.s));
    }
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

// Calls f(TPR, VPT, WIDE) with the smallest shape whose threads cover a row of N elements: a warp or
// less for the narrowest rows (no barrier), else a CTA of up to 512 threads, and 1024 for
// the widest (the forward's; backward two CTAs of 512 share such a row).  Returns -1 where none does.
template <typename T, typename F> int with_shape(bool wide, int64_t N, F&& f) {
  using std::integral_constant;
  auto go = [&](auto tpr, auto vpt, auto w) {
    return f(integral_constant<int, tpr>{}, integral_constant<int, vpt>{}, w);
  };
#define FO_SHAPE(TPR, VPT, PER, W) \
  if (N <= (int64_t)TPR * VPT * PER) return go(integral_constant<int, TPR>{}, integral_constant<int, VPT>{}, W{})
  if (wide) {
    constexpr int E = Vec16<T>::E;
    FO_SHAPE(8, 1, E, std::true_type);
    FO_SHAPE(32, 1, E, std::true_type);
    FO_SHAPE(64, 1, E, std::true_type);
    FO_SHAPE(128, 1, E, std::true_type);
    FO_SHAPE(256, 1, E, std::true_type);
    FO_SHAPE(512, 1, E, std::true_type);
    FO_SHAPE(512, 2, E, std::true_type);
    FO_SHAPE(1024, 2, E, std::true_type);
  } else {
    FO_SHAPE(32, 1, 2, std::false_type);
    FO_SHAPE(32, 2, 2, std::false_type);
    FO_SHAPE(128, 2, 2, std::false_type);
    FO_SHAPE(256, 2, 2, std::false_type);
    FO_SHAPE(512, 2, 2, std::false_type);
    FO_SHAPE(512, 4, 2, std::false_type);
  }
#undef FO_SHAPE
  return -1;
}

template <typename T>
bool wide_ok(int64_t N, const void* const* rows, const int64_t* lds, int n,
             const void* const* vectors, int nv) {
  constexpr int E = Vec16<T>::E;
  bool ok = N % E == 0;
  for (int i = 0; i < n; ++i) ok = ok && aligned16(rows[i]) && lds[i] % E == 0;
  for (int i = 0; i < nv; ++i) ok = ok && aligned16(vectors[i]);
  return ok;
}

template <typename K, typename A>
int launch(const char* what, K kernel, int64_t ctas, int threads, int smem, const A& a,
           cudaStream_t st, int cluster = 1) {
  if (smem > 40 * 1024) {
    cudaError_t e = allow_shared((const void*)kernel, 227 * 1024 - 1024);
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("%s: %s", what, cudaGetErrorString(e));
      return FO_ECUDA;
    }
  }
  if (cluster == 1) {
    kernel<<<(unsigned)ctas, threads, smem, st>>>(a);
    return check_launch(what);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(ctas * cluster));
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = cluster;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, a)) {
    cudaGetLastError();
    set_error("%s: %s", what, cudaGetErrorString(e));
    return FO_ECUDA;
  }
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
  const int rc = with_shape<T>(wide_ok<T>(a.N, rows, lds, 5, vs, 3), a.N, [&](auto tpr, auto vpt, auto wide) {
    using S = Shape<tpr>;
    constexpr int smem = Columns<T, W, tpr, vpt, wide, 3>::kRingBytes;
    const int64_t most = num_sms() * resident(1024, S::kThreads, smem);
    const int64_t need = (a.M + S::kRows - 1) / S::kRows;
    return launch("rrn_fwd_kernel", rrn_fwd_kernel<T, W, tpr, vpt, wide>, need < most ? need : most,
                  S::kThreads, smem, a, st);
  });
  if (rc != -1) return rc;
  rrn_fwd_generic_kernel<T, W><<<row_grid(a.M), 256, 0, st>>>(a);
  return check_launch("rrn_fwd_generic_kernel");
}

template <typename T, typename W>
int run_bwd(const Bwd& a, cudaStream_t st) {
  const void *rows[] = {a.y, a.r, a.gate, a.dout, a.dres, a.dy, a.dr, a.dgate},
             *vs[] = {a.w, a.wp, a.sv};
  const int64_t lds[] = {a.y_ld, a.r_ld, a.g_ld, a.N, a.N, a.N, a.N, a.N};
  int G = 0;
  int rc = with_shape<T>(wide_ok<T>(a.N, rows, lds, 8, vs, 3), a.N, [&](auto tpr, auto vpt, auto wide) {
    using S = Shape<tpr>;
    constexpr int kCtas = tpr > 512 ? 2 : 1, kTpr = tpr / kCtas;  // of a row
    using Half = Shape<kTpr>;
    const int64_t columns = (a.N + kCtas - 1) / kCtas + (kCtas > 1 ? Vec16<T>::E : 0);
    const int ring = Columns<T, W, kTpr, vpt, wide, 5>::kRingBytes + weight_bytes(columns);
    const int sums = Half::kRows > 1 ? (int)(Half::kRows * 2 * a.N * 4) : 0;
    const int smem = ring > sums ? ring : sums;
    int64_t ctas = num_sms() / kCtas * resident(512, Half::kThreads, smem);
    const int64_t need = (a.M + Half::kRows - 1) / Half::kRows, most = partial_rows(a.M, a.N);
    if (ctas > need) ctas = need;
    if (ctas > most) ctas = most;
    G = (int)ctas;
    return launch("rrn_bwd_kernel", rrn_bwd_kernel<T, W, kTpr, vpt, wide, kCtas>, ctas, Half::kThreads,
                  smem, a, st, kCtas);
  });
  if (rc == -1) {
    rrn_bwd_generic_kernel<T, W><<<row_grid(a.M), 256, 0, st>>>(a);
    if (int e = check_launch("rrn_bwd_generic_kernel")) return e;
    G = (int)(a.M < kChunks ? a.M : kChunks);
    rrn_cols_kernel<T, W><<<dim3((unsigned)((a.N + 255) / 256), G), 256, 0, st>>>(a);
    rc = check_launch("rrn_cols_kernel");
  }
  if (rc) return rc;
  rrn_reduce_kernel<W><<<dim3((unsigned)((a.N + 31) / 32), 2), 32 * kReduceWarps, 0, st>>>(a, G);
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
  *bytes = ((M + 3) / 4 * 4 + 2 * partial_rows(M, N) * N) * 4;  // c2 of each row, partial rows
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
