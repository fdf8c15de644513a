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
//   logits:  du = D (a h_{t-1} - a^2 / (1 - a^2) b),  dg = du u (1 - sigmoid(g)),
//            ddecay = sigmoid(decay) / softplus(decay) * sum du u,
//            dx = D m i,  dbeta = D b (1 - i)
//   and dg = du = 0 at a reset step; dh0 = a_0 D_0.
// The states h_{t-1} are recomputed in fp32 from the state the forward keeps in front of every
// FO_GLR_CHECKPOINT-th step: recomputing costs no traffic beyond x, g and beta, which the
// backward reads anyway, and gradients do not see the output's rounding to 16 bits.
// All of it is held in fp32; h and the gradients are rounded once when they are written.
//
// Split.  Channels are cut into slabs of 32 lanes (two channels a lane with 16-bit gates where C, the
// strides and the addresses allow it, so that a warp's row is a 128-byte line), time into rounds.
// In a round each of a CTA's 8 warps takes 16 (backward: 8) consecutive steps, whose gates it
// computes independently of any state; over them it is a map s -> A s + H (backward: R -> A R + Q),
// and it walks them once, from the state that enters them.  That state comes
//  - where slabs * B give every SM a CTA: from the neighbouring warp, as a chain through shared memory
//    (an mbarrier a link), so that warps run ahead of one another and the gates of one overlap the
//    walk of another (235 us against 266 us with a barrier for all warps when it came, forward at
//    8 x 8192 x 2048 bf16 logits; 240 us now);
//  - with fewer slabs: up to 8 CTAs of a cluster take consecutive tiles, each warp's map is put
//    together with those in front of it, and the CTAs exchange theirs as asynchronous stores that an
//    mbarrier of the receiver counts (a cluster barrier waits for the outputs' stores too: backward
//    216 us with it, 192 us so, at 1 x 16384 x 2048 bf16).
// Inputs come through a ring of two rounds in shared memory (cp.async), which each warp fills and reads
// by itself.  Every input is read once and every output written once.
//
// What bounds it (1 x B200, 8 x 8192 x 2048 bf16): gates as values 200 us forward and 355 us backward
// (floors 164 and 287 us at the measured rate of a copy), with fp32 gates 268 and 570 (246 and 451).
// With logits an element takes five exponentials, reciprocals and roots, which alone take 150 us:
// 240 us forward, 510 us backward (140 instructions for a pair of channels at 55 % of the issue rate, and
// no more than 16 warps on an SM: two CTAs of 256 threads with up to 128 registers are all its
// registers).  fp32 logits 315 and 735 us.  All of them lose an eighth to 256 CTAs on 148 SMs.

#include <type_traits>

#include "cluster.cuh"
#include "gates.cuh"

namespace fo {
namespace {

// Steps of a thread in a round, and warps of a CTA.  Forward at 8 x 8192 x 2048 bf16, in one comparison:
// 235 us; with 8 steps and 16 warps 239, 8 and 8 267, 16 and 12 263, 4 and 16 288.  Backward needs the
// registers for 8 steps.
constexpr int kFwdSteps = 16, kFwdWarps = 8;
constexpr int kFwdTile = kFwdSteps * kFwdWarps;
constexpr int kBwdSteps = 8, kBwdWarps = 8;
constexpr int kBwdTile = kBwdSteps * kBwdWarps;
constexpr int kMostCtas = 8;                   // of a cluster
constexpr int kStages = 2;                 // tiles of the ring
static_assert(kBwdTile == FO_GLR_CHECKPOINT, "a tile of the backward begins at a checkpoint");
static_assert(kMostCtas <= kFwdWarps && kMostCtas <= kBwdWarps, "a warp for each CTA");
static_assert(FO_GLR_CHECKPOINT % kFwdSteps == 0, "a warp's steps begin at a checkpoint or have none");

struct Strides {
  int64_t xb, xl, gb, gl, bb, bl;  // batch and step strides of x, g, beta, in elements
};

// a b, rounded: the compiler does not make it part of an fma, so that single values and pairs agree
__device__ __forceinline__ float product(float a, float b) { return __fmul_rn(a, b); }
__device__ __forceinline__ float2 product(float2 a, float2 b) { return mul_(a, b); }

// v = 1 - e^{-w} for w = 2 y, from a near e^{-y} on the way in.  Up to w = 1/2 it is w p(w), p the
// interpolation of (1 - e^{-w}) / w at the six Chebyshev nodes, relative error 3e-9: 1 - a^2 would lose 1 / w
// there, above it loses at most a factor 2.5.  And a, an approximate exponential, is up to 2 units of its
// last place off, mostly to one side, which a state that remembers 1 / (1 - a) steps would gather: it is
// mended by half of what 1 - a^2 (rounded once) differs from v (1 / (2 a) of it for a near 1).
template <typename F> __device__ __forceinline__ F one_minus_square(F w, F& a) {
  F p = fma_(w, all_<F>(-1.1234042e-3f), all_<F>(8.1896139e-3f));
  p = fma_(w, p, all_<F>(-4.1630074e-2f));
  p = fma_(w, p, all_<F>(0.16666242f));
  p = fma_(w, p, all_<F>(-0.49999982f));
  p = fma_(w, p, all_<F>(1.f));
  const F f = fma_(a, a, all_<F>(-1.f));  // a^2 - 1
  const F v = map_([](float w_, float s, float l) { return w_ < 0.5f ? s : -l; }, w, product(w, p), f);
  a = fma_(add_(f, v), all_<F>(-0.5f), a);
  return v;
}
__device__ __forceinline__ float sqrt_(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float rsqrt_(float x) {
  float y;
  asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float softplus(float decay) {
  return decay > 20.f ? decay : log1pf(expf(decay));
}
// -log a of a fully open gate.  Kept finite: times a closed gate's 0, and the gradient's 0 where a is 0,
// it has to be 0.
__device__ __forceinline__ float rate_of(float scale, float decay) {
  const float r = scale * softplus(decay);
  return r > 1e30f ? 1e30f : r;
}

// The state s behind a segment that maps it to A s + H.  Where a segment may hold a reset (A is 0),
// what is in front of it is not looked at, not even a NaN.
template <bool RESET, typename F> __device__ __forceinline__ F through(F s, F A, F H) {
  if (RESET) return map_([](float s_, float a, float h) { return a == 0.f ? h : fmaf(a, s_, h); }, s, A, H);
  return fma_(A, s, H);
}
// A product of gates above 1 may leave the fp32 range over a state of zero: kept finite, it adds 0.
// RESET: a segment with a reset has the factor 0, so its product is 0, or NaN where another gate is NaN
// or the others leave the range; that is 0 too, and nothing crosses the reset.  Without a reset in the
// segment a NaN gate has made H NaN, which is what passes on.  (Selecting 0 by the reset bits spills
// registers: forward 281 us so and 305 with the bits, 8 x 8192 x 2048 bf16 logits.)
template <bool RESET, typename F> __device__ __forceinline__ F finite(F A) {
  return map_([](float a) {
    const float f = fminf(fmaxf(a, -3.4028235e38f), 3.4028235e38f);
    return RESET && a != a ? 0.f : f;
  }, A);
}

// ---------------------------------------------------------------------------
// Elements of a lane: V channels of T in memory, F (float or float2) in registers
// ---------------------------------------------------------------------------
template <int V> struct Lane;
template <> struct Lane<1> { using F = float; };
template <> struct Lane<2> { using F = float2; };

template <int BYTES> struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };

template <typename T, int V> struct Elem {
  static constexpr int kBytes = V * (int)sizeof(T);
  using W = typename Word<kBytes>::type;
  using F = typename Lane<V>::F;
  static __device__ __forceinline__ F load(const void* p) {
    if constexpr (V == 1) return to_f<T>(*reinterpret_cast<const T*>(p));
    else if constexpr (sizeof(T) == 2) return unpack2<T>(*reinterpret_cast<const uint32_t*>(p));
    else return *reinterpret_cast<const float2*>(p);
  }
  static __device__ __forceinline__ void store(T* p, F v) {
    if constexpr (V == 1) *p = from_f<T>(v);
    else if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(p) = pack2<T>(v);
    else *reinterpret_cast<float2*>(p) = v;
  }
  static __device__ __forceinline__ void zero(void* smem) { *reinterpret_cast<W*>(smem) = W{}; }
  // global -> shared without waiting (2-byte elements have no such copy: through a register)
  static __device__ __forceinline__ void copy(void* smem, const T* p) {
    if constexpr (kBytes == 2) {
      *reinterpret_cast<W*>(smem) = *reinterpret_cast<const W*>(p);
    } else {
      asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(
                       (uint32_t)__cvta_generic_to_shared(smem)),
                   "l"(p), "n"(kBytes)
                   : "memory");
    }
  }
};
// One input of a warp: STEPS rows a round into its part of the ring, `round` bytes apart in memory
// from one round to the next.  wide: 16 bytes a copy, rows shared out over the lanes (so a
// __syncwarp has to follow the wait); otherwise every lane copies just its own elements.  Lanes
// without a channel and rows from `rows` on are left out.
template <typename T, int V, int STEPS> struct Stream {
  using E = Elem<T, V>;
  static constexpr int kRow = 32 * E::kBytes;     // bytes of a row in the ring
  static constexpr int kBytes = STEPS * kRow;     // of a warp's part of a stage
  static constexpr int kPer = 512 / kRow;         // rows of a warp's 16-byte copies
  const uint8_t* p;
  int64_t step, round;
  int row0;
  bool on, wide;
  // first: the first element of the slab in the warp's first row; left: channels of the slab
  __device__ __forceinline__ Stream(const T* first, int64_t step_, int64_t round_, int64_t left,
                                    bool wide_)
      : step(step_ * (int)sizeof(T)), round(round_ * (int)sizeof(T)), wide(wide_) {
    const int lane = threadIdx.x & 31;
    row0 = wide ? lane / (kRow / 16) : 0;
    const int byte = wide ? lane % (kRow / 16) * 16 : lane * E::kBytes;
    on = byte < left * (int)sizeof(T);
    p = reinterpret_cast<const uint8_t*>(first) + row0 * step + byte;
  }
  __device__ __forceinline__ void fetch(uint8_t* ring, int rows) {
    const int lane = threadIdx.x & 31;
    if (on) {
      if (wide) {
        const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring) + lane * 16;
        const uint8_t* q = p;
#pragma unroll
        for (int k = 0; k < STEPS / kPer; ++k, q += kPer * step)
          if (rows == STEPS || k * kPer + row0 < rows)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + k * 512), "l"(q)
                         : "memory");
      } else {
        const uint8_t* q = p;
#pragma unroll
        for (int i = 0; i < STEPS; ++i, q += step)
          if (i < rows) E::copy(ring + i * kRow + lane * E::kBytes, reinterpret_cast<const T*>(q));
      }
    }
    p += round;
  }
};
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// ---------------------------------------------------------------------------
// Links between warps and between the CTAs of a cluster
// ---------------------------------------------------------------------------
// Two values into CTA `cta`'s copy of `to`, counted by its copy of `bar`
__device__ __forceinline__ void send(void* to, const uint64_t* bar, uint32_t cta, float a, float h) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [%0], {%1, %2}, [%3];" ::"r"(
                   remote_address(to, cta)),
               "f"(a), "f"(h), "r"(remote_address(bar, cta))
               : "memory");
}
__device__ __forceinline__ void send(void* to, const uint64_t* bar, uint32_t cta, float2 a, float2 h) {
  asm volatile(
      "st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%1, %2, %3, %4}, [%5];" ::"r"(
          remote_address(to, cta)),
      "f"(a.x), "f"(a.y), "f"(h.x), "f"(h.y), "r"(remote_address(bar, cta))
      : "memory");
}
__device__ unsigned int g_glr_timeouts = 0;
constexpr int kMaxPolls = 1 << 22;
// Waits for phase `parity` of the mbarrier; gives up (and says so) after kMaxPolls polls.
template <bool CLUSTER> __device__ __forceinline__ bool wait_phase(const uint64_t* bar, uint32_t parity) {
  for (int i = 0; i < kMaxPolls; ++i) {
    uint32_t done;
    if (CLUSTER)
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(shared_address(bar)), "r"(parity)
          : "memory");
    else
      asm volatile(
          "{\n\t.reg .pred p;\n\t"
          "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(done)
          : "r"(shared_address(bar)), "r"(parity)
          : "memory");
    if (done) return true;
  }
  return false;
}

// A chain of states through the warps of a CTA: warp w puts the state behind its steps of a round,
// and its neighbour gets it.  Two places a warp, used in turn: a warp comes to round r + 2 only
// with the state that its neighbour has put in round r + 1, behind its get of round r.
template <typename F, int WARPS> struct Chain {
  F state[2][WARPS][32];
  uint64_t bar[2][WARPS];
  bool dead;

  __device__ __forceinline__ void init() {  // __syncthreads has to follow
    if (threadIdx.x < 2 * WARPS)
      asm volatile("mbarrier.init.shared.b64 [%0], 1;" ::"r"(shared_address(&bar[0][0] + threadIdx.x))
                   : "memory");
    if (threadIdx.x == 0) dead = false;
  }
  __device__ __forceinline__ void put(int64_t round, int w, F s) {
    const int parity = (int)(round & 1), lane = threadIdx.x & 31;
    state[parity][w][lane] = s;
    __syncwarp();
    if (lane == 0)
      asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(shared_address(&bar[parity][w])) : "memory");
  }
  __device__ __forceinline__ F get(int64_t round, int w) {
    const int parity = (int)(round & 1);
    if (!dead && !wait_phase<false>(&bar[parity][w], (uint32_t)(round >> 1) & 1)) {
      dead = true;  // no further waits: the kernel ends, its outputs are not complete
      atomicAdd(&g_glr_timeouts, 1u);
    }
    return state[parity][w][threadIdx.x & 31];
  }
};

// The maps of a round: of the CTA's warps, and (clusters) of the cluster's CTAs.  Two copies,
// used in turn.  One of the CTA is written again only behind a barrier that every reader of it has
// passed; one of the cluster only by CTAs that have what this one sent after its readers' last
// __syncthreads.
template <typename F, int WARPS, int CTAS> struct Maps {
  struct alignas(2 * sizeof(F)) Both {
    F A, H;
  };
  F A[2][WARPS][32], H[2][WARPS][32];
  Both cta[2][CTAS][32];
  uint64_t bar[2];
  bool dead;

  __device__ __forceinline__ void init() {
    if (threadIdx.x == 0) {
      dead = false;
      for (int k = 0; k < 2; ++k)
        asm volatile("mbarrier.init.shared.b64 [%0], 1;" ::"r"(shared_address(&bar[k])) : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    cluster_barrier();
  }
};

// With the maps of all warps in place, and the state S in front of round number `round`: the state
// in front of warp w's steps; S becomes the state behind the round.  REVERSE walks the warps and CTAs
// from the last to the first.
template <bool REVERSE, bool RESET, typename F, int WARPS, int CTAS>
__device__ __forceinline__ F carry_in(Maps<F, WARPS, CTAS>& m, int64_t round, int w, F& S) {
  const int lane = threadIdx.x & 31, parity = (int)(round & 1);
  const uint32_t n = cluster_size(), me = cluster_rank();
  F mine = S;
  if (threadIdx.x == 0)
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"(shared_address(&m.bar[parity])),
                 "r"(n * 32 * (uint32_t)sizeof(typename Maps<F, WARPS, CTAS>::Both))
                 : "memory");
  if (w < (int)n) {  // warp w hands the CTA's map to CTA w
    F a = all_<F>(1.f), h = all_<F>(0.f);
#pragma unroll
    for (int k = 0; k < WARPS; ++k) {
      const int q = REVERSE ? WARPS - 1 - k : k;
      const F ak = m.A[parity][q][lane];
      h = through<RESET>(h, ak, m.H[parity][q][lane]);
      a = finite<false>(mul_(a, ak));
    }
    send(&m.cta[parity][me][lane], &m.bar[parity], w, a, h);
  }
  if (!m.dead && !wait_phase<true>(&m.bar[parity], (uint32_t)(round >> 1) & 1)) {
    m.dead = true;  // no further waits: the kernel ends, its outputs are not complete
    atomicAdd(&g_glr_timeouts, 1u);
  }
  for (uint32_t k = 0; k < n; ++k) {
    const uint32_t q = REVERSE ? n - 1 - k : k;
    if (q == me) mine = S;
    S = through<RESET>(S, m.cta[parity][q][lane].A, m.cta[parity][q][lane].H);
  }
#pragma unroll
  for (int k = 0; k < WARPS - 1; ++k) {
    const int q = REVERSE ? WARPS - 1 - k : k;
    if (REVERSE ? q > w : q < w) mine = through<RESET>(mine, m.A[parity][q][lane], m.H[parity][q][lane]);
  }
  return mine;
}

// What a thread's place is: batch b, first channel c, rank and size of the cluster.
struct Place {
  int64_t b, c0, c;  // c0: the slab's first channel
  int rank, size;
  bool on;  // the lane has a channel
};
template <int V, bool CLUSTER> __device__ __forceinline__ Place place(int64_t C) {
  Place p;
  p.rank = CLUSTER ? (int)cluster_rank() : 0;
  p.size = CLUSTER ? (int)cluster_size() : 1;
  const int64_t slabs = (C + 32 * V - 1) / (32 * V), i = blockIdx.x / p.size;
  p.b = i / slabs;
  p.c0 = (i % slabs) * (32 * V);
  p.c = p.c0 + (threadIdx.x & 31) * V;
  p.on = p.c < C;
  return p;
}

// The warp of the thread, in a form that the compiler knows to be the same for all lanes.
__device__ __forceinline__ int warp_index() {
  return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0);
}

// Bit i: the warp's step t0 + i is a reset (of its `rows` steps).
__device__ __forceinline__ uint32_t reset_bits(const uint8_t* reset, int64_t t0, int rows) {
  const int lane = threadIdx.x & 31;
  const bool r = lane < rows && reset[t0 + lane] != 0;
  return __ballot_sync(0xffffffffu, r);
}

// ---------------------------------------------------------------------------
// Forward
// ---------------------------------------------------------------------------
template <typename T, typename G, int V> struct FwdRing {
  uint8_t x[kStages][kFwdWarps][Stream<T, V, kFwdSteps>::kBytes];
  uint8_t g[kStages][kFwdWarps][Stream<G, V, kFwdSteps>::kBytes];
  uint8_t b[kStages][kFwdWarps][Stream<G, V, kFwdSteps>::kBytes];
};

template <typename T, typename G, int V, bool LOGITS, bool RESET, int CTAS>
__global__ void __launch_bounds__(32 * kFwdWarps, 2)
glr_fwd_kernel(const T* __restrict__ x, const G* __restrict__ g, const G* __restrict__ beta,
               const float* __restrict__ decay, const float* __restrict__ h0,
               const uint8_t* __restrict__ reset, T* __restrict__ h, float* __restrict__ hT,
               float* __restrict__ ckpt, int64_t L, int64_t C, Strides st, float scale, bool wide) {
  using F = typename Lane<V>::F;
  using EX = Elem<T, V>;
  using EG = Elem<G, V>;
  constexpr int N = kFwdSteps;
  extern __shared__ __align__(16) uint8_t smem[];
  auto& ring = *reinterpret_cast<FwdRing<T, G, V>*>(smem);
  __shared__ std::conditional_t<(CTAS > 1), Maps<F, kFwdWarps, CTAS>, Chain<F, kFwdWarps>> link;
  link.init();
  __syncthreads();
  const Place p = place<V, (CTAS > 1)>(C);
  const int lane = threadIdx.x & 31, w = warp_index();
  const int64_t tiles = (L + kFwdTile - 1) / kFwdTile, rounds = (tiles + p.size - 1) / p.size;
  const int64_t checkpoints = (L + FO_GLR_CHECKPOINT - 1) / FO_GLR_CHECKPOINT;
  const int64_t per_round = (int64_t)p.size * kFwdTile;
  int64_t t0 = (int64_t)p.rank * kFwdTile + w * N;  // the warp's first step of the round
  Stream<T, V, N> in_x(x + p.b * st.xb + t0 * st.xl + p.c0, st.xl, per_round * st.xl, C - p.c0, wide);
  Stream<G, V, N> in_g(g + p.b * st.gb + t0 * st.gl + p.c0, st.gl, per_round * st.gl, C - p.c0, wide);
  Stream<G, V, N> in_b(beta + p.b * st.bb + t0 * st.bl + p.c0, st.bl, per_round * st.bl, C - p.c0, wide);
  if (RESET) reset += p.b * L;
  F r1 = all_<F>(0.f), r2 = all_<F>(0.f);  // log2 a and -2 log a of an open gate
  F S = all_<F>(0.f);
  if (p.on) {
    if (LOGITS) {
      const F rate = map_([&](float d) { return rate_of(scale, d); },
                          Elem<float, V>::load(decay + p.c));
      r1 = mul_(rate, all_<F>(-kLog2e));
      r2 = mul_(rate, all_<F>(2.f));
    }
    if (h0) S = Elem<float, V>::load(h0 + p.b * C + p.c);
  }
  auto rows_of = [&](int64_t t) { return t < L ? (int)(L - t < N ? L - t : N) : 0; };
  int64_t t_fetch = t0;
  auto fetch = [&](int stage) {
    if (const int n = rows_of(t_fetch)) {
      in_x.fetch(ring.x[stage][w], n);
      in_g.fetch(ring.g[stage][w], n);
      in_b.fetch(ring.b[stage][w], n);
    }
    t_fetch += per_round;
    copy_commit();
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) fetch(k);
  T* to = h + (p.b * L + t0) * C + p.c0;
  for (int64_t round = 0; round < rounds; ++round, t0 += per_round, to += per_round * C) {
    const int n = rows_of(t0), s = (int)(round % kStages);
    fetch((int)((round + kStages - 1) % kStages));
    const uint32_t rs = RESET ? reset_bits(reset, t0, n) : 0;
    copy_wait<kStages - 1>();
    __syncwarp();
    F a[N], b[N], A = all_<F>(1.f), H = all_<F>(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F xv = EX::load(&ring.x[s][w][(i * 32 + lane) * EX::kBytes]);
      const F gv = EG::load(&ring.g[s][w][(i * 32 + lane) * EG::kBytes]);
      const F bv = EG::load(&ring.b[s][w][(i * 32 + lane) * EG::kBytes]);
      if (LOGITS) {
        // sigmoid(g) = 1 / (1 + e^-g), 0 and 1 at -inf and +inf.  With v = 1 - a^2, r = e^-|beta| and
        // q = 1 + r, m i is sqrt(v) / q, times r where beta is negative; sqrt(v) / q = v rsqrt(v q^2) saves
        // one of six of the slow instructions (exponentials, reciprocals, roots) that bound this kernel.
        const F sg = map_(rcp, add_(map_(ex2, mul_(gv, all_<F>(-kLog2e))), all_<F>(1.f)));
        a[i] = map_(ex2, mul_(sg, r1));
        F v = one_minus_square(mul_(sg, r2), a[i]);
        if (RESET && (rs >> i & 1)) v = all_<F>(1.f);
        const F e = mul_(bv, all_<F>(kLog2e));
        const F r = map_([](float t) { return ex2(-fabsf(t)); }, e), q = add_(r, all_<F>(1.f));
        const F xr = mul_(xv, map_([](float t, float r_) { return t < 0.f ? r_ : 1.f; }, e, r));
        // 1e-36: no root of 0 where a == 1, and v then makes the product 0
        const F t = map_(rsqrt_, fma_(mul_(v, q), q, all_<F>(1e-36f)));
        b[i] = mul_(mul_(v, t), xr);
      } else {
        a[i] = gv;
        b[i] = mul_(bv, xv);
      }
      if (RESET && (rs >> i & 1)) a[i] = all_<F>(0.f);
    }
    if (n < N) {  // behind the end: the state passes
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i >= n) {
          a[i] = all_<F>(1.f);
          b[i] = all_<F>(0.f);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (RESET && (rs >> i & 1)) H = all_<F>(0.f);
      A = mul_(A, a[i]);
      H = fma_(a[i], H, b[i]);
    }
    A = finite<RESET>(A);
    F hv = S;  // the state in front of the warp's steps
    if constexpr (CTAS > 1) {
      link.A[round & 1][w][lane] = A;
      link.H[round & 1][w][lane] = H;
      __syncthreads();
      hv = carry_in<false, RESET>(link, round, w, S);
    } else {
      if (round > 0 || w > 0) hv = link.get(w ? round : round - 1, w ? w - 1 : kFwdWarps - 1);
      link.put(round, w, through<RESET>(hv, A, H));
    }
    if (p.on) {
      if (ckpt && n > 0 && t0 % FO_GLR_CHECKPOINT == 0)
        Elem<float, V>::store(ckpt + (p.b * checkpoints + t0 / FO_GLR_CHECKPOINT) * C + p.c, hv);
      auto walk = [&](auto full) {
        T* q = to;
#pragma unroll
        for (int i = 0; i < N; ++i, q += C) {
          if (RESET && (rs >> i & 1)) hv = all_<F>(0.f);
          hv = fma_(a[i], hv, b[i]);
          if (full || i < n) EX::store(q + lane * V, hv);
        }
      };
      if (n == N) walk(std::true_type{});
      else walk(std::false_type{});
      // the warp that has the last step
      if (hT && n > 0 && t0 + n == L) Elem<float, V>::store(hT + p.b * C + p.c, hv);
    }
    __syncwarp();
  }
  if (L == 0 && hT && p.on && w == 0) Elem<float, V>::store(hT + p.b * C + p.c, S);
  copy_wait<0>();
  if constexpr (CTAS > 1) cluster_meet();  // none leaves while another may send to it
}

// ---------------------------------------------------------------------------
// Backward
// ---------------------------------------------------------------------------
template <typename T, typename G, int V> struct BwdRing {
  using F = typename Lane<V>::F;
  uint8_t x[kStages][kBwdWarps][Stream<T, V, kBwdSteps>::kBytes];
  uint8_t d[kStages][kBwdWarps][Stream<T, V, kBwdSteps>::kBytes];
  uint8_t g[kStages][kBwdWarps][Stream<G, V, kBwdSteps>::kBytes];
  uint8_t b[kStages][kBwdWarps][Stream<G, V, kBwdSteps>::kBytes];
  // Of the round between its first and last walk, where registers would spill: m i and
  // a^2 / (1 - a^2); 1 - i takes the place of g and beta in the ring.  Gates as values do not need
  // them; leaving them out would admit no further CTA, since registers limit the number first.
  F mi[kBwdWarps][kBwdSteps][32], q[kBwdWarps][kBwdSteps][32];

  // one F a lane in the places of g and beta of step i, which are not needed any more
  __device__ __forceinline__ void put_gates(int s, int w, int i, int lane, F f) {
    uint8_t *pg = &g[s][w][(i * 32 + lane) * Elem<G, V>::kBytes],
            *pb = &b[s][w][(i * 32 + lane) * Elem<G, V>::kBytes];
    if constexpr (V == 2) {
      *reinterpret_cast<float*>(pg) = f.x;
      *reinterpret_cast<float*>(pb) = f.y;
    } else if constexpr (sizeof(G) == 4) {
      *reinterpret_cast<float*>(pg) = f;
    } else {
      *reinterpret_cast<uint16_t*>(pg) = (uint16_t)(__float_as_uint(f) >> 16);
      *reinterpret_cast<uint16_t*>(pb) = (uint16_t)__float_as_uint(f);
    }
  }
  __device__ __forceinline__ F get_gates(int s, int w, int i, int lane) const {
    const uint8_t *pg = &g[s][w][(i * 32 + lane) * Elem<G, V>::kBytes],
                  *pb = &b[s][w][(i * 32 + lane) * Elem<G, V>::kBytes];
    if constexpr (V == 2)
      return make_float2(*reinterpret_cast<const float*>(pg), *reinterpret_cast<const float*>(pb));
    else if constexpr (sizeof(G) == 4)
      return *reinterpret_cast<const float*>(pg);
    else
      return __uint_as_float((uint32_t)*reinterpret_cast<const uint16_t*>(pg) << 16 |
                             *reinterpret_cast<const uint16_t*>(pb));
  }
};

template <typename T, typename G, int V, bool LOGITS, bool RESET, int CTAS>
__global__ void __launch_bounds__(32 * kBwdWarps, 2)
glr_bwd_kernel(const T* __restrict__ x, const G* __restrict__ g, const G* __restrict__ beta,
               const float* __restrict__ decay, const uint8_t* __restrict__ reset,
               const float* __restrict__ ckpt, const T* __restrict__ dh,
               const float* __restrict__ dhT, T* __restrict__ dx, G* __restrict__ dg,
               G* __restrict__ dbeta, float* __restrict__ dh0, float* __restrict__ ddecay_part,
               int64_t L, int64_t C, Strides st, float scale, bool wide) {
  using F = typename Lane<V>::F;
  using EX = Elem<T, V>;
  using EG = Elem<G, V>;
  constexpr int N = kBwdSteps, WARPS = kBwdWarps;
  extern __shared__ __align__(16) uint8_t smem[];
  auto& ring = *reinterpret_cast<BwdRing<T, G, V>*>(smem);
  // links of the a_t D_t of the steps behind (R -> A R + Q), and of the states in front (s -> A s + H)
  __shared__ std::conditional_t<(CTAS > 1), Maps<F, WARPS, CTAS>, Chain<F, WARPS>> link;
  __shared__ std::conditional_t<(CTAS > 1), F[2][WARPS][32], Chain<F, WARPS>> link_h;
  link.init();
  if constexpr (CTAS == 1) link_h.init();
  __syncthreads();
  const Place p = place<V, (CTAS > 1)>(C);
  const int lane = threadIdx.x & 31, w = warp_index();
  const int64_t tiles = (L + kBwdTile - 1) / kBwdTile, rounds = (tiles + p.size - 1) / p.size;
  const int64_t per_round = (int64_t)p.size * kBwdTile;
  // the warp's first step of the round, from the last round to the first
  int64_t t0 = ((rounds - 1) * p.size + p.rank) * kBwdTile + w * N;
  Stream<T, V, N> in_x(x + p.b * st.xb + t0 * st.xl + p.c0, st.xl, -per_round * st.xl, C - p.c0, wide);
  Stream<G, V, N> in_g(g + p.b * st.gb + t0 * st.gl + p.c0, st.gl, -per_round * st.gl, C - p.c0, wide);
  Stream<G, V, N> in_b(beta + p.b * st.bb + t0 * st.bl + p.c0, st.bl, -per_round * st.bl, C - p.c0, wide);
  Stream<T, V, N> in_d(dh + (p.b * L + t0) * C + p.c0, C, -per_round * C, C - p.c0, wide);
  if (RESET) reset += p.b * L;
  F rate = all_<F>(0.f), sum = all_<F>(0.f);
  F R = all_<F>(0.f);  // a_t D_t of the step behind the round
  if (p.on) {
    if (LOGITS)
      rate = map_([&](float d) { return -rate_of(scale, d); }, Elem<float, V>::load(decay + p.c));
    if (dhT) R = Elem<float, V>::load(dhT + p.b * C + p.c);
  }
  auto rows_of = [&](int64_t t) { return t >= 0 && t < L ? (int)(L - t < N ? L - t : N) : 0; };
  int64_t t_fetch = t0;
  auto fetch = [&](int stage) {
    const int n = rows_of(t_fetch);  // 0 behind the end and in front of the first round
    in_x.fetch(ring.x[stage][w], n);
    in_d.fetch(ring.d[stage][w], n);
    in_g.fetch(ring.g[stage][w], n);
    in_b.fetch(ring.b[stage][w], n);
    t_fetch -= per_round;
    copy_commit();
  };
#pragma unroll
  for (int k = 0; k < kStages - 1; ++k) fetch(k);
  int64_t o0 = (p.b * L + t0) * C + p.c0;  // of the slab in the warp's first row
  const float* from = ckpt + (p.b * tiles + (rounds - 1) * p.size + p.rank) * C + p.c;
  for (int64_t k = 0; k < rounds; ++k, t0 -= per_round, o0 -= per_round * C, from -= p.size * C) {
    const int n = rows_of(t0), s = (int)(k % kStages), parity = (int)(k & 1);
    F hv = all_<F>(0.f);  // the state in front of the tile
    if (p.on && t0 - w * N < L) hv = Elem<float, V>::load(from);
    fetch((int)((k + kStages - 1) % kStages));
    const uint32_t rs = RESET ? reset_bits(reset, t0, n) : 0;
    copy_wait<kStages - 1>();
    if (n < N) {  // behind the end nothing comes in
      __syncwarp();
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (i >= n) {
          EX::zero(&ring.x[s][w][(i * 32 + lane) * EX::kBytes]);
          EX::zero(&ring.d[s][w][(i * 32 + lane) * EX::kBytes]);
          EG::zero(&ring.g[s][w][(i * 32 + lane) * EG::kBytes]);
          EG::zero(&ring.b[s][w][(i * 32 + lane) * EG::kBytes]);
        }
    }
    __syncwarp();
    auto x_of = [&](int i) { return EX::load(&ring.x[s][w][(i * 32 + lane) * EX::kBytes]); };
    auto d_of = [&](int i) { return EX::load(&ring.d[s][w][(i * 32 + lane) * EX::kBytes]); };
    auto beta_of = [&](int i) { return EG::load(&ring.b[s][w][(i * 32 + lane) * EG::kBytes]); };
    F a[N], u[N], c[N];  // u = log a and c = 1 - sigmoid(g) of logits
    F A = all_<F>(1.f), H = all_<F>(0.f), Q = all_<F>(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const F gv = EG::load(&ring.g[s][w][(i * 32 + lane) * EG::kBytes]);
      F b;
      if (LOGITS) {
        F sg, si, ci;
        sigmoid_pair(gv, sg, c[i]);
        sigmoid_pair(beta_of(i), si, ci);
        u[i] = mul_(rate, sg);
        a[i] = map_(ex2, mul_(u[i], all_<F>(kLog2e)));
        // 1 - a^2, kept off 0: a == 1 leaves its limits, m = 0 and (a^2 / m) u = 0, to 1e-18
        const F v = map_([](float t) { return fmaxf(t, 1e-36f); },
                         one_minus_square(mul_(u[i], all_<F>(-2.f)), a[i]));
        const F rv = map_(rsqrt_, v);
        F m = mul_(v, rv);
        if (RESET && (rs >> i & 1)) m = all_<F>(1.f);
        const F mi = mul_(m, si);
        ring.q[w][i][lane] = mul_(mul_(a[i], a[i]), mul_(rv, rv));
        ring.mi[w][i][lane] = mi;
        ring.put_gates(s, w, i, lane, ci);
        b = mul_(mi, x_of(i));
      } else {
        a[i] = gv;
        b = mul_(beta_of(i), x_of(i));
      }
      if (RESET && (rs >> i & 1)) {
        a[i] = all_<F>(0.f);
        H = all_<F>(0.f);
      }
      if (i >= n) a[i] = all_<F>(1.f);  // behind the end: the state passes
      A = mul_(A, a[i]);
      H = fma_(a[i], H, b);
    }
#pragma unroll
    for (int i = N - 1; i >= 0; --i) {  // Q: D of step i, without what enters
      if (i + 1 < N) Q = RESET && (rs >> (i + 1) & 1) ? d_of(i) : fma_(a[i + 1], Q, d_of(i));
      else Q = d_of(i);
    }
    A = finite<RESET>(A);
    Q = RESET && (rs & 1) ? all_<F>(0.f) : mul_(a[0], Q);
    F d = R;  // a_t D_t of the step behind the warp's
    if constexpr (CTAS > 1) {
      link.A[parity][w][lane] = A;
      link.H[parity][w][lane] = Q;
      link_h[parity][w][lane] = H;
      __syncthreads();
      d = carry_in<true, RESET>(link, k, w, R);
#pragma unroll 4
      for (int q = 0; q < WARPS - 1; ++q)
        if (q < w) hv = through<RESET>(hv, link.A[parity][q][lane], link_h[parity][q][lane]);
    } else {
      auto from_front = [&] {
        if (w > 0) hv = link_h.get(k, w - 1);
        if (w + 1 < WARPS) link_h.put(k, w, through<RESET>(hv, A, H));
      };
      auto from_behind = [&] {
        if (k > 0 || w + 1 < WARPS) d = link.get(w + 1 < WARPS ? k : k - 1, w + 1 < WARPS ? w + 1 : 0);
        R = through<RESET>(d, A, Q);
        link.put(k, w, R);
      };
      // the end of the tile that is nearer comes first
      if (w < WARPS / 2) from_front();
      from_behind();
      if (w >= WARPS / 2) from_front();
    }
    if (p.on) {
      F D[N];
#pragma unroll
      for (int i = N - 1; i >= 0; --i) {
        if (i + 1 == N) d = add_(d, d_of(i));
        else d = RESET && (rs >> (i + 1) & 1) ? d_of(i) : fma_(a[i + 1], d, d_of(i));
        D[i] = d;
      }
      auto walk = [&](auto full) {
        int64_t o = o0 + lane * V;
#pragma unroll
        for (int i = 0; i < N; ++i, o += C) {
          const bool zero = RESET && (rs >> i & 1);
          const F xv = x_of(i);
          F ox, og, ob, b;
          if (LOGITS) {
            const F mi = ring.mi[w][i][lane], ci = ring.get_gates(s, w, i, lane);
            b = mul_(mi, xv);
            F du = mul_(D[i], fma_(a[i], hv, mul_(mul_(ring.q[w][i][lane], b), all_<F>(-1.f))));
            du = mul_(du, u[i]);
            if (zero) du = all_<F>(0.f);  // whatever u is
            if (full || i < n) sum = add_(sum, du);
            og = mul_(du, c[i]);
            ox = mul_(D[i], mi);
            ob = mul_(mul_(D[i], b), ci);
          } else {
            const F be = beta_of(i);
            b = mul_(be, xv);
            ox = mul_(D[i], be);
            ob = mul_(D[i], xv);
            og = zero ? all_<F>(0.f) : mul_(D[i], hv);
          }
          if (zero) hv = all_<F>(0.f);
          hv = fma_(a[i], hv, b);
          if (full || i < n) {
            EX::store(dx + o, ox);
            EG::store(dg + o, og);
            EG::store(dbeta + o, ob);
          }
        }
      };
      if (n == N) walk(std::true_type{});
      else walk(std::false_type{});
    }
    __syncwarp();
  }
  copy_wait<0>();
  if (dh0 && p.on && p.rank == 0 && w == 0) Elem<float, V>::store(dh0 + p.b * C + p.c, R);
  if (LOGITS && ddecay_part) {
    auto& sums = ring.mi;  // of no use any more
    __syncthreads();
    sums[w][0][lane] = sum;
    __syncthreads();
    if (w == 0 && p.on) {
      F t = sums[0][0][lane];
#pragma unroll
      for (int k = 1; k < WARPS; ++k) t = add_(t, sums[k][0][lane]);
      Elem<float, V>::store(ddecay_part + (p.b * p.size + p.rank) * C + p.c, t);
    }
  }
  if constexpr (CTAS > 1) cluster_meet();  // none leaves while another may send to it
}

// ddecay[c] = sigmoid(decay) / softplus(decay) * the sum of the partial rows of du u, in their
// order: u = rate s and rate = -scale softplus, so -scale sigmoid(decay) du s is that.  The
// quotient goes to 1 where softplus leaves the fp32 range.
__global__ void __launch_bounds__(128)
glr_ddecay_kernel(const float* __restrict__ part, int64_t rows, const float* __restrict__ decay,
                  float* __restrict__ ddecay, int64_t C) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= C) return;
  float t = 0.f;
  for (int64_t r = 0; r < rows; ++r) t += part[r * C + c];
  float s, cs;
  sigmoid2(decay[c], s, cs);
  const float sp = softplus(decay[c]);
  ddecay[c] = t * (sp > 1e-30f ? s / sp : 1.f);
}

// ---------------------------------------------------------------------------
// One step
// ---------------------------------------------------------------------------
template <typename T, typename G, bool LOGITS>
__global__ void __launch_bounds__(128)
glr_step_kernel(const T* __restrict__ x, const G* __restrict__ g, const G* __restrict__ beta,
                const float* __restrict__ decay, float* __restrict__ state, T* __restrict__ h,
                int64_t B, int64_t C, Strides st, float scale) {
  const int64_t c = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= C) return;
  const float rate = LOGITS ? -rate_of(scale, decay[c]) : 0.f;
  for (int64_t b = blockIdx.y; b < B; b += gridDim.y) {
    float a = to_f<G>(g[b * st.gb + c]), in = to_f<G>(beta[b * st.bb + c]);
    if (LOGITS) {
      float s, i, unused;
      sigmoid2(a, s, unused);
      sigmoid2(in, i, unused);
      const float u = rate * s;
      a = ex2(u * kLog2e);
      in = sqrt_(one_minus_square(-2.f * u, a)) * i;
    }
    const float s = fmaf(a, state[b * C + c], in * to_f<T>(x[b * st.xb + c]));
    state[b * C + c] = s;
    h[b * C + c] = from_f<T>(s);
  }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
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

// Calls f with three truth values as constants.
template <typename F> int with_flags(bool two, bool logits, bool reset, F&& f) {
  auto b = [](bool v, auto&& k) {
    return v ? k(std::true_type{}) : k(std::false_type{});
  };
  return b(two, [&](auto t) {
    return b(logits, [&](auto l) { return b(reset, [&](auto r) { return f(t, l, r); }); });
  });
}

int check_sizes(const char* what, int64_t B, int64_t L, int64_t C) {
  FO_CHECK_ARG(B >= 0 && L >= 0 && C >= 0, "%s: negative size B=%lld L=%lld C=%lld", what,
               (long long)B, (long long)L, (long long)C);
  FO_CHECK_ARG(C == 0 || B <= ((int64_t)1 << 31) / 8 / ((C + 31) / 32),
               "%s: B=%lld sequences of %lld channels are over the grid's limit", what,
               (long long)B, (long long)C);
  return FO_OK;
}

bool multiple(const void* p, int64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

// Two channels a lane (packed arithmetic, 128-byte rows of a warp), for 16-bit gates and where
// pairs start at a multiple of their size everywhere.  fp32 rows of a warp are 128 bytes as they
// are, and pairs of them would leave room for one CTA on an SM instead of two.
bool pairs_ok(const void* const* xs, int nx, const void* const* gs, int ng, const void* const* fs,
              int nf, const int64_t* strides, int64_t C, int xbytes, int gbytes) {
  bool ok = gbytes == 2 && C % 2 == 0;
  for (int i = 0; i < nx; ++i) ok = ok && multiple(xs[i], 2 * xbytes);
  for (int i = 0; i < ng; ++i) ok = ok && multiple(gs[i], 2 * gbytes);
  for (int i = 0; i < nf; ++i) ok = ok && multiple(fs[i], 8);
  for (int i = 0; i < 6; ++i) ok = ok && strides[i] % 2 == 0;
  return ok;
}

// 16-byte copies: rows have to start at, and be, multiples of 16 bytes.
bool wide_ok(const void* const* xs, int nx, const void* const* gs, int ng, const int64_t* strides,
             int64_t C, int xbytes, int gbytes) {
  const int px = 16 / xbytes, pg = 16 / gbytes, least = px < pg ? pg : px;
  bool ok = C % least == 0;
  for (int i = 0; i < nx; ++i) ok = ok && multiple(xs[i], 16);
  for (int i = 0; i < ng; ++i) ok = ok && multiple(gs[i], 16);
  for (int i = 0; i < 6; ++i) ok = ok && strides[i] % least == 0;
  return ok;
}

// CTAs of a cluster along time: doubled, up to `most` and up to the number of tiles, until there
// are `want` CTAs.
int cluster_for(int64_t ctas, int64_t tiles, int64_t want, int most) {
  int n = 1;
  while (n < most && ctas * n < want && 2 * n <= tiles) n *= 2;
  return n;
}

template <typename K, typename... Args>
int launch(const char* what, K kernel, int64_t ctas, int cluster, int threads, int smem, cudaStream_t st,
           Args... args) {
  cudaError_t e = allow_shared((const void*)kernel, smem);
  if (e == cudaSuccess) {
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
    cfg.numAttrs = cluster > 1 ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, args...);
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    set_error("%s: %s", what, cudaGetErrorString(e));
    return FO_ECUDA;
  }
  return check_launch(what);
}

constexpr int64_t kZeroStrides[6] = {};

int64_t slabs_of(int64_t C, int v) { return (C + 32 * v - 1) / (32 * v); }

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
  const int64_t* q = strides ? strides : kZeroStrides;
  const Strides s{q[0], q[1], q[2], q[3], q[4], q[5]};
  return with_types(dtype, gate_dtype, [&](auto t, auto gt) {
    using T = decltype(t);
    using G = decltype(gt);
    const void *xs[] = {x, h}, *gs[] = {g, beta}, *fs[] = {decay, h0, hT, ckpt};
    const bool two = pairs_ok(xs, 2, gs, 2, fs, 4, q, C, sizeof(T), sizeof(G));
    const bool wide = wide_ok(xs, 1, gs, 2, q, C, sizeof(T), sizeof(G));
    const int64_t ctas = B * slabs_of(C, two ? 2 : 1);
    // CTAs of a cluster until every SM has one: 242 us without, 292 with two at 8 x 8192 x 2048 bf16, where
    // there are 256 CTAs as it is; 242 and 228 with 160 or 192 CTAs (batches of 5 and 6).  (One comparison.)
    const int cl = cluster_for(ctas, (L + kFwdTile - 1) / kFwdTile, num_sms(), kMostCtas);
    return with_flags(two, decay, reset, [&](auto tw, auto lo, auto rs) {
      constexpr int V = tw && sizeof(G) == 2 ? 2 : 1;
      auto run = [&](auto kernel) {
        return launch("glr_fwd_kernel", kernel, ctas, cl, 32 * kFwdWarps,
                      (int)sizeof(FwdRing<T, G, V>), as_stream(stream), (const T*)x, (const G*)g,
                      (const G*)beta, decay, h0, reset, (T*)h, hT, ckpt, L, C, s, scale, wide);
      };
      return cl > 1 ? run(glr_fwd_kernel<T, G, V, lo, rs, kMostCtas>)
                    : run(glr_fwd_kernel<T, G, V, lo, rs, 1>);
    });
  });
}

extern "C" int fo_glr_step(const void* x, const void* g, const void* beta, const float* decay,
                           float* state, void* h, int64_t B, int64_t C, const int64_t* strides,
                           float scale, int dtype, int gate_dtype, void* stream) {
  clear_error();
  if (int rc = check_sizes("gated recurrence step", B, 1, C)) return rc;
  if (B == 0 || C == 0) return FO_OK;
  FO_CHECK_ARG(x && g && beta && state && h && strides, "gated recurrence step: null pointer");
  const Strides s{strides[0], 0, strides[1], 0, strides[2], 0};
  return with_types(dtype, gate_dtype, [&](auto t, auto gt) {
    using T = decltype(t);
    using G = decltype(gt);
    auto run = [&](auto k) {
      k<<<dim3((unsigned)((C + 127) / 128), (unsigned)(B < 65535 ? B : 65535)), 128, 0,
          as_stream(stream)>>>((const T*)x, (const G*)g, (const G*)beta, decay, state, (T*)h, B, C,
                               s, scale);
      return check_launch("glr_step_kernel");
    };
    return decay ? run(glr_step_kernel<T, G, true>) : run(glr_step_kernel<T, G, false>);
  });
}

extern "C" int fo_glr_bwd_workspace_bytes(int64_t B, int64_t L, int64_t C, int64_t* bytes) {
  clear_error();
  FO_CHECK_ARG(bytes, "gated recurrence backward: null pointer");
  if (int rc = check_sizes("gated recurrence backward", B, L, C)) return rc;
  *bytes = B * 8 * C * 4;
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
  FO_CHECK_ARG(!need || multiple(workspace, 8),
               "gated recurrence backward: workspace must be 8-byte aligned");
  const int64_t* sq = strides ? strides : kZeroStrides;
  const Strides s{sq[0], sq[1], sq[2], sq[3], sq[4], sq[5]};
  float* part = ddecay ? (float*)workspace : nullptr;
  int cl = 1;
  return with_types(dtype, gate_dtype, [&](auto t, auto gt) {
    using T = decltype(t);
    using G = decltype(gt);
    const void *xs[] = {x, dh, dx}, *gs[] = {g, beta, dg, dbeta}, *fs[] = {decay, ckpt, dhT, dh0};
    const bool two = pairs_ok(xs, 3, gs, 4, fs, 4, sq, C, sizeof(T), sizeof(G));
    const bool wide = wide_ok(xs, 2, gs, 2, sq, C, sizeof(T), sizeof(G));
    const int64_t ctas = B * slabs_of(C, two ? 2 : 1);
    // Clusters of 8 leave room for one CTA on an SM instead of two, so they are for few CTAs: 372 us
    // with 4, 202 with 8 at 1 x 32768 x 512 bf16 (8 slabs), 56 and 88 us at 2 x 4096 x 1024 (32).
    const int most = ctas * kMostCtas <= num_sms() ? kMostCtas : 4;
    cl = cluster_for(ctas, (L + kBwdTile - 1) / kBwdTile, num_sms(), most);
    int rc = with_flags(two, decay, reset, [&](auto tw, auto lo, auto rs) {
      constexpr int V = tw && sizeof(G) == 2 ? 2 : 1;
      auto run = [&](auto kernel) {
        return launch("glr_bwd_kernel", kernel, ctas, cl, 32 * kBwdWarps,
                      (int)sizeof(BwdRing<T, G, V>), q, (const T*)x, (const G*)g, (const G*)beta,
                      decay, reset, ckpt, (const T*)dh, dhT, (T*)dx, (G*)dg, (G*)dbeta, dh0, part,
                      L, C, s, scale, wide);
      };
      return cl > 4   ? run(glr_bwd_kernel<T, G, V, lo, rs, 8>)
             : cl > 1 ? run(glr_bwd_kernel<T, G, V, lo, rs, 4>)
                      : run(glr_bwd_kernel<T, G, V, lo, rs, 1>);
    });
    if (rc || !ddecay) return rc;
    glr_ddecay_kernel<<<(unsigned)((C + 127) / 128), 128, 0, q>>>(part, B * cl, decay, ddecay, C);
    return check_launch("glr_ddecay_kernel");
  });
}

extern "C" int fo_glr_timeouts(unsigned int* count) {
  clear_error();
  FO_CHECK_ARG(count, "fo_glr_timeouts: null pointer");
  if (cudaMemcpyFromSymbol(count, g_glr_timeouts, sizeof(unsigned int)) != cudaSuccess)
    return check_launch("fo_glr_timeouts");
  return FO_OK;
}
