// Embedding lookup with a scale, and its gradient, for sm_100a.
//
//   out[t] = scale * W[ids[t]],   dW[v] = scale * sum of dout[t] over the t with ids[t] == v
//
// Both are bound by memory: the lookup reads and writes T rows, the gradient reads T rows and
// writes V.  Sums are in fp32 and in a fixed order, so the gradient is the same in every run.
//
// Gradient:
//  1. emb_sort_kernel: the tokens are cut into chunks of kChunk, and a CTA sorts the positions of
//     a chunk by id in shared memory (stable, 9 bits of the id a pass).  Ids that do not count
//     get the key V.  No chunk waits for another.
//  2. emb_merge_kernel (more than one chunk): a token's place in the order of all chunks is its
//     place in its own plus the numbers of smaller keys in the others, found by bisection: T^2 / kChunk
//     bisections, where all else is linear in T.
//  3. emb_piece_kernel: a CTA adds up 32 consecutive sorted tokens, whatever their ids: each row of
//     dout is read once, and an id with many tokens (padding, frequent words) costs no CTA more
//     than 32.  Rows of dW whose tokens all lie in the piece are written, the sums of the ids
//     that go on across its ends are kept in fp32.
//  4. emb_join_kernel: adds those up, from piece to piece (emb_run_kernel before it adds up
//     runs of 16 pieces of one id, so that no chain is long).
// Most rows of dW have no token and are zeros: spare CTAs of the kernels 1 and 2, which leave the
// memory idle, write all of dW as zeros meanwhile.
//
// Measured (B200, 16384 tokens distributed as words, 128256 x 4096 bf16): lookup 30 us (268 MB less
// what repeats); gradient 127 us sort (with 788 MB of zeros), 48 us merge (with 262 MB), 33 us
// pieces, 4 us runs, 11 us join, which is 1.25 GB at 5.6 TB/s.  Finding each row's tokens in the
// kernel that writes dW was slower (241 us for that kernel alone: its CTAs wait for bounds,
// positions and rows one after the other).  30011 tokens, a third of them one id, 5003 x 771 fp32:
// 27 us and 74 us; there the bisections and the unaligned rows' 4-byte accesses count.  Gradients of
// 32000 x 1024 bf16: 53 us with 16384 tokens, 97 with 65536, 162 with 131072, 326 with 262144, of
// which the merge is more than half, and 2.4 ms with 1048576, of which it is 1.9.
#include <type_traits>

#include "common.cuh"

namespace fo {
namespace {

constexpr int kThreads = 256;

// 16 bytes of a row, or one element where rows are not 16-byte aligned
template <typename T, bool WIDE> struct Vec {
  static constexpr int E = WIDE ? Vec16<T>::E : 1;
  using Raw = std::conditional_t<WIDE, uint4, T>;
  static __device__ __forceinline__ Raw load(const T* p) {
    if constexpr (WIDE) return ld_global_nc_v4(p);
    else return *p;
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float* f) {
    if constexpr (WIDE) unpack16<T>(r, f);
    else f[0] = to_f<T>(r);
  }
  // E floats of an fp32 row of sums
  static __device__ __forceinline__ void add_sums(const float* p, float* f) {
    if constexpr (WIDE) {
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        const float4 v = *reinterpret_cast<const float4*>(p + e);
        f[e] += v.x;
        f[e + 1] += v.y;
        f[e + 2] += v.z;
        f[e + 3] += v.w;
      }
    } else {
      f[0] += *p;
    }
  }
  static __device__ __forceinline__ void store_sums(float* p, const float* f) {
    if constexpr (WIDE) {
#pragma unroll
      for (int e = 0; e < E; e += 4)
        *reinterpret_cast<float4*>(p + e) = make_float4(f[e], f[e + 1], f[e + 2], f[e + 3]);
    } else {
      *p = f[0];
    }
  }
  static __device__ __forceinline__ void store(T* p, const float* f) {
    if constexpr (WIDE) st_global_stream_v4(p, pack16<T>(f));
    else *p = from_f<T>(f[0]);
  }
};

// ---------------------------------------------------------------------------
// Lookup: a CTA copies ROWS rows (or a slab of them); all of a thread's loads, which wait for the
// ids, come before its stores.
// ---------------------------------------------------------------------------
template <typename T, typename I, bool WIDE, int ROWS>
__global__ void __launch_bounds__(kThreads)
emb_fwd_kernel(const I* __restrict__ ids, const T* __restrict__ w, T* __restrict__ out, int64_t T_,
               int64_t V, int64_t N, int64_t ld, float scale, unsigned slabs) {
  using X = Vec<T, WIDE>;
  constexpr int K = WIDE ? 2 : 4;  // vectors of a thread in a row
  const int64_t t0 = (int64_t)(blockIdx.x / slabs) * ROWS;
  const int v0 = (int)(blockIdx.x % slabs) * (int)blockDim.x * K + threadIdx.x;
  const int left = (int)(N / X::E) - v0;  // vectors from the thread's first on
  if (left <= 0) return;
  // Offsets in W of the thread's first vector.  An id outside [0, V) is replaced before any address
  // is made from it.
  bool inside[ROWS];
  int64_t from[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int64_t id = t0 + r < T_ ? (int64_t)ids[t0 + r] : -1;
    inside[r] = id >= 0 && id < V;
    from[r] = (inside[r] ? id : 0) * ld + (int64_t)v0 * X::E;
  }
  typename X::Raw raw[ROWS][K];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (inside[r] && k * (int)blockDim.x < left)
        raw[r][k] = X::load(w + from[r] + k * (int)blockDim.x * X::E);
  T* to = out + t0 * N + (int64_t)v0 * X::E;
#pragma unroll
  for (int r = 0; r < ROWS; ++r, to += N) {
    if (t0 + r >= T_) break;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k * (int)blockDim.x < left) {
        float f[X::E] = {};
        if (inside[r]) {
          X::unpack(raw[r][k], f);
#pragma unroll
          for (int e = 0; e < X::E; ++e) f[e] *= scale;
        }
        X::store(to + k * (int)blockDim.x * X::E, f);
      }
  }
}

// A part of dW to be written as zeros by the CTAs of a kernel from `first_cta` on.
struct Zeros {
  uint8_t* p;
  int64_t bytes;
  unsigned first_cta;
};
__device__ __forceinline__ void write_zeros(const Zeros& z) {
  const int64_t n = (int64_t)(gridDim.x - z.first_cta) * blockDim.x;
  const int64_t me = (int64_t)(blockIdx.x - z.first_cta) * blockDim.x + threadIdx.x;
  // dW begins at a multiple of its element size; the middle is written in 16-byte words
  int64_t head = (int64_t)(-reinterpret_cast<intptr_t>(z.p) & 15);
  if (head > z.bytes) head = z.bytes;
  const int64_t words = (z.bytes - head) / 16, tail = head + words * 16;
  for (int64_t i = 2 * me; i < head; i += 2 * n) *reinterpret_cast<uint16_t*>(z.p + i) = 0;
  uint4* w = reinterpret_cast<uint4*>(z.p + head);
  for (int64_t i = me; i < words; i += n) st_global_stream_v4(w + i, make_uint4(0, 0, 0, 0));
  for (int64_t i = tail + 2 * me; i < z.bytes; i += 2 * n) *reinterpret_cast<uint16_t*>(z.p + i) = 0;
}

// ---------------------------------------------------------------------------
// 1. Sort
// ---------------------------------------------------------------------------
constexpr int kChunk = 4096;
constexpr int kSortThreads = 512;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kItems = kChunk / kSortThreads;
constexpr int kBits = 9, kBins = 1 << kBits;

struct SortSmem {
  int32_t key[kChunk];
  uint16_t pos[2][kChunk];
  uint16_t count[kSortWarps][kBins];
  int32_t warp_total[kSortWarps];
};

// Sorted keys and token positions of each chunk.  A warp owns consecutive items, so that ranks by
// (digit, warp, order within the warp) keep equal digits in order.
template <typename I>
__global__ void __launch_bounds__(kSortThreads)
emb_sort_kernel(const I* __restrict__ ids, int32_t* __restrict__ skey, int32_t* __restrict__ spos,
                int64_t T, int64_t V, int64_t padding_idx, int passes, Zeros zeros) {
  if (blockIdx.x >= zeros.first_cta) return write_zeros(zeros);
  extern __shared__ __align__(16) uint8_t raw[];
  SortSmem& s = *reinterpret_cast<SortSmem*>(raw);
  const int64_t base = (int64_t)blockIdx.x * kChunk;
  const int n = (int)(T - base < kChunk ? T - base : kChunk);
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  for (int i = tid; i < n; i += kSortThreads) {
    const int64_t id = ids[base + i];
    s.key[i] = (int32_t)(id >= 0 && id < V && id != padding_idx ? id : V);
    s.pos[0][i] = (uint16_t)i;
  }
  const int per = (n + kSortThreads - 1) / kSortThreads;  // items of a thread, 32 apart
  for (int pass = 0; pass < passes; ++pass) {
    const uint16_t* from = s.pos[pass & 1];
    uint16_t* to = s.pos[(pass & 1) ^ 1];
    for (int i = tid; i < kSortWarps * kBins / 2; i += kSortThreads)
      reinterpret_cast<uint32_t*>(s.count)[i] = 0;
    __syncthreads();
    uint16_t item[kItems];
    int rank[kItems], digit[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      digit[k] = kBins;
      if (k >= per) continue;
      const int i = (w * per + k) * 32 + lane;
      const bool on = i < n;
      item[k] = on ? from[i] : 0;
      digit[k] = on ? (s.key[item[k]] >> (pass * kBits)) & (kBins - 1) : kBins;
      unsigned peers = 0xffffffffu;  // lanes of the same digit, bit by bit
#pragma unroll
      for (int bit = 0; bit <= kBits; ++bit) {
        const int mine = (int)((unsigned)digit[k] << (31 - bit)) >> 31;  // all ones or zeros
        peers &= ~(__ballot_sync(0xffffffffu, mine) ^ mine);
      }
      const int before = __popc(peers & ((1u << lane) - 1));
      int first = 0;
      if (on) first = s.count[w][digit[k]];
      rank[k] = first + before;
      __syncwarp();
      if (on && before == 0) s.count[w][digit[k]] = (uint16_t)(first + __popc(peers));
      __syncwarp();
    }
    __syncthreads();
    // exclusive offsets by (digit, warp): thread d has digit d
    int total = 0;
    if (tid < kBins)
      for (int k = 0; k < kSortWarps; ++k) total += s.count[k][tid];
    int up = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, up, o);
      if (lane >= o) up += v;
    }
    if (lane == 31) s.warp_total[w] = up;
    __syncthreads();
    if (tid < kBins) {
      int at = up - total;
      for (int k = 0; k < w; ++k) at += s.warp_total[k];
      for (int k = 0; k < kSortWarps; ++k) {
        const int c = s.count[k][tid];
        s.count[k][tid] = (uint16_t)at;
        at += c;
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      if (digit[k] < kBins) to[s.count[w][digit[k]] + rank[k]] = item[k];
    __syncthreads();
  }
  if (passes == 0) __syncthreads();
  const uint16_t* sorted = s.pos[passes & 1];
  for (int i = tid; i < n; i += kSortThreads) {
    skey[base + i] = s.key[sorted[i]];
    spos[base + i] = (int32_t)(base + sorted[i]);
  }
}

// ---------------------------------------------------------------------------
// 2. Merge
// ---------------------------------------------------------------------------
// key and pos: the tokens of all chunks in one stable order.  Eight bisections at a time, whose
// loads do not wait for one another.
__global__ void __launch_bounds__(kThreads)
emb_merge_kernel(const int32_t* __restrict__ skey, const int32_t* __restrict__ spos,
                 int32_t* __restrict__ key, int32_t* __restrict__ pos, int T, int chunks,
                 Zeros zeros) {
  if (blockIdx.x >= zeros.first_cta) return write_zeros(zeros);
  constexpr int kAtOnce = 8;
  // every kCoarse-th key of eight chunks, for the first half of their bisections
  constexpr int kCoarse = 64, kMarks = kChunk / kCoarse;
  __shared__ int32_t marks[kAtOnce][kMarks];
  const int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int t = (int)(i < T ? i : T - 1), mine = t / kChunk;
  const int32_t k = skey[t];
  int to = t - mine * kChunk;
  for (int c0 = 0; c0 < chunks; c0 += kAtOnce) {
    __syncthreads();
    for (int m = threadIdx.x; m < kAtOnce * kMarks; m += kThreads) {
      const int64_t at = (int64_t)(c0 + m / kMarks) * kChunk + m % kMarks * kCoarse;
      marks[m / kMarks][m % kMarks] = at < T ? skey[at] : INT32_MAX;
    }
    __syncthreads();
    int below[kAtOnce];
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) below[q] = 0;
#pragma unroll 1
    for (int s = kMarks; s > 0; s >>= 1)
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int j = below[q] + s - 1;
        if (j < kMarks && marks[q][j] < k + (c0 + q < mine)) below[q] += s;
      }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q) below[q] = below[q] ? (below[q] - 1) * kCoarse + 1 : 0;
#pragma unroll 1
    for (int s = kCoarse / 2; s > 0; s >>= 1)
#pragma unroll
      for (int q = 0; q < kAtOnce; ++q) {
        const int c = c0 + q, j = below[q] + s - 1;
        // equal keys of earlier chunks are in front
        if (c < chunks && c != mine && j < kChunk && j < T - c * kChunk &&
            skey[c * kChunk + j] < k + (c < mine))
          below[q] += s;
      }
#pragma unroll
    for (int q = 0; q < kAtOnce; ++q)
      if (c0 + q < chunks && c0 + q != mine) to += below[q];
  }
  if (i < T) {
    key[to] = k;
    pos[to] = spos[t];
  }
}

// ---------------------------------------------------------------------------
// 3. and 4. Sums
// ---------------------------------------------------------------------------
constexpr int kPiece = 32;   // sorted tokens of a piece
constexpr int kRun = 16;     // pieces of a run

// A thread's columns of a row: one vector, or four elements blockDim.x apart.
template <typename T, bool WIDE> struct Columns {
  using X = Vec<T, WIDE>;
  static constexpr int K = WIDE ? 1 : 4, E = X::E;
  int first, step, left;  // in vectors; left: from the first on
  float acc[K][E];
  __device__ __forceinline__ Columns(int64_t N, unsigned slab)
      : first((int)slab * (int)blockDim.x * K + (int)threadIdx.x), step((int)blockDim.x),
        left((int)(N / E) - first) {
    clear();
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int e = 0; e < E; ++e) acc[k][e] = 0.f;
  }
  __device__ __forceinline__ bool on(int k) const { return k * step < left; }
  __device__ __forceinline__ int at(int k) const { return (first + k * step) * E; }
  __device__ __forceinline__ void write(T* row, float scale) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (on(k)) {
#pragma unroll
        for (int e = 0; e < E; ++e) acc[k][e] *= scale;
        X::store(row + at(k), acc[k]);
      }
  }
  __device__ __forceinline__ void keep(float* row) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (on(k)) X::store_sums(row + at(k), acc[k]);
  }
};

// Sums kept of piece p: row 2 p of the id that is in front of the piece too, row 2 p + 1 of an
// id that begins in the piece and goes on behind it.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
emb_piece_kernel(const T* __restrict__ dout, const int32_t* __restrict__ key,
                 const int32_t* __restrict__ pos, float* __restrict__ part, T* __restrict__ dw,
                 int T_, int64_t V, int64_t N, float scale, unsigned slabs) {
  using X = Vec<T, WIDE>;
  using Cols = Columns<T, WIDE>;
  constexpr int kUnroll = WIDE ? 8 : 4;  // rows in flight a thread
  __shared__ int32_t pos_s[kPiece], key_s[kPiece + 2];  // keys from the one in front on
  const int64_t p = blockIdx.x / slabs;
  const int i0 = (int)(p * kPiece), n = T_ - i0 < kPiece ? T_ - i0 : kPiece;
  for (int k = threadIdx.x; k < n; k += blockDim.x) pos_s[k] = pos[i0 + k];
  for (int k = threadIdx.x; k < n + 2; k += blockDim.x) {
    const int i = i0 + k - 1;
    key_s[k] = i >= 0 && i < T_ ? key[i] : -1;
  }
  __syncthreads();
  if (key_s[1] >= V) return;  // what does not count is behind everything
  Cols c(N, blockIdx.x % slabs);
  if (!c.on(0)) return;
  bool front = key_s[0] == key_s[1];  // the running sum began in front of the piece
  for (int u0 = 0; u0 < n; u0 += kUnroll) {
    typename X::Raw r[kUnroll][Cols::K];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (u0 + u < n && key_s[u0 + u + 1] < V) {
        const T* row = dout + pos_s[u0 + u] * N;
#pragma unroll
        for (int k = 0; k < Cols::K; ++k)
          if (c.on(k)) r[u][k] = X::load(row + c.at(k));
      }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = u0 + u;
      if (i >= n) break;
      const int32_t me = key_s[i + 1];
      if (me >= V) return;
#pragma unroll
      for (int k = 0; k < Cols::K; ++k)
        if (c.on(k)) {
          float f[X::E];
          X::unpack(r[u][k], f);
#pragma unroll
          for (int e = 0; e < X::E; ++e) c.acc[k][e] += f[e];
        }
      const bool last = i + 1 == n;
      if (key_s[i + 2] != me || last) {
        if (front) c.keep(part + 2 * p * N);
        else if (key_s[i + 2] != me) c.write(dw + me * N, scale);
        else c.keep(part + (2 * p + 1) * N);
        c.clear();
        front = false;
      }
    }
  }
}

// Sums of kRun consecutive pieces that hold one id only and do not begin it, a column a thread.
__global__ void __launch_bounds__(kThreads)
emb_run_kernel(const int32_t* __restrict__ key, const float* __restrict__ part,
               float* __restrict__ runs, int64_t V, int64_t N, unsigned slabs) {
  const int64_t j = blockIdx.x / slabs, i = j * kPiece * kRun;
  const int64_t col = (int64_t)(blockIdx.x % slabs) * kThreads + threadIdx.x;
  const int32_t k = key[i];
  if (k >= V || i == 0 || key[i - 1] != k || key[i + kPiece * kRun - 1] != k || col >= N) return;
  float acc = 0.f;
#pragma unroll 16
  for (int b = 0; b < kRun; ++b) acc += part[2 * (j * kRun + b) * N + col];
  runs[j * N + col] = acc;
}

// The id that begins in piece p and goes on: its sums in the pieces, from p on.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
emb_join_kernel(const int32_t* __restrict__ key, const float* __restrict__ part,
                const float* __restrict__ runs, T* __restrict__ dw, int T_, int64_t V, int64_t N,
                float scale, unsigned slabs) {
  using X = Vec<T, WIDE>;
  using Cols = Columns<T, WIDE>;
  const int p = (int)(blockIdx.x / slabs), end = (p + 1) * kPiece;
  const int32_t me = key[end - 1];
  if (me >= V || end >= T_ || key[end] != me) return;  // nothing goes on
  if (key[end - kPiece] == me && p > 0 && key[end - kPiece - 1] == me) return;  // began earlier
  // The first sorted token behind it: every warp splits [lo, hi] in 32 until it is found.
  int lo = end, hi = T_;
  while (lo < hi) {
    const int step = (hi - lo + 31) / 32, at = lo + (int)(threadIdx.x & 31) * step;
    const unsigned more = __ballot_sync(0xffffffffu, at < hi && key[at] <= me);
    const int n = __popc(more);  // of the lanes' keys, that many are not behind it
    const int top = lo + n * step;
    if (n) lo = top - step + 1;
    if (top < hi) hi = top;
  }
  const int q1 = (lo - 1) / kPiece + 1;  // behind the last piece
  Cols c(N, blockIdx.x % slabs);
  if (!c.on(0)) return;
  auto add = [&](const float* row) {
#pragma unroll
    for (int k = 0; k < Cols::K; ++k)
      if (c.on(k)) X::add_sums(row + c.at(k), c.acc[k]);
  };
  add(part + (2 * (int64_t)p + 1) * N);
  // whole runs [r0, r1); the pieces in front of and behind them one by one
  const int q0 = p + 1, r0 = (q0 + kRun - 1) / kRun, full = lo / kPiece / kRun;
  const int r1 = full > r0 ? full : r0, a1 = r0 * kRun < q1 ? r0 * kRun : q1;
#pragma unroll 8
  for (int q = q0; q < a1; ++q) add(part + 2 * (int64_t)q * N);
#pragma unroll 8
  for (int r = r0; r < r1; ++r) add(runs + (int64_t)r * N);
#pragma unroll 8
  for (int q = r1 * kRun > a1 ? r1 * kRun : a1; q < q1; ++q) add(part + 2 * (int64_t)q * N);
  c.write(dw + me * N, scale);
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------
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
  const int64_t most = (int64_t)1 << 30;
  FO_CHECK_ARG(T <= most && V <= most && N <= most,
               "embedding: T=%lld, V=%lld and N=%lld must not be over 2^30", (long long)T,
               (long long)V, (long long)N);
  return FO_OK;
}

// CTAs of kThreads vectors (times per) that cover a row; 0 if rows * that leave the grid.
int64_t slabs_of(int64_t nv, int64_t rows, int64_t per) {
  const int64_t s = (nv + per - 1) / per;
  return rows > (((int64_t)1 << 31) - 1) / s ? 0 : s;
}

int grid_error() {
  set_error("embedding: too many rows of this width for one grid");
  return FO_EUNSUPPORTED;
}

// Offsets of the workspace's parts, and its size.  key and pos are the chunks' own where there is
// one chunk.
struct Workspace {
  int64_t spos, key, pos, part, runs, bytes;
};
Workspace workspace(int64_t T, int64_t N) {
  int64_t at = 0;
  auto take = [&](int64_t b) {
    const int64_t o = at;
    at += (b + 255) / 256 * 256;
    return o;
  };
  Workspace w;
  take(T * 4);  // the chunks' keys
  w.spos = take(T * 4);
  w.key = T > kChunk ? take(T * 4) : 0;
  w.pos = T > kChunk ? take(T * 4) : w.spos;
  w.part = T > kPiece ? take((T + kPiece - 1) / kPiece * 2 * N * 4) : 0;
  w.runs = T > kPiece ? take(T / (kPiece * kRun) * N * 4) : 0;
  w.bytes = at;
  return w;
}

// CTAs that write `bytes` of zeros: up to four an SM, 64 KB each at least.
unsigned zero_ctas(int64_t bytes) {
  const int64_t most = 4 * (int64_t)num_sms(), n = (bytes + 65535) / 65536;
  return (unsigned)(n < most ? n : most);
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
    // Four rows a CTA, where that leaves enough CTAs: 41 us with one, 37 with four for 30011 rows of
    // 771 fp32 elements.
    const bool four = T >= 16 * (int64_t)num_sms();
    auto run = [&](auto wide) {
      constexpr int K = wide ? 2 : 4;
      const int64_t nv = N / Vec<E, wide>::E, ctas = four ? (T + 3) / 4 : T;
      int threads = 32;  // a CTA no wider than the row
      while (threads < kThreads && threads * K < nv) threads *= 2;
      const int64_t slabs = slabs_of(nv, ctas, threads * K);
      if (!slabs) return grid_error();
      auto go = [&](auto kernel) {
        kernel<<<(unsigned)(ctas * slabs), threads, 0, as_stream(stream)>>>(
            (const I*)ids, (const E*)weight, (E*)out, T, V, N, ld, scale, (unsigned)slabs);
        return check_launch("emb_fwd_kernel");
      };
      return four ? go(emb_fwd_kernel<E, I, wide, 4>) : go(emb_fwd_kernel<E, I, wide, 1>);
    };
    constexpr int per = Vec16<E>::E;
    const bool wide = N % per == 0 && ld % per == 0 && aligned16(weight) && aligned16(out);
    return wide ? run(std::true_type{}) : run(std::false_type{});
  });
}

extern "C" int fo_embedding_bwd_workspace_bytes(int64_t T, int64_t V, int64_t N, int64_t* bytes) {
  clear_error();
  FO_CHECK_ARG(bytes, "embedding backward: null pointer");
  if (int rc = check_sizes(T, V, N)) return rc;
  *bytes = workspace(T, N).bytes;
  return FO_OK;
}

extern "C" int fo_embedding_bwd(const void* dout, const void* ids, void* dw, int64_t T, int64_t V,
                                int64_t N, int64_t padding_idx, float scale, int dtype,
                                int index_dtype, void* workspace_, int64_t ws_bytes,
                                void* stream) {
  clear_error();
  if (int rc = check_sizes(T, V, N)) return rc;
  if (V == 0 || N == 0) return FO_OK;
  FO_CHECK_ARG(dw && (T == 0 || (dout && ids)), "embedding backward: null pointer");
  const Workspace ws = workspace(T, N);
  if (T && (!workspace_ || ws_bytes < ws.bytes)) {
    set_error("embedding backward: workspace of %lld bytes required", (long long)ws.bytes);
    return FO_EWORKSPACE;
  }
  FO_CHECK_ARG(!T || aligned16(workspace_), "embedding backward: workspace must be 16-byte aligned");
  const int chunks = (int)((T + kChunk - 1) / kChunk);
  cudaStream_t st = as_stream(stream);
  return with_types(dtype, index_dtype, [&](auto t, auto i) {
    using E = decltype(t);
    using I = decltype(i);
    const int64_t bytes = V * N * (int64_t)sizeof(E);
    if (T == 0) {
      cudaMemsetAsync(dw, 0, (size_t)bytes, st);
      return check_launch("embedding backward (empty)");
    }
    auto at = [&](int64_t o) { return (char*)workspace_ + o; };
    int32_t *skey = (int32_t*)at(0), *spos = (int32_t*)at(ws.spos), *key = (int32_t*)at(ws.key),
            *pos = (int32_t*)at(ws.pos);
    float *part = (float*)at(ws.part), *runs = (float*)at(ws.runs);
    // Zeros: all with the sort, or a quarter of them with the merge, which takes about a third
    // of the sort's time.
    const int64_t first = chunks > 1 ? bytes / 4 * 3 / 256 * 256 : bytes;
    int bits = 0;
    while (bits < 31 && V >> bits) ++bits;
    cudaError_t e = allow_shared((const void*)emb_sort_kernel<I>, (int)sizeof(SortSmem));
    if (e != cudaSuccess) {
      cudaGetLastError();
      set_error("emb_sort_kernel: %s", cudaGetErrorString(e));
      return (int)FO_ECUDA;
    }
    emb_sort_kernel<I><<<chunks + zero_ctas(first), kSortThreads, sizeof(SortSmem), st>>>(
        (const I*)ids, skey, spos, T, V, padding_idx, (bits + kBits - 1) / kBits,
        Zeros{(uint8_t*)dw, first, (unsigned)chunks});
    if (int rc = check_launch("emb_sort_kernel")) return rc;
    if (chunks > 1) {
      const unsigned n = (unsigned)((T + kThreads - 1) / kThreads);
      emb_merge_kernel<<<n + zero_ctas(bytes - first), kThreads, 0, st>>>(
          skey, spos, key, pos, (int)T, chunks, Zeros{(uint8_t*)dw + first, bytes - first, n});
      if (int rc = check_launch("emb_merge_kernel")) return rc;
    }
    auto run = [&](auto wide) {
      constexpr int K = Columns<E, wide>::K;
      const int64_t nv = N / Vec<E, wide>::E, pieces = (T + kPiece - 1) / kPiece;
      int threads = 32;  // a CTA no wider than the row
      while (threads < kThreads && threads * K < nv) threads *= 2;
      const int64_t slabs = slabs_of(nv, pieces, threads * K);
      if (!slabs) return grid_error();
      emb_piece_kernel<E, wide><<<(unsigned)(pieces * slabs), threads, 0, st>>>(
          (const E*)dout, key, pos, part, (E*)dw, (int)T, V, N, scale, (unsigned)slabs);
      if (int rc = check_launch("emb_piece_kernel")) return rc;
      if (pieces == 1) return (int)FO_OK;
      if (const int64_t n = T / (kPiece * kRun)) {
        const int64_t sl = slabs_of(N, n, kThreads);
        if (!sl) return grid_error();
        emb_run_kernel<<<(unsigned)(n * sl), kThreads, 0, st>>>(key, part, runs, V, N, (unsigned)sl);
        if (int rc = check_launch("emb_run_kernel")) return rc;
      }
      emb_join_kernel<E, wide><<<(unsigned)((pieces - 1) * slabs), threads, 0, st>>>(
          key, part, runs, (E*)dw, (int)T, V, N, scale, (unsigned)slabs);
      return check_launch("emb_join_kernel");
    };
    constexpr int per = Vec16<E>::E;
    const bool wide = N % per == 0 && aligned16(dout) && aligned16(dw);
    return wide ? run(std::true_type{}) : run(std::false_type{});
  });
}
