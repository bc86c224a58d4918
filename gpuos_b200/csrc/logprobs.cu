// gpuos_logprobs / gpuos_logprobs_grad: over a row x of V logits, temperature t,
// with m = max x and z = (x - m) / t,
//
//   s = sum e^z         log p(y) = z_y - ln s         H = ln s - (sum z e^z) / s
//
// and the k likeliest tokens (ties: the lowest index) with their log
// probabilities; the gradient, with p = e^z / s, is
//
//   dx_j = (g (1[j = y] - p_j) - h p_j (z_j - ln s + H)) / t
//
// for the gradients g of log p(y) and h of H.
//
// Forward reads the row once.  A thread keeps its own running maximum, sum and
// weighted sum in 32 bits, rescaled when a step of U 16-byte packs raises the
// maximum; they are joined at the row's end.  The alternatives cost nothing
// while the row streams but a maximum that each thread leaves behind now and
// then.  At the row's end the k-th largest of the threads' maxima is a bound
// that k elements reach, and only packs under a maximum that reaches it are read
// again (a few KB).  Rows of many equal or masked logits make more candidates than that:
// they are read again whole, through lists of a warp each, cut back when full
// to the k largest, which raises the bound.  Few or
// long rows are split over a cluster of up to 8 CTAs, which join through
// distributed shared memory: no workspace, and the same order of sums each time.
//
// At 16 bits an SM's share of the memory rate is about 12 elements a cycle,
// its exponentials 16, its instructions 128 lanes: the loop is kept to about 5
// instructions an element (maxima of two elements at once, packed 32-bit sums and products).
// 2048 x 128257 bf16 take 85 us (6.2 TB/s), with 5 alternatives 96; 1500 x 50257 fp32 with entropy
// 49 (6.1 TB/s); their gradient, which reads and writes, 89 (6.7 TB/s).
#include <cooperative_groups.h>

#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = 64;
constexpr int kRowThreads = 256;  // of a row; short rows take a warp each, 8 to a CTA
constexpr int kList = 128;    // candidates a warp holds
constexpr int kWarpPacks = 128;  // 16-byte packs of a row that a warp has in flight at once
constexpr int kWarpTop = 24;     // alternatives of a row that a warp takes, at most
constexpr int kWarpReads = 16000;  // packs times alternatives of such a row
constexpr int kLongPacks = 14000;  // of a row whose threads have eight packs in flight

constexpr int kSeeds = 64;
constexpr int kFewTop = 32;   // alternatives up to which 64 maxima give a close bound
constexpr int kFewRounds = 8;  // and up to which a warp takes a round for each (8192 x 300 with 5: 14.1 us, by bits 14.7)
constexpr float kLn2 = 0.693147180559945309f;
constexpr float kLowest = -3.402823466e38f;  // the lowest finite number: where a maximum starts

struct LogArgs {
  const void* x;
  int64_t xs;
  const void* targets;
  int64_t ts;
  int64_t rows, cols;
  float* logprob; int64_t ls;
  float* entropy; int64_t es;
  float* top; int64_t tps, tpk;
  void* tokens; int64_t tks, tkk;
  float* stats; int64_t ss, sk;     // (m, s) of each row
  // gradient
  void* gx; int64_t gs;
  const float* gl; int64_t gls;
  const float* ge; int64_t ges;
  float k2;       // log2(e) / t
  float t, inv_t;
  uint32_t top_k;
  uint32_t parts;   // gradient: CTAs of a row
  int target_wide, token_wide, vec;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// An unsigned integer that orders as x does (NaN as -inf), above the
// complement of the index: unique, and of equal values the lowest index is the largest.
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) {
  if (x != x) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t k = (b >> 31) ? ~b : b | 0x80000000u;
  return ((unsigned long long)k << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float value_of(unsigned long long key) {
  const uint32_t k = (uint32_t)(key >> 32);
  return k == 0 ? -INFINITY : __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// Running maximum m, s = sum 2^y and w = sum y 2^y with y = (x - m) log2(e) / t.
// m starts at the lowest finite number, so a masked (-inf) element is just a zero term.
struct Running {
  float m = kLowest, s = 0.f, w = 0.f;
  __device__ Running() {}
  __device__ Running(float m_, float s_, float w_) : m(m_), s(s_), w(w_) {}
};

template <bool ENT>
__device__ __forceinline__ void join(Running& a, float m, float s, float w, float k2) {
  const float top = fmaxf(a.m, m);
  // far apart: the factor is 0, and the product with the difference must not be inf * 0
  const float da = fmaxf((a.m - top) * k2, -1e4f), db = fmaxf((m - top) * k2, -1e4f);
  const float fa = ex2(da), fb = ex2(db);
  if (ENT) a.w = fa * (a.w + da * a.s) + fb * (w + db * s);
  a.s = fa * a.s + fb * s;
  a.m = top;
}

// Joins the first LANES lanes of a warp.
template <int LANES, bool ENT>
__device__ __forceinline__ Running join_lanes(Running t, float k2) {
#pragma unroll
  for (int d = LANES / 2; d; d >>= 1) {
    const float m = __shfl_xor_sync(~0u, t.m, d), s = __shfl_xor_sync(~0u, t.s, d), w = __shfl_xor_sync(~0u, t.w, d);
    join<ENT>(t, m, s, w, k2);
  }
  return t;
}

// The maximum of a pack's elements; a NaN does not count.
template <typename T, int N>
__device__ __forceinline__ float max_of(const Pack<T, N>& x) {
  if constexpr (sizeof(T) == 2 && N % 2 == 0) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* h = reinterpret_cast<const T2*>(&x);
    T2 m = h[0];
#pragma unroll
    for (int i = 1; i < N / 2; ++i) m = __hmax2(m, h[i]);
    return fmaxf(to_f(m.x), to_f(m.y));
  } else {
    float m = to_f(x.v[0]);
#pragma unroll
    for (int i = 1; i < N; ++i) m = fmaxf(m, to_f(x.v[i]));
    return m;
  }
}

// Running sums of a thread: s and w in two parts each, for packed arithmetic.
struct Sums {
  float m = kLowest;
  float2 s = {0.f, 0.f}, w = {0.f, 0.f};
};

// Raises the maximum to cm (a NaN or anything smaller does nothing).
template <bool ENT>
__device__ __forceinline__ void raise(Sums& r, float cm, float k2) {
  if (cm > r.m) {
    const float d = fmaxf((r.m - cm) * k2, -1e4f), f = ex2(d);
    if (ENT) r.w = mul2(both(f), fma2(both(d), r.s, r.w));
    r.s = mul2(both(f), r.s);
    r.m = cm;
  }
}

template <bool ENT>
__device__ __forceinline__ void add_two(Sums& r, float2 x, float k2) {
  const float2 y = mul2(add2(x, both(-r.m)), both(k2));
  const float2 e = make_float2(ex2(y.x), ex2(y.y));
  r.s = add2(r.s, e);
  // a masked element's y is -inf: its term is 0, not inf * 0
  if (ENT) r.w = fma2(make_float2(fmaxf(y.x, -1e4f), fmaxf(y.y, -1e4f)), e, r.w);
}

constexpr uint32_t kMarks = 16;    // maxima a thread leaves on its way along a row
constexpr uint32_t kReach = 4;     // of them a thread, on average, may reach the bound, and
constexpr uint32_t kFew = 4;       // packs a thread then reads again at once

// Kept small: what the CTAs of an SM do not take of its memory holds their loads
// in flight (at 45 KB a CTA the loop ran a third slower than at 15).
template <typename T, int THREADS>
struct TopShared {
  static constexpr uint32_t kWarps = THREADS / 32;
  static constexpr uint32_t kPool = std::max<uint32_t>(kMarks * THREADS * sizeof(T) / 8, kWarps * (kList + kMaxTop));
  static constexpr uint32_t kAll = std::min<uint32_t>(kPool, 1024);
  static constexpr uint32_t kReached = kReach * THREADS;
  unsigned long long bound;          // no candidate below it is needed
  uint32_t count;                    // of the candidates
  uint32_t reached;                  // of `reach`
  alignas(16) float seeds[kSeeds];
  uint32_t reach[kReached];           // (mark, thread) whose maximum reaches the bound
  unsigned long long last[kMaxTop];  // the top_k, sorted
  // one after the other: the marks; the candidates; where those are too many, each
  // warp's list, and behind them the lists joined
  unsigned long long pool[kPool];
  unsigned long long best[];         // of a cluster's first CTA: each part's top_k
  __device__ T* marks() { return reinterpret_cast<T*>(pool); }
  __device__ unsigned long long* list(uint32_t warp) { return pool + warp * kList; }
  __device__ unsigned long long* joined() { return pool + kWarps * kList; }
};

__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// The threads of a row: a CTA, or a warp of one.
template <int THREADS>
__device__ __forceinline__ void row_sync() {
  if constexpr (THREADS == 32) __syncwarp();
  else __syncthreads();
}

template <int THREADS> constexpr int kRowsOfCta = THREADS == 32 ? 8 : 1;

template <int THREADS> struct RowShared;
template <int THREADS> constexpr size_t kTopAt = (sizeof(RowShared<THREADS>) + 15) / 16 * 16;

template <int THREADS>
struct RowShared {
  float m[THREADS / 32], s[THREADS / 32], w[THREADS / 32];
  Running part[8];                   // each part's m, s, w
};

// Cuts a warp's list of n keys to its k largest, sorted, and raises the bound.
__device__ __forceinline__ uint32_t cut(unsigned long long* list, uint32_t n, uint32_t k, unsigned long long* bound) {
  const uint32_t lane = threadIdx.x & 31;
  unsigned long long mine[kList / 32];
  uint32_t rank[kList / 32];
#pragma unroll
  for (int i = 0; i < kList / 32; ++i) {
    mine[i] = lane + 32 * i < n ? list[lane + 32 * i] : 0;
    rank[i] = 0;
  }
  for (uint32_t j = 0; j < n; ++j) {
    const unsigned long long o = list[j];
#pragma unroll
    for (int i = 0; i < kList / 32; ++i) rank[i] += o > mine[i];
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kList / 32; ++i)
    if (mine[i] != 0 && rank[i] < k) {
      list[rank[i]] = mine[i];
      if (rank[i] == k - 1) atomicMax(bound, mine[i]);
    }
  __syncwarp();
  return n < k ? n : k;
}

// The whole warp offers N elements a lane from index `at` on; `open` says which.
template <typename T, int N>
__device__ __forceinline__ void offer(const Pack<T, N>& x, uint32_t open, uint32_t at, uint32_t k,
                                      unsigned long long* list, uint32_t& count, unsigned long long* bound) {
  const uint32_t lane = threadIdx.x & 31;
  unsigned long long b = *(volatile unsigned long long*)bound;
  while (__any_sync(~0u, open)) {
    if (count > kList - 32) {
      count = cut(list, count, k, bound);
      b = *(volatile unsigned long long*)bound;
    }
    const int first = __ffs(open) - 1;
    float v = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (first == i) v = to_f(x.v[i]);
    const unsigned long long key = key_of(v, at + first);
    const bool take = open != 0 && key >= b;
    open &= open - 1;
    const uint32_t who = __ballot_sync(~0u, take);
    if (take) list[count + __popc(who & ((1u << lane) - 1))] = key;
    count += __popc(who);
    __syncwarp();
  }
}

// Which of the elements of a pack at index `at` have a key of at least `bound` (a NaN
// stands for -inf in the order).
template <typename T, int N>
__device__ __forceinline__ uint32_t candidates(const Pack<T, N>& x, uint32_t at, unsigned long long bound) {
  const float least = value_of(bound);
  const uint32_t last = ~(uint32_t)bound;  // of elements equal to it, those up to its index
  uint32_t open = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float v = to_f(x.v[i]);
    if (v > least || (!(v < least) && (v == least || least == -INFINITY) && at + i <= last)) open |= 1u << i;
  }
  return open;
}

// Ranks n unique keys by counting the larger ones; those below k go to out, sorted.
// In a CTA 8 lanes count for a key; a warp's lanes take a key each and read all keys together.
template <int THREADS>
__device__ __forceinline__ void rank_into(const unsigned long long* keys, uint32_t n, uint32_t k, unsigned long long* out) {
  constexpr uint32_t L = THREADS == 32 ? 1 : 8;  // lanes to a key
  const uint32_t tid = threadIdx.x % THREADS;
  for (uint32_t i0 = 0; i0 < n; i0 += THREADS / L) {
    const uint32_t i = i0 + tid / L;
    const unsigned long long mine = i < n ? keys[i] : 0;
    uint32_t rank = 0;
#pragma unroll 4
    for (uint32_t j = tid % L; j < n; j += L) rank += keys[j] > mine;
#pragma unroll
    for (uint32_t d = 1; d < L; d <<= 1) rank += __shfl_xor_sync(~0u, rank, d);
    if (tid % L == 0 && i < n && rank < k) out[rank] = mine;
  }
}

template <int THREADS>
__device__ __forceinline__ uint32_t row_count(bool p) {
  if constexpr (THREADS == 32) return __popc(__ballot_sync(~0u, p));
  else return __syncthreads_count(p);
}

// The bound: a value that k of the row's elements reach, from the threads' maxima.  A maximum
// that is still where it started was reached by nothing and does not count: with fewer than k
// others there is no bound.  (8 x 32000 with 20 alternatives: 7.7 us by 64 maxima, 8.2 by bits; with 64,
// too many for 64 maxima, 10.5 by bits.)
template <typename T, int THREADS>
__device__ __forceinline__ void find_bound(TopShared<T, THREADS>& top, float m, uint32_t k, uint32_t packs) {
  const int tid = threadIdx.x % THREADS;
  if (THREADS == 32 && k <= kFewRounds) {
    // a round for each alternative: the largest of those left
    float me = m;
    for (uint32_t i = 0; i < k; ++i) {
      me = warp_max(m);
      if (tid == __ffs(__ballot_sync(~0u, m == me)) - 1) m = -INFINITY;
    }
    if (tid == 0 && me > kLowest) top.bound = key_of(me, 0) & ~0xffffffffull;
  } else if (THREADS > 32 && k <= kFewTop && packs >= THREADS) {
    // the k-th largest of 64 maxima over neighbouring threads, 4 lanes to each
    constexpr int S = kSeeds, L = THREADS > S ? THREADS / S : 1;
    const int at = tid / L;
    uint32_t rank = 0;
#pragma unroll
    for (int d = 1; d < L; d <<= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, d));
    if (tid % L == 0) top.seeds[at] = m;
    row_sync<THREADS>();
#pragma unroll
    for (int j = tid % L * 4; j < S; j += L * 4) {
      const float4 o = *reinterpret_cast<const float4*>(top.seeds + j);
      rank += (o.x > m || (o.x == m && j < at)) + (o.y > m || (o.y == m && j + 1 < at)) +
              (o.z > m || (o.z == m && j + 2 < at)) + (o.w > m || (o.w == m && j + 3 < at));
    }
#pragma unroll
    for (int d = 1; d < L; d <<= 1) rank += __shfl_xor_sync(~0u, rank, d);
    if (tid % L == 0 && rank == k - 1 && m > kLowest) top.bound = key_of(m, 0) & ~0xffffffffull;
  } else {
    // the largest leading bits that k of all the maxima reach (of 32 bits the value to 2^-11)
    constexpr int kBits = std::is_same_v<T, __nv_bfloat16> ? 16 : 20;
    const uint32_t mine = m > kLowest ? (uint32_t)(key_of(m, 0) >> 32) : 0;
    uint32_t t = 0;
    for (int b = 31; b >= 32 - kBits; --b)
      if (row_count<THREADS>(mine >= (t | 1u << b)) >= k) t |= 1u << b;
    if (tid == 0) top.bound = (unsigned long long)t << 32;
  }
  row_sync<THREADS>();
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

template <typename T, int THREADS, bool TOP>
constexpr size_t kSharedOfRow = (kTopAt<THREADS> + (TOP ? sizeof(TopShared<T, THREADS>) : 0) + 15) / 16 * 16;

// U packs a thread in flight: four, with more CTAs of an SM, or eight, with fewer.
template <typename T, int THREADS, int U, bool ENT, bool TOP>
__global__ void __launch_bounds__(THREADS * kRowsOfCta<THREADS>, THREADS == 32 ? 5 : U == 4 ? 6 : 4)
gpuos_logprobs_kernel(const __grid_constant__ LogArgs a) {
  constexpr int W = 16 / sizeof(T);
  extern __shared__ __align__(16) uint8_t smem[];
  const uint32_t tid = threadIdx.x % THREADS, lane = tid & 31, warp = tid / 32;
  uint8_t* mem = smem + threadIdx.x / THREADS * kSharedOfRow<T, THREADS, TOP>;
  RowShared<THREADS>& sh = *reinterpret_cast<RowShared<THREADS>*>(mem);
  TopShared<T, THREADS>& top = *reinterpret_cast<TopShared<T, THREADS>*>(mem + kTopAt<THREADS>);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts = THREADS == 32 ? 1 : cluster.num_blocks(), part = THREADS == 32 ? 0 : cluster.block_rank();
  const int64_t row = (int64_t)(blockIdx.x / parts) * kRowsOfCta<THREADS> + threadIdx.x / THREADS;
  if (THREADS == 32 && row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;

  // the row is a head up to the first 16-byte boundary, whole packs, and a tail
  const uint32_t cols = (uint32_t)a.cols;
  const uint32_t off = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const uint32_t head = min(cols, off ? W - off : 0u);
  const uint32_t packs = (cols - head) / W;
  const uint32_t p0 = (uint32_t)((uint64_t)packs * part / parts), p1 = (uint32_t)((uint64_t)packs * (part + 1) / parts);
  const uint32_t tail = head + packs * W;
  const T* body = x + head;

  // read ahead: the row's end needs it
  int64_t target = -1;
  float target_x = 0.f;
  if (part == 0 && tid == 0) {
    target = load_index(a.targets, a.target_wide, row * a.ts);
    if (target >= 0 && target < a.cols) target_x = to_f(x[target]);
  }
  if (parts > 1) cluster_arrive();

  Sums r;
  if (TOP) {
    if (tid == 0) {
      top.bound = 0;
      top.count = 0;
      top.reached = 0;
    }
    for (uint32_t i = tid; i < a.top_k; i += THREADS) top.last[i] = 0;
  }

  // the loose elements, at most 2 (W - 1), go to the last part's first warp
  Pack<T, 1> loose;
  uint32_t loose_at = 0;
  bool has_loose = false;
  if (part == parts - 1 && warp == 0) {
    has_loose = lane < head + (cols - tail);
    if (has_loose) {
      loose_at = lane < head ? lane : tail + (lane - head);
      loose.v[0] = x[loose_at];
      raise<ENT>(r, to_f(loose.v[0]), a.k2);
      add_two<ENT>(r, make_float2(to_f(loose.v[0]), -INFINITY), a.k2);
    }
  }

  // the candidates of a pack at index `at`, of `bound` and above
  auto push = [&](const auto& q, uint32_t at, unsigned long long bound) {
    constexpr int N = sizeof(q.v) / sizeof(T);
    uint32_t open = candidates<T, N>(q, at, bound);
    while (open) {
      const int e = __ffs(open) - 1;
      open &= open - 1;
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (e == i) v = to_f(q.v[i]);
      const uint32_t n = atomicAdd(&top.count, 1u);
      if (n < top.kAll) top.pool[n] = key_of(v, at + e);
    }
  };

  const uint32_t steps = (p1 - p0 + THREADS * U - 1) / (THREADS * U);
  const uint32_t stretch = (steps + kMarks - 1) / kMarks;  // steps a mark covers
  uint32_t mark = 0, left = stretch;
  float marked = -INFINITY;
  for (uint32_t base = p0; base < p1; base += THREADS * U) {
    // a step: U packs a thread, all of them or (the last step) those below p1
    Pack<T, W> q[U];
    const uint32_t mine = base + tid;
    const bool whole = base + THREADS * U <= p1;
    if (whole) {
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = load_pack<T, W>(body + (uint64_t)(mine + u * THREADS) * W);
    } else {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (mine + u * THREADS < p1) {
          q[u] = load_pack<T, W>(body + (uint64_t)(mine + u * THREADS) * W);
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) q[u].v[i] = from_f<T>(-INFINITY);
        }
      }
    }
    float cm = max_of(q[0]);
#pragma unroll
    for (int u = 1; u < U; ++u) cm = fmaxf(cm, max_of(q[u]));
    raise<ENT>(r, cm, a.k2);
    if (TOP) {
      if (THREADS == 32 && steps == 1) {
        // the whole row is in registers: its candidates are taken from there
        find_bound<T, THREADS>(top, r.m, a.top_k, p1 - p0);
        const unsigned long long bound = top.bound;
        if (!(cm < value_of(bound)))
#pragma unroll
          for (int u = 0; u < U; ++u)
            if (mine + u * THREADS < p1) push(q[u], head + (mine + u * THREADS) * W, bound);
        if (has_loose) push(loose, loose_at, bound);
      } else {
        marked = fmaxf(marked, cm);
        if (--left == 0 || base + THREADS * U >= p1) {
          top.marks()[mark++ * THREADS + tid] = from_f<T>(marked);
          marked = -INFINITY;
          left = stretch;
        }
      }
    }
    // a last step's missing packs are -inf: terms of 0
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < W; i += 2) add_two<ENT>(r, make_float2(to_f(q[u].v[i]), to_f(q[u].v[i + 1])), a.k2);
  }

  // join: lanes, warps, then the cluster's CTAs, always in the same order
  const Running t = join_lanes<32, ENT>(Running{r.m, r.s.x + r.s.y, r.w.x + r.w.y}, a.k2);
  if (THREADS > 32 && lane == 0) {
    sh.m[warp] = t.m;
    sh.s[warp] = t.s;
    sh.w[warp] = t.w;
  }
  bool few = true;
  if (TOP && !(THREADS == 32 && steps == 1)) {
    find_bound<T, THREADS>(top, r.m, a.top_k, p1 - p0);
    const unsigned long long bound = top.bound;
    if (r.m >= value_of(bound))
      for (uint32_t i = 0; i < mark; ++i)
        if (to_f(top.marks()[i * THREADS + tid]) >= value_of(bound)) {
          const uint32_t n = atomicAdd(&top.reached, 1u);
          if (n < top.kReached) top.reach[n] = i << 16 | tid;
        }
    row_sync<THREADS>();
    // the packs under those marks, a lane each
    const uint32_t each = stretch * U;
    few = top.reached <= top.kReached &&
          (uint64_t)top.reached * each <= max(kFew * THREADS, (p1 - p0) / 4);
    if (few) {
      const uint32_t items = top.reached * each;
      for (uint32_t i0 = 0; i0 < items; i0 += kFew * THREADS) {
        Pack<T, W> q[kFew];
        uint32_t at[kFew];
#pragma unroll
        for (int u = 0; u < kFew; ++u) {
          const uint32_t it = i0 + u * THREADS + tid;
          at[u] = p1;
          if (it < items) {
            const uint32_t i = it / each, to = top.reach[i];
            at[u] = p0 + ((to >> 16) * each + (it - i * each)) * THREADS + (to & 0xffff);
          }
          if (at[u] < p1) q[u] = load_pack<T, W, false>(body + (uint64_t)at[u] * W);
        }
#pragma unroll
        for (int u = 0; u < kFew; ++u)
          if (at[u] < p1) push(q[u], head + at[u] * W, bound);
      }
      if (has_loose) push(loose, loose_at, bound);
    }
  }
  row_sync<THREADS>();
  if (TOP) {
    if (!few || top.count > top.kAll) {
      // many equal or masked logits: the row again, through lists that are cut
      row_sync<THREADS>();
      if (tid == 0) top.count = 0;
      uint32_t count = 0;  // of this warp's list
      for (uint32_t p = p0 + tid; __any_sync(~0u, p < p1); p += THREADS) {
        Pack<T, W> q;
        uint32_t open = 0;
        if (p < p1) {
          q = load_pack<T, W>(body + (uint64_t)p * W);
          open = candidates<T, W>(q, head + p * W, *(volatile unsigned long long*)&top.bound);
        }
        offer<T, W>(q, open, head + p * W, a.top_k, top.list(warp), count, &top.bound);
      }
      if (part == parts - 1 && warp == 0)
        offer<T, 1>(loose, has_loose ? candidates<T, 1>(loose, loose_at, *(volatile unsigned long long*)&top.bound) : 0u,
                    loose_at, a.top_k, top.list(warp), count, &top.bound);
      if (count > a.top_k) count = cut(top.list(warp), count, a.top_k, &top.bound);
      row_sync<THREADS>();
      const unsigned long long b = *(volatile unsigned long long*)&top.bound;
      for (uint32_t i = lane; i < count; i += 32) {
        const unsigned long long key = top.list(warp)[i];
        if (key >= b) top.joined()[atomicAdd(&top.count, 1u)] = key;
      }
      row_sync<THREADS>();
      rank_into<THREADS>(top.joined(), top.count, a.top_k, top.last);
    } else {
      rank_into<THREADS>(top.pool, top.count, a.top_k, top.last);
    }
    if (parts > 1) __syncthreads();
  }
  // every part writes its results into the shared memory of the row's first CTA,
  // which has started (the barrier above) and waits for them (the one below)
  Running* to = &sh.part[part];
  if (parts > 1) {
    cluster_wait();
    to = cluster.map_shared_rank(to, 0);
    if (TOP) {
      unsigned long long* best = cluster.map_shared_rank(top.best, 0) + part * a.top_k;
      for (uint32_t i = tid; i < a.top_k; i += THREADS) best[i] = top.last[i];
    }
  }
  if (THREADS > 32 && warp == THREADS / 32 - 1) {
    Running c;
    if (lane < THREADS / 32) c = Running{sh.m[lane], sh.s[lane], sh.w[lane]};
    c = join_lanes<THREADS / 32, ENT>(c, a.k2);
    if (lane == 0) *to = c;
  }
  if (parts > 1) {
    cluster_arrive();
    if (part != 0) return;
    cluster_wait();
    if (TOP) {
      // each part has `share` keys no smaller than the smallest of the parts' share-th ones, so
      // all together top_k or more: smaller ones drop out before the rest are ranked
      const uint32_t share = (a.top_k + parts - 1) / parts;
      unsigned long long least = ~0ull;
      for (uint32_t i = 0; i < parts; ++i) least = min(least, top.best[i * a.top_k + share - 1]);
      if (tid == 0) top.count = 0;
      __syncthreads();
      for (uint32_t i = tid; i < parts * a.top_k; i += THREADS)
        if (top.best[i] >= least && top.best[i] != 0) top.pool[atomicAdd(&top.count, 1u)] = top.best[i];
      __syncthreads();
      rank_into<THREADS>(top.pool, top.count, a.top_k, top.last);
    }
  }
  row_sync<THREADS>();
  if (warp != 0) return;
  Running c = THREADS == 32 ? t : sh.part[0];
  if (parts > 1) {
    c = Running{};
    if (lane < parts) c = sh.part[lane];
    c = join_lanes<8, ENT>(c, a.k2);
    c = Running{__shfl_sync(~0u, c.m, 0), __shfl_sync(~0u, c.s, 0), __shfl_sync(~0u, c.w, 0)};
  }
  const float ln_s = logf(c.s);
  const bool none = c.s == 0.f;  // every logit is -inf
  if (lane == 0) {
    float lp;
    if (target < 0) lp = 0.f;
    else if (target >= a.cols) lp = NAN;
    else lp = none ? -INFINITY : (target_x - c.m) / a.t - ln_s;
    a.logprob[row * a.ls] = lp;
    if (ENT) a.entropy[row * a.es] = none ? 0.f : ln_s - kLn2 * c.w / c.s;
    if (a.stats) {
      a.stats[row * a.ss] = c.m;
      a.stats[row * a.ss + a.sk] = c.s;
    }
  }
  if (TOP) {
    for (uint32_t i = lane; i < a.top_k; i += 32) {
      const unsigned long long key = top.last[i];
      a.top[row * a.tps + i * a.tpk] = none ? -INFINITY : (value_of(key) - c.m) / a.t - ln_s;
      const uint32_t token = ~(uint32_t)key;
      if (a.token_wide) static_cast<int64_t*>(a.tokens)[row * a.tks + i * a.tkk] = token;
      else static_cast<int32_t*>(a.tokens)[row * a.tks + i * a.tkk] = (int32_t)token;
    }
  }
}

constexpr int kGradThreads = 128;
constexpr int kGradPacks = 4;

// One CTA a stretch of a row: the row's constants are folded into
// dx = e (A + B y) with y = (x - m) log2(e) / t, e = 2^y.
template <typename T, bool VEC, bool ENT>
__global__ void __launch_bounds__(kGradThreads)
gpuos_logprobs_grad_kernel(const __grid_constant__ LogArgs a) {
  constexpr int W = VEC ? 16 / sizeof(T) : 1;
  const int64_t row = blockIdx.x / a.parts;
  const uint32_t part = blockIdx.x - (uint32_t)row * a.parts;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  T* o = static_cast<T*>(a.gx) + row * a.gs;
  const uint32_t cols = (uint32_t)a.cols;
  uint32_t head = 0;
  if (VEC) {
    const uint32_t off = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    head = min(cols, off ? W - off : 0u);
  }
  const uint32_t packs = (cols - head) / W, tail = head + packs * W;
  const uint32_t base = part * (kGradThreads * kGradPacks) + threadIdx.x;
  Pack<T, W> q[kGradPacks];
#pragma unroll
  for (int u = 0; u < kGradPacks; ++u) {
    const uint32_t p = base + u * kGradThreads;
    if (p < packs) q[u] = load_pack<T, W>(x + head + (uint64_t)p * W);
  }

  const int64_t y = load_index(a.targets, a.target_wide, row * a.ts);
  const float m = a.stats[row * a.ss], s = a.stats[row * a.ss + a.sk];
  float g = a.gl && y >= 0 ? a.gl[row * a.gls] : 0.f;
  if (a.gl && y >= a.cols) g = NAN;
  const float h = ENT ? a.ge[row * a.ges] : 0.f, H = ENT ? a.entropy[row * a.es] : 0.f;
  const bool none = s == 0.f;
  const float c0 = none ? 0.f : -a.inv_t / s;
  const float A = none ? 0.f : ENT ? c0 * (g + h * (H - logf(s))) : c0 * g, B = c0 * h * kLn2;
  const float hit = none ? 0.f : g * a.inv_t;
  const uint32_t at_y = y >= 0 && y < a.cols ? (uint32_t)y : ~0u;

  auto two = [&](float2 v) {
    const float2 z = mul2(add2(v, both(-m)), both(a.k2));
    const float2 e = make_float2(ex2(z.x), ex2(z.y));
    if (!ENT) return mul2(e, both(A));
    // a masked element's z is -inf: e is 0, and its factor must stay finite
    return mul2(e, fma2(make_float2(fmaxf(z.x, -1e4f), fmaxf(z.y, -1e4f)), both(B), both(A)));
  };
  auto one = [&](uint32_t i) {
    const float d = two(make_float2(to_f(x[i]), 0.f)).x + (i == at_y ? hit : 0.f);
    o[i] = from_f<T>(d);
  };
  if (VEC && part == 0) {
    if (threadIdx.x < head) one(threadIdx.x);
    if (threadIdx.x < cols - tail) one(tail + threadIdx.x);
  }
#pragma unroll
  for (int u = 0; u < kGradPacks; ++u) {
    const uint32_t p = base + u * kGradThreads;
    if (p >= packs) break;
    const uint32_t at = head + p * W;
    float d[W];
    if constexpr (W == 1) {
      d[0] = two(make_float2(to_f(q[u].v[0]), 0.f)).x;
    } else {
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        const float2 r = two(make_float2(to_f(q[u].v[i]), to_f(q[u].v[i + 1])));
        d[i] = r.x;
        d[i + 1] = r.y;
      }
    }
    if (at_y - at < (uint32_t)W) {
#pragma unroll
      for (int i = 0; i < W; ++i)
        if (at + i == at_y) d[i] += hit;
    }
#pragma unroll
    for (int i = 0; i < W; ++i) q[u].v[i] = from_f<T>(d[i]);
    if constexpr (VEC) __stcs(reinterpret_cast<uint4*>(o + at), *reinterpret_cast<const uint4*>(&q[u]));
    else o[at] = q[u].v[0];
  }
}

template <typename T, int THREADS, int U, bool ENT, bool TOP>
void launch(const LogArgs& a, uint32_t parts, cudaStream_t s) {
  constexpr int kRows = kRowsOfCta<THREADS>;
  const size_t smem = kRows * kSharedOfRow<T, THREADS, TOP> + (TOP && parts > 1 ? parts * a.top_k * 8 : 0);
  auto kernel = gpuos_logprobs_kernel<T, THREADS, U, ENT, TOP>;  // (up to 30 KB of shared memory)
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((a.rows + kRows - 1) / kRows * parts));
  cfg.blockDim = dim3(THREADS * kRows);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = parts > 1 ? 1 : 0;
  cuda_ok(cudaLaunchKernelEx(&cfg, kernel, a), "launch");
}

template <typename T, int THREADS, int U>
void by_outputs(const LogArgs& a, uint32_t parts, cudaStream_t s) {
  if (a.entropy && a.top_k) launch<T, THREADS, U, true, true>(a, parts, s);
  else if (a.entropy) launch<T, THREADS, U, true, false>(a, parts, s);
  else if (a.top_k) launch<T, THREADS, U, false, true>(a, parts, s);
  else launch<T, THREADS, U, false, false>(a, parts, s);
}

template <typename T>
void forward(const LogArgs& a, cudaStream_t s) {
  constexpr int64_t kStep = kRowThreads * 16 / sizeof(T);  // elements a CTA reads at once
  const int64_t sms = sm_count();
  // A warp a row: short rows with few alternatives (8 x 250 with 8: 5.5 us, a CTA a row 7.0), or rows
  // enough for the warps of every SM, the more the longer they are (1183 x 24000 with 5 alternatives:
  // 33 us, CTAs 24; 4096 x 24000: 57 and 64; 4096 x 1000: 10 and 42).  Its 32 maxima give a loose
  // bound, so that what it reads again grows with the alternatives and the row (4096 x 8000 with 16: 34
  // us, CTAs 46, with 24: 58 and 48; x 24000 with 16: 76 and 67).
  const int64_t packs = a.cols * (int64_t)sizeof(T) / 16, k = a.top_k;
  if ((packs <= kWarpPacks && k <= kFewRounds) ||
      (a.rows >= sms * (2 + packs / 160) && k <= kWarpTop && packs * std::max<int64_t>(k, 5) <= kWarpReads))
    return by_outputs<T, 32, 4>(a, 1, s);
  uint32_t parts = 1;
  // (8 x 32000 with 20 alternatives: 8.4 us over 4 CTAs a row, 9.3 over 8, 8.8 over 2)
  while (parts < 8 && a.rows * parts < 2 * sms && a.cols >= kStep * parts * 4) parts *= 2;
  // Long whole rows: fewer CTAs with more in flight each keep the memory busy while the last rows
  // run (1000 x 128000 bf16: 46.5 us, 53.6 with four packs in flight).  Many shorter rows of 16 bits lose
  // by it: 1000 and 3000 of them take 0.94 and 1.06 of the time at 13000 packs, 0.90 and 1.01
  // at 14000, 0.87 and 1.01 at 16000 (6282: 1.02 and 1.12; of 32 bits 0.91 and 1.00 at 13000, 0.87 and 0.98 above).
  if (parts == 1 && packs >= kLongPacks) by_outputs<T, kRowThreads, 8>(a, parts, s);
  else by_outputs<T, kRowThreads, 4>(a, parts, s);
}

LogArgs prepare(const gpuos_tensor* x, const gpuos_tensor* targets, float temperature) {
  check_tensor(x, 2, "logits");
  check_tensor(targets, 1, "targets");
  need(is_real(x->dtype), "logits must be float32, float16 or bfloat16");
  need(is_index(targets->dtype), "targets must be int32 or int64");
  need(targets->sizes[0] == x->sizes[0], "targets must name one token for each row");
  need(temperature > 0.f && temperature <= 1e30f && temperature >= 1e-30f, "temperature must be in [1e-30, 1e30]");
  need(x->sizes[1] >= 1 && x->sizes[1] < (1ll << 30), "the number of tokens must be in [1, 2^30)");
  need(x->sizes[0] < (1ll << 27), "too many rows");
  if (numel(*x)) need(x->sizes[1] == 1 || x->strides[1] == 1, "the last dim of logits must be contiguous");
  LogArgs a{};
  a.x = x->data;
  a.xs = x->strides[0];
  a.targets = targets->data;
  a.ts = targets->strides[0];
  a.target_wide = targets->dtype == GPUOS_I64;
  a.rows = x->sizes[0];
  a.cols = x->sizes[1];
  a.k2 = (float)(1.4426950408889634074 / (double)temperature);
  a.t = temperature;
  a.inv_t = (float)(1.0 / (double)temperature);
  return a;
}

// A float32 tensor of a value for each row.
void row_values(const gpuos_tensor* t, const gpuos_tensor& x, const char* name) {
  check_tensor(t, 1, name);
  if (t->dtype != GPUOS_F32 || t->sizes[0] != x.sizes[0])
    invalid(std::string(name) + " must be float32, one for each row");
}

void row_stats(const gpuos_tensor* t, const gpuos_tensor& x) {
  check_tensor(t, 2, "stats");
  need(t->dtype == GPUOS_F32 && t->sizes[0] == x.sizes[0] && t->sizes[1] == 2, "stats must be float32, two for each row");
}

void logprobs(const gpuos_tensor* x, const gpuos_tensor* targets, const gpuos_tensor* logprob, const gpuos_tensor* entropy,
              const gpuos_tensor* top, const gpuos_tensor* tokens, const gpuos_tensor* stats, float temperature,
              cudaStream_t stream) {
  LogArgs a = prepare(x, targets, temperature);
  row_values(logprob, *x, "logprob");
  a.logprob = static_cast<float*>(logprob->data);
  a.ls = logprob->strides[0];
  if (entropy) {
    row_values(entropy, *x, "entropy");
    a.entropy = static_cast<float*>(entropy->data);
    a.es = entropy->strides[0];
  }
  need(!top == !tokens, "top_logprobs and top_tokens come together");
  if (top) {
    check_tensor(top, 2, "top_logprobs");
    check_tensor(tokens, 2, "top_tokens");
    need(top->dtype == GPUOS_F32 && is_index(tokens->dtype), "top_logprobs must be float32, top_tokens int32 or int64");
    need(top->sizes[0] == a.rows && tokens->sizes[0] == a.rows && top->sizes[1] == tokens->sizes[1],
         "top_logprobs and top_tokens must have a row for each row of logits");
    need(top->sizes[1] >= 1 && top->sizes[1] <= kMaxTop && top->sizes[1] <= a.cols,
         "the alternatives must be in [1, min(64, tokens)]");
    a.top_k = (uint32_t)top->sizes[1];
    a.top = static_cast<float*>(top->data);
    a.tps = top->strides[0];
    a.tpk = top->strides[1];
    a.tokens = tokens->data;
    a.tks = tokens->strides[0];
    a.tkk = tokens->strides[1];
    a.token_wide = tokens->dtype == GPUOS_I64;
  }
  if (stats) {
    row_stats(stats, *x);
    a.stats = static_cast<float*>(stats->data);
    a.ss = stats->strides[0];
    a.sk = stats->strides[1];
  }
  const gpuos_tensor* outs[5] = {logprob, entropy, top, tokens, stats};
  for (int i = 0; i < 5; ++i) {
    if (!outs[i]) continue;
    check_output(*outs[i], "an output");
    no_overlap(*outs[i], *x, "an output overlaps logits");
    no_overlap(*outs[i], *targets, "an output overlaps targets");
    for (int k = 0; k < i; ++k)
      if (outs[k]) no_overlap(*outs[i], *outs[k], "two outputs overlap");
  }
  if (a.rows == 0) return;
  if (x->dtype == GPUOS_F32) forward<float>(a, stream);
  else if (x->dtype == GPUOS_F16) forward<__half>(a, stream);
  else forward<__nv_bfloat16>(a, stream);
}

template <typename T>
void backward(LogArgs a, cudaStream_t s) {
  const int64_t per = (int64_t)kGradThreads * kGradPacks * (a.vec ? 16 / (int)sizeof(T) : 1);
  const int64_t parts = (a.cols + per - 1) / per;
  need(a.rows * parts < 0x7fffffffll, "too many logits");
  a.parts = (uint32_t)parts;
  const unsigned grid = (unsigned)(a.rows * parts);
  if (a.vec && a.ge) run(gpuos_logprobs_grad_kernel<T, true, true>, grid, kGradThreads, 0, s, a);
  else if (a.vec) run(gpuos_logprobs_grad_kernel<T, true, false>, grid, kGradThreads, 0, s, a);
  else if (a.ge) run(gpuos_logprobs_grad_kernel<T, false, true>, grid, kGradThreads, 0, s, a);
  else run(gpuos_logprobs_grad_kernel<T, false, false>, grid, kGradThreads, 0, s, a);
}

void logprobs_grad(const gpuos_tensor* x, const gpuos_tensor* targets, const gpuos_tensor* stats, const gpuos_tensor* entropy,
                   const gpuos_tensor* gl, const gpuos_tensor* ge, const gpuos_tensor* gx, float temperature,
                   cudaStream_t stream) {
  LogArgs a = prepare(x, targets, temperature);
  row_stats(stats, *x);
  a.stats = static_cast<float*>(stats->data);
  a.ss = stats->strides[0];
  a.sk = stats->strides[1];
  need(gl || ge, "grad_logprob or grad_entropy must be given");
  if (gl) {
    row_values(gl, *x, "grad_logprob");
    a.gl = static_cast<const float*>(gl->data);
    a.gls = gl->strides[0];
  }
  if (ge) {
    need(entropy != nullptr, "grad_entropy needs entropy");
    row_values(ge, *x, "grad_entropy");
    row_values(entropy, *x, "entropy");
    a.ge = static_cast<const float*>(ge->data);
    a.ges = ge->strides[0];
    a.entropy = static_cast<float*>(entropy->data);
    a.es = entropy->strides[0];
  }
  check_tensor(gx, 2, "grad_logits");
  need(gx->dtype == x->dtype, "grad_logits must have the dtype of logits");
  same_sizes(*gx, *x, "grad_logits must have the sizes of logits");
  if (numel(*gx)) need(gx->sizes[1] == 1 || gx->strides[1] == 1, "the last dim of grad_logits must be contiguous");
  check_output(*gx, "grad_logits");
  need(same_view(*gx, *x) || !overlap(*gx, *x), "grad_logits must be logits or not overlap them");
  const gpuos_tensor* ins[5] = {targets, stats, ge ? entropy : nullptr, gl, ge};
  for (const gpuos_tensor* t : ins)
    if (t) no_overlap(*gx, *t, "grad_logits overlap an input");
  a.gx = gx->data;
  a.gs = gx->strides[0];
  if (a.rows == 0) return;
  // packs of both rows start together where their addresses agree modulo 16 bytes
  const int w = 16 / esize(x->dtype);
  a.vec = (reinterpret_cast<uintptr_t>(x->data) - reinterpret_cast<uintptr_t>(gx->data)) % 16 == 0 &&
          (a.rows == 1 || (a.xs - a.gs) % w == 0);
  if (x->dtype == GPUOS_F32) backward<float>(a, stream);
  else if (x->dtype == GPUOS_F16) backward<__half>(a, stream);
  else backward<__nv_bfloat16>(a, stream);
}

}  // namespace
}  // namespace rowops
}  // namespace gpuos

extern "C" int32_t gpuos_logprobs(const gpuos_tensor* logits, const gpuos_tensor* targets, const gpuos_tensor* logprob,
                                  const gpuos_tensor* entropy, const gpuos_tensor* top_logprobs,
                                  const gpuos_tensor* top_tokens, const gpuos_tensor* stats, float temperature,
                                  void* stream) {
  return gpuos::rowops::entry("gpuos_logprobs", [&] {
    gpuos::rowops::logprobs(logits, targets, logprob, entropy, top_logprobs, top_tokens, stats, temperature,
                            static_cast<cudaStream_t>(stream));
  });
}

extern "C" int32_t gpuos_logprobs_grad(const gpuos_tensor* logits, const gpuos_tensor* targets, const gpuos_tensor* stats,
                                       const gpuos_tensor* entropy, const gpuos_tensor* grad_logprob,
                                       const gpuos_tensor* grad_entropy, const gpuos_tensor* grad_logits,
                                       float temperature, void* stream) {
  return gpuos::rowops::entry("gpuos_logprobs_grad", [&] {
    gpuos::rowops::logprobs_grad(logits, targets, stats, entropy, grad_logprob, grad_entropy, grad_logits, temperature,
                                 static_cast<cudaStream_t>(stream));
  });
}
