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
// weighted sum (rescaled when a pack of 16 bytes raises the maximum) in 32 bits; they
// are joined at the row's end.  For the alternatives every warp keeps a list of
// candidates no smaller than a bound that the whole row shares: the k-th
// largest of 64 maxima taken from the row's first packs, raised whenever a list fills up
// and is cut back to its k largest.  Elements below the bound cost one comparison a pack.
// Few long rows are split over a cluster of up to 8 CTAs, which join through
// distributed shared memory: no workspace, and the same order of sums each time.
#include <cooperative_groups.h>

#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = 64;
constexpr int kList = 128;    // candidates a warp holds
constexpr int kSeeds = 64;    // maxima that give the first bound
constexpr float kLn2 = 0.693147180559945309f;

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
  float m = -3.402823466e38f, s = 0.f, w = 0.f;
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

template <bool ENT, int N>
__device__ __forceinline__ void add_pack(Running& r, const float (&x)[N], float cm, float k2) {
  if (cm > r.m) {
    const float d = fmaxf((r.m - cm) * k2, -1e4f), f = ex2(d);
    if (ENT) r.w = f * (r.w + d * r.s);
    r.s *= f;
    r.m = cm;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float y = (x[i] - r.m) * k2;
    const float e = ex2(y);
    r.s += e;
    if (ENT) r.w = fmaf(fmaxf(y, -1e4f), e, r.w);
  }
}

template <int THREADS>
struct LogShared {
  unsigned long long bound;                       // no candidate below it is needed
  uint32_t count;
  unsigned long long lists[THREADS / 32][kList];
  unsigned long long all[THREADS / 32 * kList];   // the lists joined; seeds before that
  float m[THREADS / 32], s[THREADS / 32], w[THREADS / 32];
  unsigned long long best[kMaxTop];               // this CTA's top_k, sorted
  float part[3];                                  // this CTA's m, s, w
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

// The whole warp offers N elements a lane from index `at` on (valid ones: n).
template <int N>
__device__ __forceinline__ void offer(const float (&x)[N], uint32_t at, int n, uint32_t k, unsigned long long* list,
                                      uint32_t& count, volatile unsigned long long* bound) {
  const uint32_t lane = threadIdx.x & 31;
  unsigned long long b = *bound;
  uint32_t open = 0;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n && key_of(x[i], at + i) >= b) open |= 1u << i;
  while (__any_sync(~0u, open)) {
    if (count > kList - 32) {
      count = cut(list, count, k, const_cast<unsigned long long*>(bound));
      b = *bound;
    }
    unsigned long long key = 0;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (__ffs(open) - 1 == i) key = key_of(x[i], at + i);
    open &= open - 1;
    const bool take = key != 0 && key >= b;
    const uint32_t who = __ballot_sync(~0u, take);
    if (take) list[count + __popc(who & ((1u << lane) - 1))] = key;
    count += __popc(who);
    __syncwarp();
  }
}

// Ranks n unique keys by counting; those below k go to out, sorted.
template <int THREADS>
__device__ __forceinline__ void rank_into(const unsigned long long* keys, uint32_t n, uint32_t k, unsigned long long* out) {
  for (uint32_t i = threadIdx.x; i < n; i += THREADS) {
    const unsigned long long mine = keys[i];
    uint32_t rank = 0;
    for (uint32_t j = 0; j < n; ++j) rank += keys[j] > mine;
    if (rank < k) out[rank] = mine;
  }
}

template <typename T, int THREADS, bool ENT, bool TOP>
__global__ void __launch_bounds__(THREADS)
gpuos_logprobs_kernel(const __grid_constant__ LogArgs a) {
  constexpr int W = 16 / sizeof(T);
  constexpr int U = 4;  // packs a thread has in flight
  extern __shared__ __align__(16) uint8_t smem[];
  LogShared<THREADS>& sh = *reinterpret_cast<LogShared<THREADS>*>(smem);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t parts = cluster.num_blocks(), part = cluster.block_rank();
  const int64_t row = blockIdx.x / parts;
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;

  // the row is a head up to the first 16-byte boundary, whole packs, and a tail
  const uint32_t cols = (uint32_t)a.cols;
  const uint32_t off = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const uint32_t head = min(cols, off ? W - off : 0u);
  const uint32_t packs = (cols - head) / W;
  const uint32_t p0 = (uint32_t)((uint64_t)packs * part / parts), p1 = (uint32_t)((uint64_t)packs * (part + 1) / parts);
  const uint32_t tail = head + packs * W;
  const T* body = x + head;

  Running r;
  uint32_t count = 0;
  if (TOP && threadIdx.x == 0) {
    sh.bound = 0;
    sh.count = 0;
  }

  // the loose elements, at most 2 (W - 1), go to the last part's first warp
  float loose = -INFINITY;
  uint32_t loose_at = 0;
  bool has_loose = false;
  if (part == parts - 1 && warp == 0) {
    const uint32_t nl = head + (cols - tail);
    has_loose = lane < nl;
    if (has_loose) {
      loose_at = lane < head ? lane : tail + (lane - head);
      loose = to_f(x[loose_at]);
    }
  }

  for (uint32_t base = p0; base < p1; base += THREADS * U) {
    Pack<T, W> q[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t p = base + u * THREADS + threadIdx.x;
      if (p < p1) q[u] = load_pack<T, W>(body + (uint64_t)p * W);
    }
    if (TOP && base == p0) {
      // the first bound: the k-th largest of 64 maxima, each over its own lanes' first packs
      unsigned long long best = 0;
      if (p0 + threadIdx.x < p1) {
        const uint32_t at = head + (p0 + threadIdx.x) * W;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const unsigned long long key = key_of(to_f(q[0].v[i]), at + i);
          best = key > best ? key : best;
        }
      }
#pragma unroll
      for (int d = 1; d < THREADS / kSeeds; d <<= 1) {
        const unsigned long long o = __shfl_xor_sync(~0u, best, d);
        best = o > best ? o : best;
      }
      if (threadIdx.x % (THREADS / kSeeds) == 0) sh.all[threadIdx.x / (THREADS / kSeeds)] = best;
      __syncthreads();
      if (threadIdx.x < kSeeds) {
        const unsigned long long mine = sh.all[threadIdx.x];
        uint32_t rank = 0;
        for (int j = 0; j < kSeeds; ++j) rank += sh.all[j] > mine;
        if (mine != 0 && rank == a.top_k - 1) sh.bound = mine;
      }
      __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t first = base + u * THREADS + warp * 32;  // the warp's first pack
      if (first >= p1) break;
      const uint32_t p = first + lane;
      float v[W];
      float cm = -INFINITY;
      const bool in = p < p1;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        v[i] = in ? to_f(q[u].v[i]) : -INFINITY;
        cm = fmaxf(cm, v[i]);
      }
      add_pack<ENT, W>(r, v, cm, a.k2);
      if (TOP) {
        const float least = value_of(*(volatile unsigned long long*)&sh.bound);
        if (__any_sync(~0u, in && cm >= least))
          offer<W>(v, head + p * W, in ? W : 0, a.top_k, sh.lists[warp], count, &sh.bound);
      }
    }
  }
  if (TOP && p0 >= p1) __syncthreads();  // the bound's start is set
  if (part == parts - 1 && warp == 0) {
    const float v[1] = {loose};
    if (has_loose) add_pack<ENT, 1>(r, v, fmaxf(loose, -INFINITY), a.k2);
    if (TOP) offer<1>(v, loose_at, has_loose ? 1 : 0, a.top_k, sh.lists[warp], count, &sh.bound);
  }

  // join: lanes, warps, then the cluster's CTAs, always in the same order
#pragma unroll
  for (int d = 16; d; d >>= 1) {
    const float m = __shfl_xor_sync(~0u, r.m, d), s = __shfl_xor_sync(~0u, r.s, d), w = __shfl_xor_sync(~0u, r.w, d);
    join<ENT>(r, m, s, w, a.k2);
  }
  if (lane == 0) {
    sh.m[warp] = r.m;
    sh.s[warp] = r.s;
    sh.w[warp] = r.w;
  }
  __syncthreads();
  if (TOP) {
    const unsigned long long b = *(volatile unsigned long long*)&sh.bound;
    for (uint32_t i = lane; i < count; i += 32) {
      const unsigned long long key = sh.lists[warp][i];
      if (key >= b) sh.all[atomicAdd(&sh.count, 1u)] = key;
    }
    for (uint32_t i = threadIdx.x; i < a.top_k; i += THREADS) sh.best[i] = 0;
    __syncthreads();
    rank_into<THREADS>(sh.all, sh.count, a.top_k, sh.best);
  }
  if (threadIdx.x == 0) {
    Running c;
    for (int i = 0; i < THREADS / 32; ++i) join<ENT>(c, sh.m[i], sh.s[i], sh.w[i], a.k2);
    sh.part[0] = c.m;
    sh.part[1] = c.s;
    sh.part[2] = c.w;
  }
  if (parts > 1) cluster.sync();
  else __syncthreads();
  if (part == 0) {
    Running c;
    for (uint32_t i = 0; i < parts; ++i) {
      const float* o = parts > 1 ? cluster.map_shared_rank(sh.part, i) : sh.part;
      join<ENT>(c, o[0], o[1], o[2], a.k2);
    }
    const float ln_s = logf(c.s);
    const bool none = c.s == 0.f;  // every logit is -inf
    if (threadIdx.x == 0) {
      const int64_t y = load_index(a.targets, a.target_wide, row * a.ts);
      float lp;
      if (y < 0) lp = 0.f;
      else if (y >= a.cols) lp = NAN;
      else lp = none ? -INFINITY : (to_f(x[y]) - c.m) / a.t - ln_s;
      a.logprob[row * a.ls] = lp;
      if (ENT) a.entropy[row * a.es] = none ? 0.f : ln_s - kLn2 * c.w / c.s;
      if (a.stats) {
        a.stats[row * a.ss] = c.m;
        a.stats[row * a.ss + a.sk] = c.s;
      }
    }
    if (TOP) {
      const unsigned long long* best = sh.best;
      if (parts > 1) {
        // the parts' lists, joined and ranked again
        for (uint32_t i = threadIdx.x; i < parts * a.top_k; i += THREADS)
          sh.all[i] = cluster.map_shared_rank(sh.best, i / a.top_k)[i % a.top_k];
        __syncthreads();
        unsigned long long* out = sh.lists[0];
        rank_into<THREADS>(sh.all, parts * a.top_k, a.top_k, out);
        __syncthreads();
        best = out;
      }
      for (uint32_t i = threadIdx.x; i < a.top_k; i += THREADS) {
        const float v = value_of(best[i]);
        a.top[row * a.tps + i * a.tpk] = none ? -INFINITY : (v - c.m) / a.t - ln_s;
        const uint32_t token = ~(uint32_t)best[i];
        if (a.token_wide) static_cast<int64_t*>(a.tokens)[row * a.tks + i * a.tkk] = token;
        else static_cast<int32_t*>(a.tokens)[row * a.tks + i * a.tkk] = (int32_t)token;
      }
    }
  }
  if (parts > 1) cluster.sync();  // the other CTAs' shared memory is read above
}

constexpr int kGradThreads = 256;
constexpr int kGradPacks = 4;

// One CTA a stretch of a row: the row's constants are folded into
// dx = e (A + B y) with y = (x - m) log2(e) / t, e = 2^y.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kGradThreads)
gpuos_logprobs_grad_kernel(const __grid_constant__ LogArgs a) {
  constexpr int W = VEC ? 16 / sizeof(T) : 1;
  const int64_t row = blockIdx.x;
  const T* x = static_cast<const T*>(a.x) + row * a.xs;
  T* o = static_cast<T*>(a.gx) + row * a.gs;
  const int64_t y = load_index(a.targets, a.target_wide, row * a.ts);
  const float m = a.stats[row * a.ss], s = a.stats[row * a.ss + a.sk];
  float g = a.gl && y >= 0 ? a.gl[row * a.gls] : 0.f;
  if (a.gl && y >= a.cols) g = NAN;
  const float h = a.ge ? a.ge[row * a.ges] : 0.f;
  const float H = a.ge ? a.entropy[row * a.es] : 0.f;
  const bool none = s == 0.f;
  const float c0 = none ? 0.f : -a.inv_t / s;
  const float A = none ? 0.f : c0 * (g + h * (H - logf(s))), B = c0 * h * (kLn2);
  const float hit = none ? 0.f : g * a.inv_t;

  auto value = [&](float v, int64_t at) {
    const float y2 = fmaxf((v - m) * a.k2, -1e4f);
    float d = v == v ? ex2(y2) * fmaf(B, y2, A) : NAN;
    if (at == y) d += hit;
    return d;
  };
  const uint32_t cols = (uint32_t)a.cols;
  uint32_t head = 0;
  if (VEC) {
    const uint32_t off = (uint32_t)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
    head = min(cols, off ? W - off : 0u);
  }
  const uint32_t packs = (cols - head) / W, tail = head + packs * W;
  const uint32_t base = blockIdx.y * (kGradThreads * kGradPacks) + threadIdx.x;
  if (VEC && blockIdx.y == 0) {
    for (uint32_t i = threadIdx.x; i < head; i += kGradThreads) o[i] = from_f<T>(value(to_f(x[i]), i));
    for (uint32_t i = tail + threadIdx.x; i < cols; i += kGradThreads) o[i] = from_f<T>(value(to_f(x[i]), i));
  }
  Pack<T, W> q[kGradPacks];
#pragma unroll
  for (int u = 0; u < kGradPacks; ++u) {
    const uint32_t p = base + u * kGradThreads;
    if (p < packs) q[u] = load_pack<T, W>(x + head + (uint64_t)p * W);
  }
#pragma unroll
  for (int u = 0; u < kGradPacks; ++u) {
    const uint32_t p = base + u * kGradThreads;
    if (p >= packs) break;
    const int64_t at = head + (int64_t)p * W;
#pragma unroll
    for (int i = 0; i < W; ++i) q[u].v[i] = from_f<T>(value(to_f(q[u].v[i]), at + i));
    store_pack<T, W>(o + at, q[u]);
  }
}

template <typename T, int THREADS, bool ENT, bool TOP>
void launch(const LogArgs& a, uint32_t parts, cudaStream_t s) {
  const size_t smem = sizeof(LogShared<THREADS>);
  auto kernel = gpuos_logprobs_kernel<T, THREADS, ENT, TOP>;
  if (smem > 48 * 1024)
    cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "shared memory");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(a.rows * parts));
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = parts;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&cfg, kernel, a), "launch");
}

template <typename T, int THREADS>
void by_outputs(const LogArgs& a, uint32_t parts, cudaStream_t s) {
  if (a.entropy && a.top_k) launch<T, THREADS, true, true>(a, parts, s);
  else if (a.entropy) launch<T, THREADS, true, false>(a, parts, s);
  else if (a.top_k) launch<T, THREADS, false, true>(a, parts, s);
  else launch<T, THREADS, false, false>(a, parts, s);
}

template <typename T>
void forward(const LogArgs& a, cudaStream_t s) {
  constexpr int64_t kStep = 512 * 16 / sizeof(T);  // elements a CTA reads at once
  uint32_t parts = 1;
  while (parts < 8 && a.rows * parts < 2 * sm_count() && a.cols >= kStep * parts * 2) parts *= 2;
  // a row of one step of 128 threads leaves most of a larger CTA idle
  if (parts == 1 && a.cols <= kStep / 2) by_outputs<T, 128>(a, parts, s);
  else by_outputs<T, 512>(a, parts, s);
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
void backward(const LogArgs& a, cudaStream_t s) {
  const int64_t per = (int64_t)kGradThreads * kGradPacks * (a.vec ? 16 / (int)sizeof(T) : 1);
  const int64_t parts = (a.cols + per - 1) / per;
  need(parts < 65536, "too many tokens");
  const dim3 grid((unsigned)a.rows, (unsigned)parts);
  if (a.vec) gpuos_logprobs_grad_kernel<T, true><<<grid, kGradThreads, 0, s>>>(a);
  else gpuos_logprobs_grad_kernel<T, false><<<grid, kGradThreads, 0, s>>>(a);
  cuda_ok(cudaGetLastError(), "launch");
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
