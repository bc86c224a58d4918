// gpuos_order / gpuos_dispatch / gpuos_combine / gpuos_combine_grad: token rows
// sorted by the experts that gpuos_route chose, and the experts' results brought
// back.  Choice i = t * k + j of token t has expert e_i; with n_e choices of
// expert e and their number rounded up to a multiple of `align`,
//
//   first_e = sum over e' < e of ceil(n_e' / align) * align
//   place_i = first_(e_i) + #{i' < i : e_i' = e_i}            (a stable counting sort)
//   dispatch:  row[place_i] = x[t]                             zeros elsewhere
//   combine:   out[t] = sum_j w_i y[place_i]
//   gradient:  dy[place_i] = w_i dout[t]   dw_i = <dout[t], y[place_i]>
//
// dispatch's gradient is combine without weights.  All but the sort move rows:
// each is bound by memory and moves every byte once, so dispatch reads a token's row once
// and writes it to its k places rather than gather by place (a gather reads it k times).
// 16384 tokens x 2 of 8 x 4096 bf16: dispatch 73 us (403 MB, 5.5 TB/s), combine 66 (6.1 TB/s), its gradient 147
// (671 MB, 4.6 TB/s); the sort of 72008 choices over 256 experts 20 us, latency on 8 SMs.
#include <cooperative_groups.h>

#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kMaxExperts = 1024, kMaxChoices = 64;
constexpr uint32_t kCounts = 7168;    // 32-bit counters a CTA of the sort holds (28 KB)
constexpr uint32_t kSortCluster = 8;
constexpr uint32_t kAhead = 8;        // steps of 32 choices that a warp loads at once

// ---- the sort --------------------------------------------------------------------
struct OrderArgs {
  const void* experts;
  int64_t st, sk;
  int32_t *places, *sources, *offsets, *counts;
  FastDiv k;
  uint32_t n, count, align, rows;
  uint32_t warps;     // of a CTA
  uint32_t per_warp;  // choices, a multiple of 32
  int wide, plain;    // plain: choices lie one behind the other
};

__device__ __forceinline__ int32_t expert_of(const OrderArgs& a, uint32_t i) {
  int64_t at = i;
  if (!a.plain) {
    const uint32_t t = a.k.div(i);
    at = t * a.st + (i - t * a.k.d) * a.sk;
  }
  const int64_t e = load_index(a.experts, a.wide, at);
  return e >= 0 && e < a.count ? (int32_t)e : -1;
}

// One cluster.  A warp takes neighbouring choices 32 at a time and counts those of an
// expert by one vote, in counters of its own; the counters become places by sums over
// warps, CTAs (through distributed shared memory) and experts, and a second pass hands
// the places out in the same order: no atomics, the same result each time.
__global__ void __launch_bounds__(1024)
gpuos_order_kernel(const __grid_constant__ OrderArgs a) {
  extern __shared__ uint32_t counters[];  // [warps][count]
  __shared__ uint32_t total[kMaxExperts];   // of this CTA, read by the others
  __shared__ uint32_t amount[kMaxExperts];  // of all
  __shared__ uint32_t ahead[kMaxExperts];   // of the CTAs before this one; then where this one's rows begin
  __shared__ uint32_t first[kMaxExperts + 1], group[32];
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), parts = cluster.num_blocks();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, threads = blockDim.x;
  const uint32_t below = (1u << lane) - 1;
  uint32_t* mine = counters + warp * a.count;

  for (uint32_t i = threadIdx.x; i < a.warps * a.count; i += threads) counters[i] = 0;
  __syncthreads();
  const uint32_t lo = (uint32_t)min((uint64_t)(rank * a.warps + warp) * a.per_warp, (uint64_t)a.n);
  const uint32_t hi = (uint32_t)min((uint64_t)lo + a.per_warp, (uint64_t)a.n);
  // (kAhead steps' choices are loaded before the first is looked at: 72008 choices of 256 experts took 24 us one by one)
  for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kAhead) {
    int32_t e[kAhead];
#pragma unroll
    for (uint32_t s = 0; s < kAhead; ++s) e[s] = i0 + 32 * s + lane < hi ? expert_of(a, i0 + 32 * s + lane) : -1;
#pragma unroll
    for (uint32_t s = 0; s < kAhead; ++s) {
      if (i0 + 32 * s >= hi) break;
      const uint32_t same = __match_any_sync(~0u, e[s]);
      if (e[s] >= 0 && !(same & below)) mine[e[s]] += __popc(same);
      __syncwarp();
    }
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < a.count; e += threads) {
    uint32_t sum = 0;
    for (uint32_t w = 0; w < a.warps; ++w) {
      const uint32_t c = counters[w * a.count + e];
      counters[w * a.count + e] = sum;
      sum += c;
    }
    total[e] = sum;
  }
  cluster.sync();
  // a warp takes 32 experts: the sum before each of them, then before each 32
  const uint32_t groups = (a.count + 31) / 32;
  for (uint32_t g = warp; g < groups; g += a.warps) {
    const uint32_t e = g * 32 + lane;
    uint32_t before = 0, all = 0;
    if (e < a.count)
      for (uint32_t c = 0; c < parts; ++c) {
        const uint32_t v = *cluster.map_shared_rank(&total[e], c);
        if (c < rank) before += v;
        all += v;
      }
    const uint32_t padded = (all + a.align - 1) / a.align * a.align;
    uint32_t sum = padded;
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const uint32_t v = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += v;
    }
    if (lane == 31) group[g] = sum;
    if (e < a.count) {
      ahead[e] = before;
      amount[e] = all;
      first[e] = sum - padded;
    }
  }
  cluster.sync();  // no CTA leaves, or goes on, while another reads its `total`
  if (warp == 0) {
    const uint32_t v = lane < groups ? group[lane] : 0;
    uint32_t sum = v;
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const uint32_t u = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += u;
    }
    group[lane] = sum - v;
    if (lane == 31) first[a.count] = sum;
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < a.count; e += threads) {
    first[e] += group[e >> 5];
    ahead[e] += first[e];
    if (rank == 0) {
      a.offsets[e] = (int32_t)first[e];
      a.counts[e] = (int32_t)amount[e];
    }
  }
  if (rank == 0 && threadIdx.x == 0) a.offsets[a.count] = (int32_t)first[a.count];
  __syncthreads();
  for (uint32_t i0 = lo; i0 < hi; i0 += 32 * kAhead) {
    int32_t e[kAhead];
#pragma unroll
    for (uint32_t s = 0; s < kAhead; ++s) e[s] = i0 + 32 * s + lane < hi ? expert_of(a, i0 + 32 * s + lane) : -1;
#pragma unroll
    for (uint32_t s = 0; s < kAhead; ++s) {
      const uint32_t i = i0 + 32 * s + lane;
      if (i0 + 32 * s >= hi) break;
      const uint32_t same = __match_any_sync(~0u, e[s]);
      uint32_t at = 0;
      if (e[s] >= 0) at = ahead[e[s]] + mine[e[s]] + __popc(same & below);
      __syncwarp();
      if (e[s] >= 0 && !(same & below)) mine[e[s]] += __popc(same);
      __syncwarp();
      if (i < hi) a.places[i] = e[s] >= 0 ? (int32_t)at : -1;
      if (e[s] >= 0) a.sources[at] = (int32_t)i;
    }
  }
  // rows of no choice: behind each expert's, and behind the last expert's
  if (a.align > 1)
    for (uint32_t e = rank * a.warps + warp; e < a.count; e += parts * a.warps)
      for (uint32_t r = first[e] + amount[e] + lane; r < first[e + 1]; r += 32) a.sources[r] = -1;
  for (uint64_t r = (uint64_t)first[a.count] + rank * threads + threadIdx.x; r < a.rows; r += parts * threads)
    a.sources[r] = -1;
}

// ---- moving rows -------------------------------------------------------------------
// A row is cut into chunks of 32 lanes x kUnroll packs; (token, chunk) pairs are
// numbered through and a warp takes one.  Behind the tokens' warps come those that
// write zeros into rows of no choice.
constexpr uint32_t kThreads = 256, kWarps = kThreads / 32, kUnroll = 4;

struct MoveArgs {
  const void* x;        // dispatch: tokens; combine: rows; gradient: rows
  void* out;            // dispatch: rows; combine: tokens; gradient: rows
  const void* g;        // gradient: tokens
  const float* w;       // may be NULL: ones
  float* gw;            // gradient of the weights, (token, k); may be NULL
  const int32_t *places, *sources;
  int64_t xs, gs, ws, wk;  // strides of a row, and of the weights
  uint32_t tokens, k, rows;
  uint32_t width;       // of a row in elements
  uint32_t packs;       // of a row
  FastDiv chunks;       // of a row
  uint32_t units;       // tokens x chunks
};

// Zeros where a row is of no choice: unit u of rows x chunks.
template <typename P>
__device__ __forceinline__ void blank(const MoveArgs& a, uint64_t u, uint32_t lane) {
  const uint64_t r = u / a.chunks.d;
  if (r >= a.rows || __ldg(a.sources + r) >= 0) return;
  P* o = static_cast<P*>(a.out) + r * a.packs;
  const uint32_t p0 = (uint32_t)(u - r * a.chunks.d) * 32 * kUnroll + lane;
  const P zero{};
#pragma unroll
  for (uint32_t i = 0; i < kUnroll; ++i)
    if (p0 + 32 * i < a.packs) o[p0 + 32 * i] = zero;
}

template <typename P>  // uint4, uint32_t or uint16_t: rows are copied as bits
__global__ void __launch_bounds__(kThreads)
gpuos_dispatch_kernel(const __grid_constant__ MoveArgs a) {
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t unit = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= a.units) return blank<P>(a, unit - a.units, lane);
  const uint32_t t = a.chunks.div((uint32_t)unit), p0 = ((uint32_t)unit - t * a.chunks.d) * 32 * kUnroll + lane;
  const P* x = static_cast<const P*>(a.x) + t * a.xs;
  P v[kUnroll];
#pragma unroll
  for (uint32_t i = 0; i < kUnroll; ++i)
    if (p0 + 32 * i < a.packs) v[i] = __ldcs(x + p0 + 32 * i);
  for (uint32_t j = 0; j < a.k; ++j) {
    const int32_t r = __ldg(a.places + (uint64_t)t * a.k + j);
    if (r < 0 || r >= a.rows) continue;
    P* o = static_cast<P*>(a.out) + (uint64_t)r * a.packs;
#pragma unroll
    for (uint32_t i = 0; i < kUnroll; ++i)
      if (p0 + 32 * i < a.packs) o[p0 + 32 * i] = v[i];
  }
}

// Sums in 32 bits, in the order of the choices.
template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
gpuos_combine_kernel(const __grid_constant__ MoveArgs a) {
  constexpr uint32_t U = 2;
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t unit = (uint64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
  if (unit >= a.units) return;
  const uint32_t t = a.chunks.div((uint32_t)unit), p0 = ((uint32_t)unit - t * a.chunks.d) * 32 * U + lane;
  float sum[U][N];
#pragma unroll
  for (uint32_t i = 0; i < U; ++i)
#pragma unroll
    for (int c = 0; c < N; ++c) sum[i][c] = 0.f;
#pragma unroll 4
  for (uint32_t j = 0; j < a.k; ++j) {
    const int32_t r = __ldg(a.places + (uint64_t)t * a.k + j);
    if (r < 0 || r >= a.rows) continue;
    const float w = a.w ? __ldg(a.w + t * a.ws + j * a.wk) : 1.f;
    const T* y = static_cast<const T*>(a.x) + r * a.xs;
#pragma unroll
    for (uint32_t i = 0; i < U; ++i)
      if (p0 + 32 * i < a.packs) {
        const Pack<T, N> v = load_pack<T, N>(y + (p0 + 32 * i) * N);
#pragma unroll
        for (int c = 0; c < N; ++c) sum[i][c] = fmaf(w, to_f(v.v[c]), sum[i][c]);
      }
  }
  T* o = static_cast<T*>(a.out) + (uint64_t)t * a.width;
#pragma unroll
  for (uint32_t i = 0; i < U; ++i)
    if (p0 + 32 * i < a.packs) {
      Pack<T, N> v;
#pragma unroll
      for (int c = 0; c < N; ++c) v.v[c] = from_f<T>(sum[i][c]);
      store_pack(o + (p0 + 32 * i) * N, v);
    }
}

// A CTA takes a token: its gradient's row once for every kBatch choices, of which it
// writes the scaled rows and sums the products.
constexpr int kBatch = 8;

template <typename T, int N>
__global__ void __launch_bounds__(kThreads)
gpuos_combine_grad_kernel(const __grid_constant__ MoveArgs a) {
  __shared__ float part[kWarps][kBatch];
  const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  using P = std::conditional_t<sizeof(T) * N == 16, uint4, std::conditional_t<sizeof(T) * N == 4, uint32_t, uint16_t>>;
  if (blockIdx.x >= a.tokens) {
    for (uint64_t u = (uint64_t)(blockIdx.x - a.tokens) * kWarps + warp; u < (uint64_t)a.rows * a.chunks.d;
         u += (uint64_t)(gridDim.x - a.tokens) * kWarps)
      blank<P>(a, u, lane);
    return;
  }
  const uint32_t t = blockIdx.x;
  const T* g = static_cast<const T*>(a.g) + t * a.gs;
  for (uint32_t j0 = 0; j0 < a.k; j0 += kBatch) {
    int32_t r[kBatch];
    float w[kBatch], dot[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      r[j] = j0 + j < a.k ? __ldg(a.places + (uint64_t)t * a.k + j0 + j) : -1;
      if (r[j] >= a.rows) r[j] = -1;
      w[j] = r[j] < 0 ? 0.f : __ldg(a.w + t * a.ws + (j0 + j) * a.wk);
      dot[j] = 0.f;
    }
    for (uint32_t p = threadIdx.x; p < a.packs; p += kThreads) {
      const Pack<T, N> v = load_pack<T, N, false>(g + p * N);
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (r[j] < 0) continue;
        if (a.gw) {
          const Pack<T, N> y = load_pack<T, N>(static_cast<const T*>(a.x) + r[j] * a.xs + p * N);
#pragma unroll
          for (int c = 0; c < N; ++c) dot[j] = fmaf(to_f(v.v[c]), to_f(y.v[c]), dot[j]);
        }
        if (a.out) {
          Pack<T, N> o;
#pragma unroll
          for (int c = 0; c < N; ++c) o.v[c] = from_f<T>(w[j] * to_f(v.v[c]));
          store_pack(static_cast<T*>(a.out) + (uint64_t)r[j] * a.width + p * N, o);
        }
      }
    }
    if (!a.gw) continue;
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      for (int d = 16; d; d >>= 1) dot[j] += __shfl_xor_sync(~0u, dot[j], d);
    if (lane == 0)
#pragma unroll
      for (int j = 0; j < kBatch; ++j) part[warp][j] = dot[j];
    __syncthreads();
    if (threadIdx.x < kBatch && j0 + threadIdx.x < a.k) {
      float s = 0.f;
#pragma unroll
      for (uint32_t i = 0; i < kWarps; ++i) s += part[i][threadIdx.x];
      a.gw[(uint64_t)t * a.k + j0 + threadIdx.x] = s;
    }
    __syncthreads();
  }
}

// ---- host --------------------------------------------------------------------------
// The places of an order and the rows they lie in.
void check_order(const gpuos_tensor* places, const gpuos_tensor* sources) {
  check_tensor(places, 2, "places");
  check_tensor(sources, 1, "sources");
  need(places->dtype == GPUOS_I32 && sources->dtype == GPUOS_I32, "places and sources must be int32");
  need(places->sizes[1] >= 1 && places->sizes[1] <= kMaxChoices, "a token has between 1 and 64 choices");
  const int64_t n = numel(*places);
  need(n < (1ll << 31) && sources->sizes[0] < (1ll << 31), "too many choices");
  need(n == 0 || (places->strides[1] == 1 || places->sizes[1] == 1), "places must be contiguous");
  need(n == 0 || places->sizes[0] == 1 || places->strides[0] == places->sizes[1], "places must be contiguous");
  need(sources->sizes[0] <= 1 || sources->strides[0] == 1, "sources must be contiguous");
}

void check_rows(const gpuos_tensor* t, const char* name) {
  check_tensor(t, 2, name);
  if (!is_real(t->dtype)) invalid(std::string(name) + " must be float32, float16 or bfloat16");
  if (t->sizes[1] > 1 && t->strides[1] != 1) invalid(std::string(name) + ": the last dim must be contiguous");
  if (t->sizes[1] >= (1ll << 24)) invalid(std::string(name) + ": rows are too wide");
}

void check_plain(const gpuos_tensor* t, const char* name) {
  if (numel(*t) && t->sizes[0] > 1 && t->strides[0] != t->sizes[1]) invalid(std::string(name) + " must be contiguous");
}

void check_weights(const gpuos_tensor* w, const gpuos_tensor* places) {
  check_tensor(w, 2, "weights");
  need(w->dtype == GPUOS_F32, "weights must be float32");
  same_sizes(*w, *places, "weights must have the sizes of places");
}

MoveArgs move(const gpuos_tensor& places, const gpuos_tensor& sources, const gpuos_tensor& rows) {
  MoveArgs a{};
  a.places = static_cast<const int32_t*>(places.data);
  a.sources = static_cast<const int32_t*>(sources.data);
  a.tokens = (uint32_t)places.sizes[0];
  a.k = (uint32_t)places.sizes[1];
  a.rows = (uint32_t)sources.sizes[0];
  a.width = (uint32_t)rows.sizes[1];
  return a;
}

// Bytes moved at once: 16 where all rows start on a multiple of it and have whole packs, else 4, else an element.
int pack_bytes(const gpuos_tensor* const* t, int n) {
  const int size = esize(t[0]->dtype);
  for (const int b : {16, 4}) {
    bool fits = b >= size;
    for (int i = 0; i < n && fits; ++i) fits = t[i]->sizes[1] % (b / size) == 0 && rows_aligned(*t[i], b / size);
    if (fits) return b;
  }
  return size;
}

void cut(MoveArgs& a, int bytes, int size, uint32_t unroll) {
  a.packs = a.width / (bytes / size);
  const uint32_t chunks = (a.packs + 32 * unroll - 1) / (32 * unroll);
  a.chunks = FastDiv(chunks);
  need((uint64_t)a.tokens * chunks < (1ull << 31), "the call is too large");
  a.units = a.tokens * chunks;
}

uint32_t blocks(uint64_t units) {
  const uint64_t n = (units + kWarps - 1) / kWarps;
  need(n < (1ull << 31), "the call is too large");
  return (uint32_t)n;
}

template <typename T>
void launch_combine(const MoveArgs& a, int bytes, cudaStream_t stream) {
  const dim3 grid(blocks(a.units));
  if (bytes == 16) run(gpuos_combine_kernel<T, 16 / sizeof(T)>, grid, kThreads, 0, stream, a);
  else if (bytes == 4) run(gpuos_combine_kernel<T, 4 / sizeof(T)>, grid, kThreads, 0, stream, a);
  else if constexpr (sizeof(T) == 2) run(gpuos_combine_kernel<T, 1>, grid, kThreads, 0, stream, a);
}

template <typename T>
void launch_grad(const MoveArgs& a, int bytes, dim3 grid, cudaStream_t stream) {
  if (bytes == 16) run(gpuos_combine_grad_kernel<T, 16 / sizeof(T)>, grid, kThreads, 0, stream, a);
  else if (bytes == 4) run(gpuos_combine_grad_kernel<T, 4 / sizeof(T)>, grid, kThreads, 0, stream, a);
  else if constexpr (sizeof(T) == 2) run(gpuos_combine_grad_kernel<T, 1>, grid, kThreads, 0, stream, a);
}

}  // namespace
}  // namespace rowops
}  // namespace gpuos

using namespace gpuos::rowops;

extern "C" int32_t gpuos_order_rows(int64_t choices, int64_t count, int64_t align, int64_t* rows) {
  return entry("gpuos_order_rows", [&] {
    need(rows != nullptr, "rows is NULL");
    need(choices >= 0 && choices < (1ll << 31), "too many choices");
    need(count >= 1 && count <= kMaxExperts, "between 1 and 1024 experts");
    need(align >= 1 && align <= 65536, "align must be in [1, 65536]");
    *rows = (choices + std::min(count, choices) * (align - 1)) / align * align;
  });
}

extern "C" int32_t gpuos_order(const gpuos_tensor* experts, int32_t align, const gpuos_tensor* places,
                               const gpuos_tensor* sources, const gpuos_tensor* offsets, const gpuos_tensor* counts,
                               void* stream) {
  return entry("gpuos_order", [&] {
    check_tensor(experts, 2, "experts");
    need(is_index(experts->dtype), "experts must be int32 or int64");
    check_order(places, sources);
    check_tensor(offsets, 1, "offsets");
    check_tensor(counts, 1, "counts");
    need(offsets->dtype == GPUOS_I32 && counts->dtype == GPUOS_I32, "offsets and counts must be int32");
    same_sizes(*places, *experts, "places must have the sizes of experts");
    const int64_t count = counts->sizes[0], n = numel(*experts);
    need(count >= 1 && count <= kMaxExperts, "between 1 and 1024 experts");
    need(align >= 1 && align <= 65536, "align must be in [1, 65536]");
    need(offsets->sizes[0] == count + 1, "offsets must have one more element than counts");
    need((count == 1 || counts->strides[0] == 1) && offsets->strides[0] == 1, "offsets and counts must be contiguous");
    need(sources->sizes[0] >= (n + std::min(count, n) * (align - 1)) / align * align,
         "sources is too small: gpuos_order_rows says how many rows there can be");
    const gpuos_tensor* outs[4] = {places, sources, offsets, counts};
    for (int i = 0; i < 4; ++i) {
      no_overlap(*outs[i], *experts, "outputs must not overlap experts");
      for (int j = 0; j < i; ++j) no_overlap(*outs[i], *outs[j], "outputs overlap");
    }
    OrderArgs a{};
    a.experts = experts->data;
    a.wide = experts->dtype == GPUOS_I64;
    a.st = experts->strides[0];
    a.sk = experts->strides[1];
    a.plain = (a.sk == 1 || experts->sizes[1] == 1) && (a.st == experts->sizes[1] || experts->sizes[0] <= 1);
    a.places = static_cast<int32_t*>(places->data);
    a.sources = static_cast<int32_t*>(sources->data);
    a.offsets = static_cast<int32_t*>(offsets->data);
    a.counts = static_cast<int32_t*>(counts->data);
    a.k = FastDiv((uint32_t)experts->sizes[1]);
    a.n = (uint32_t)n;
    a.count = (uint32_t)count;
    a.align = (uint32_t)align;
    a.rows = (uint32_t)sources->sizes[0];
    const uint32_t steps = (a.n + 31) / 32;
    a.warps = std::min(std::min(32u, kCounts / a.count), std::max(steps, 4u));
    const uint32_t parts = steps <= 4 * a.warps ? 1 : std::min(kSortCluster, (steps + 4 * a.warps - 1) / (4 * a.warps));
    a.per_warp = (steps + parts * a.warps - 1) / (parts * a.warps) * 32;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3(parts);
    c.blockDim = dim3(a.warps * 32);
    c.dynamicSmemBytes = a.warps * a.count * sizeof(uint32_t);
    c.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {parts, 1, 1};
    c.attrs = at;
    c.numAttrs = 1;
    cuda_ok(cudaLaunchKernelEx(&c, gpuos_order_kernel, (const OrderArgs)a), "launch");
  });
}

extern "C" int32_t gpuos_dispatch(const gpuos_tensor* x, const gpuos_tensor* places, const gpuos_tensor* sources,
                                  const gpuos_tensor* rows, void* stream) {
  return entry("gpuos_dispatch", [&] {
    check_rows(x, "x");
    check_order(places, sources);
    check_rows(rows, "rows");
    need(x->dtype == rows->dtype, "x and rows must have one dtype");
    need(x->sizes[0] == places->sizes[0], "x must have the tokens of places");
    need(rows->sizes[0] == sources->sizes[0] && rows->sizes[1] == x->sizes[1], "rows must be (row of sources, element of x)");
    check_plain(rows, "rows");
    for (const gpuos_tensor* t : {x, places, sources}) no_overlap(*rows, *t, "rows must not overlap an input");
    if (numel(*rows) == 0) return;
    MoveArgs a = move(*places, *sources, *rows);
    const gpuos_tensor* both[2] = {x, rows};
    const int size = esize(x->dtype), bytes = pack_bytes(both, 2);
    cut(a, bytes, size, kUnroll);
    a.x = x->data;
    a.out = rows->data;
    a.xs = x->strides[0] / (bytes / size);
    const dim3 grid(blocks(a.units + (uint64_t)a.rows * a.chunks.d));
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bytes == 16) run(gpuos_dispatch_kernel<uint4>, grid, kThreads, 0, st, a);
    else if (bytes == 4) run(gpuos_dispatch_kernel<uint32_t>, grid, kThreads, 0, st, a);
    else run(gpuos_dispatch_kernel<uint16_t>, grid, kThreads, 0, st, a);
  });
}

extern "C" int32_t gpuos_combine(const gpuos_tensor* y, const gpuos_tensor* places, const gpuos_tensor* sources,
                                 const gpuos_tensor* weights, const gpuos_tensor* out, void* stream) {
  return entry("gpuos_combine", [&] {
    check_rows(y, "y");
    check_order(places, sources);
    if (weights) check_weights(weights, places);
    check_rows(out, "out");
    need(y->dtype == out->dtype, "y and out must have one dtype");
    need(y->sizes[0] == sources->sizes[0], "y must have the rows of sources");
    need(out->sizes[0] == places->sizes[0] && out->sizes[1] == y->sizes[1], "out must be (token of places, element of y)");
    check_plain(out, "out");
    for (const gpuos_tensor* t : {y, places, sources, weights})
      if (t) no_overlap(*out, *t, "out must not overlap an input");
    if (numel(*out) == 0) return;
    MoveArgs a = move(*places, *sources, *out);
    const gpuos_tensor* both[2] = {y, out};
    const int size = esize(y->dtype), bytes = pack_bytes(both, 2);
    cut(a, bytes, size, 2);
    a.x = y->data;
    a.out = out->data;
    a.xs = y->strides[0];
    if (weights) {
      a.w = static_cast<const float*>(weights->data);
      a.ws = weights->strides[0];
      a.wk = weights->strides[1];
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (y->dtype == GPUOS_F32) launch_combine<float>(a, bytes, st);
    else if (y->dtype == GPUOS_F16) launch_combine<__half>(a, bytes, st);
    else launch_combine<__nv_bfloat16>(a, bytes, st);
  });
}

extern "C" int32_t gpuos_combine_grad(const gpuos_tensor* grad, const gpuos_tensor* y, const gpuos_tensor* places,
                                      const gpuos_tensor* sources, const gpuos_tensor* weights, const gpuos_tensor* grad_y,
                                      const gpuos_tensor* grad_weights, void* stream) {
  return entry("gpuos_combine_grad", [&] {
    need(grad_y || grad_weights, "neither grad_y nor grad_weights is wanted");
    check_rows(grad, "grad");
    check_order(places, sources);
    check_weights(weights, places);
    need(grad->sizes[0] == places->sizes[0], "grad must have the tokens of places");
    const gpuos_tensor* t[3] = {grad};
    int n = 1;
    if (grad_weights) {
      check_rows(y, "y");
      need(y->dtype == grad->dtype, "grad and y must have one dtype");
      need(y->sizes[0] == sources->sizes[0] && y->sizes[1] == grad->sizes[1], "y must be (row of sources, element of grad)");
      check_tensor(grad_weights, 2, "grad_weights");
      need(grad_weights->dtype == GPUOS_F32, "grad_weights must be float32");
      same_sizes(*grad_weights, *places, "grad_weights must have the sizes of places");
      need(grad_weights->sizes[1] == 1 || grad_weights->strides[1] == 1, "grad_weights must be contiguous");
      check_plain(grad_weights, "grad_weights");
      t[n++] = y;
    }
    if (grad_y) {
      check_rows(grad_y, "grad_y");
      need(grad_y->dtype == grad->dtype, "grad and grad_y must have one dtype");
      need(grad_y->sizes[0] == sources->sizes[0] && grad_y->sizes[1] == grad->sizes[1], "grad_y must be (row of sources, element of grad)");
      check_plain(grad_y, "grad_y");
      t[n++] = grad_y;
    }
    for (const gpuos_tensor* o : {grad_y, grad_weights}) {
      if (!o) continue;
      for (const gpuos_tensor* i : {grad, grad_weights ? y : nullptr, places, sources, weights})
        if (i) no_overlap(*o, *i, "an output must not overlap an input");
    }
    if (grad_y && grad_weights) no_overlap(*grad_y, *grad_weights, "outputs overlap");
    const uint32_t rows = grad_y && grad->sizes[1] ? (uint32_t)sources->sizes[0] : 0;
    if (places->sizes[0] == 0 && rows == 0) return;
    MoveArgs a = move(*places, *sources, *grad);
    const int size = esize(grad->dtype), bytes = pack_bytes(t, n);
    cut(a, bytes, size, kUnroll);
    a.rows = (uint32_t)sources->sizes[0];
    a.g = grad->data;
    a.gs = grad->strides[0];
    a.w = static_cast<const float*>(weights->data);
    a.ws = weights->strides[0];
    a.wk = weights->strides[1];
    if (grad_weights) {
      a.x = y->data;
      a.xs = y->strides[0];
      a.gw = static_cast<float*>(grad_weights->data);
    }
    if (grad_y) a.out = grad_y->data;
    const uint32_t extra = rows ? std::min(blocks((uint64_t)rows * a.chunks.d), 65536u) : 0;
    need((uint64_t)a.tokens + extra < (1ull << 31), "the call is too large");
    const dim3 grid(a.tokens + extra);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (grad->dtype == GPUOS_F32) launch_grad<float>(a, bytes, grid, st);
    else if (grad->dtype == GPUOS_F16) launch_grad<__half>(a, bytes, grid, st);
    else launch_grad<__nv_bfloat16>(a, bytes, grid, st);
  });
}
