// gpuos_verify: drafted tokens d_0 .. d_(n-1) of a sequence checked against the
// target's n + 1 rows of logits x from given random numbers u_0 .. u_n, and the
// next token drawn.  With temperature t, m_i = max x_i,
//
//   w_ij = e^((x_ij - m_i) / t)      S_i = sum_j w_ij      p_ij = w_ij / S_i
//
// draft i is accepted where u_i q_i(d_i) S_i < w_i(d_i) (q: the draft's
// probabilities; 1 at d_i where none are given).  At the first that is not, a, the
// next token is drawn from r_j = max(w_aj - q_aj S_a, 0), or from w_a where
// that leaves nothing; where all are accepted, from r = w_n: the lowest j with
//
//   sum_(i <= j) r_i  >  u_n sum_i r_i
//
// which gives tokens as the target alone would.  t = 0 takes the likeliest token instead.
// Counts and tokens are those of 64-bit arithmetic.  A cluster takes a sequence, so
// that nothing but its tokens leaves it:
//   1. every row is read once for m_i and S_i in 32 bits, whose error is below 2^-13;
//   2. a draft for which that could matter has S_i summed again in 64 bits;
//   3. the one row that is drawn from is read again (from L2) and summed in 64 bits:
//      an SM's 64-bit rate is half its 32-bit rate, and it is one row of a sequence.
// Reading all rows is the bound at many long rows; else the chain of 3 to 5 steps that the cluster
// takes together, whose exponentials are by a table (10 instructions of 64 bits each, where exp()
// takes twice as many) and whose sums are kept a lane, so that the token is found without a third pass.
// 32 sequences x 8 rows x 128257 bf16 with probabilities: 60 to 69 us (129 with exp() and one CTA an SM), where reading
// takes 13; 64 x 50257 fp32 drawn: 18; 1 x 5 x 32000: 14.
#include <cooperative_groups.h>

#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

namespace cg = cooperative_groups;

constexpr uint32_t kThreads = 256, kWarps = kThreads / 32;
constexpr uint32_t kCluster = 8;
constexpr uint32_t kKept = 16;             // steps of a warp whose lanes' sums are kept
constexpr uint32_t kMaxDrafts = 63;
constexpr uint32_t kMaxTokens = 1u << 24;  // of a row
constexpr int kPack = 8;                   // elements a lane takes at once
// Packs a lane has in flight: 128 bytes.  (32 x 8 x 128257 bf16 with probabilities: 65 us with half of that.)
template <typename T> constexpr int kFlight = 16 / sizeof(T);
constexpr float kLowest = -3.402823466e38f;

struct VerifyArgs {
  const void* x;
  int64_t xs, xr;       // strides of sequence and row
  const void* drafts;
  int64_t ds, di;
  const float* u;
  int64_t us, ui;
  const void* q;        // may be NULL
  int64_t qs, qr;
  int64_t* tokens;      // (sequence, n + 1)
  int64_t* accepted;
  uint32_t n, cols;
  uint32_t groups;      // of a CTA's warps, a row each at a time: 1, 2, 4 or 8
  double k64;           // 64 log2(e) / t
  float k2;             // log2(e) / t
  int draft_wide, greedy, q_type;
};

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

template <typename T>
struct alignas(16) Elements {
  T v[kPack];
};

// A row as packs of 8 elements that start on 16 bytes (of 16-bit elements; 32 of 32-bit ones): the first and the last
// may lie partly outside the row.
template <typename T>
struct Row {
  const T* x;
  uint32_t cols, shift;  // elements of the first pack that are before the row
  __device__ Row(const T* p, uint32_t n)
      : x(p), cols(n), shift((uint32_t)(reinterpret_cast<uintptr_t>(p) % (kPack * sizeof(T)) / sizeof(T))) {}
  __device__ uint32_t packs() const { return (cols + shift + kPack - 1) / kPack; }
  // the 8 elements from `first()` of pack p on; -inf outside the row
  __device__ int64_t first(uint32_t p) const { return (int64_t)p * kPack - shift; }
  __device__ void load(uint32_t p, Elements<T>& v) const {
    const int64_t e = first(p);
    if (e >= 0 && e + kPack <= cols) {
      constexpr int W = 16 / sizeof(T);
#pragma unroll
      for (int k = 0; k < kPack; k += W) *reinterpret_cast<Pack<T, W>*>(&v.v[k]) = load_pack<T, W, false>(x + e + k);
    } else {
#pragma unroll
      for (int i = 0; i < kPack; ++i) v.v[i] = e + i >= 0 && e + i < cols ? x[e + i] : from_f<T>(-INFINITY);
    }
  }
  __device__ void load(uint32_t p, float (&v)[kPack]) const {
    Elements<T> q;
    load(p, q);
#pragma unroll
    for (int i = 0; i < kPack; ++i) v[i] = to_f(q.v[i]);
  }
};

__device__ __forceinline__ float prob(const void* q, int type, int64_t i) {
  if (type == GPUOS_F32) return __ldg(static_cast<const float*>(q) + i);
  if (type == GPUOS_F16) return to_f(static_cast<const __half*>(q)[i]);
  return to_f(static_cast<const __nv_bfloat16*>(q)[i]);
}

// An integer that orders as (x, lowest index first) does.
__device__ __forceinline__ unsigned long long key_of(float x, uint32_t index) {
  const uint32_t b = __float_as_uint(x + 0.f);
  const uint32_t k = (b >> 31) ? ~b : b | 0x80000000u;
  return ((unsigned long long)k << 32) | (uint32_t)~index;
}

// A row's maximum, and its sum in units of e^(maximum / t); greedy: the key of the likeliest token, and NaN where there is no such.
struct Stat {
  float m, s;
  unsigned long long key;
};

__device__ __forceinline__ void join(Stat& a, const Stat& b, float k2) {
  const float m = fmaxf(a.m, b.m);
  a.s = a.s * ex2(fmaxf((a.m - m) * k2, -1e4f)) + b.s * ex2(fmaxf((b.m - m) * k2, -1e4f));
  a.m = m;
  a.key = max(a.key, b.key);
}

// (the sum in units of e^(maximum / t) of one maximum)
__device__ __forceinline__ Stat join_warp(Stat v, float k2) {
  float m;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v.m));
  v.s *= ex2(fmaxf((v.m - m) * k2, -1e4f));
  v.m = m;
#pragma unroll
  for (int d = 16; d; d >>= 1) v.s += __shfl_xor_sync(~0u, v.s, d);
  return v;
}
__device__ __forceinline__ unsigned long long max_warp(unsigned long long v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v = max(v, __shfl_xor_sync(~0u, v, d));
  return v;
}

// The largest of 8 elements (16-bit ones two at a time; a NaN does not count).
template <typename T>
__device__ __forceinline__ float largest(const Elements<T>& x) {
  if constexpr (sizeof(T) == 2) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* h = reinterpret_cast<const T2*>(&x);
    const T2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(to_f(m.x), to_f(m.y));
  } else {
    float m = x.v[0];
#pragma unroll
    for (int i = 1; i < kPack; ++i) m = fmaxf(m, x.v[i]);
    return m;
  }
}

// Sums over a warp, the same in all lanes.
__device__ __forceinline__ double sum_warp(double v) {
#pragma unroll
  for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

struct Shared {
  Stat part[kMaxDrafts + 1][kWarps];
  Stat mine[kMaxDrafts + 1];      // of this CTA, read by the others
  Stat all[kMaxDrafts + 1];
  double warp[kWarps];
  double sum[2];                  // of this CTA, read by the others (two, taken in turn)
  double power[64];               // 2^(i / 64)
  double kept[kWarps][kKept][32];
};

// e^(d / t) for d <= 0, in 64 bits: with d 64 log2(e) / t = 64 k + j + r, |r| <= 1/2 (Tang's table-driven
// reduction), 2^k 2^(j / 64) e^y, y = r ln 2 / 64, whose series ends at y^5 / 120 (the next term is below 4e-17).
__device__ __forceinline__ double power_of(double d, double k64, const double* table) {
  const double x = fmax(d * k64, -64.0 * 1020.0);  // (2^-1020 stays a normal number; it changes no sum)
  constexpr double kRound = 6755399441055744.0;    // 1.5 * 2^52: the sum's low bits are the nearest integer
  const double n = x + kRound;
  const int i = __double2loint(n);
  const double y = (x - (n - kRound)) * (0.69314718055994530942 / 64.0);
  double p = fma(y, 1.0 / 120.0, 1.0 / 24.0);
  p = fma(y, p, 1.0 / 6.0);
  p = fma(y, p, 0.5);
  p = fma(y, p, 1.0);
  const double t = table[i & 63];
  p = fma(y * p, t, t);
  return __hiloint2double(__double2hiint(p) + ((i >> 6) << 20), __double2loint(p));
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 3)
gpuos_verify_kernel(const __grid_constant__ VerifyArgs a) {
  extern __shared__ __align__(16) uint8_t room[];
  Shared& sh = *reinterpret_cast<Shared*>(room);
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t rank = cluster.block_rank(), parts = cluster.num_blocks();
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t seq = blockIdx.x / parts;
  const T* x0 = static_cast<const T*>(a.x) + seq * a.xs;
  const uint32_t rows = a.n + 1;
  if (threadIdx.x < 64) sh.power[threadIdx.x] = exp2((double)threadIdx.x / 64.0);

  // the packs of a row that this warp takes, neighbours
  auto share = [&](const Row<T>& r, uint32_t& lo, uint32_t& hi) {
    const uint32_t packs = r.packs(), each = (packs + parts * kWarps - 1) / (parts * kWarps);
    lo = min((rank * kWarps + warp) * each, packs);
    hi = min(lo + each, packs);
  };

  // 1. maxima and sums of all rows; short ones several at a time, a group of the CTA's warps each (a.groups of them)
  const uint32_t of_row = kWarps / a.groups;  // warps
  for (uint32_t i = warp / of_row; i < rows; i += a.groups) {
    const Row<T> row(x0 + i * a.xr, a.cols);
    const uint32_t packs = row.packs(), each = (packs + parts * of_row - 1) / (parts * of_row);
    const uint32_t lo = min((rank * of_row + warp % of_row) * each, packs), hi = min(lo + each, packs);
    Stat st{a.greedy ? -INFINITY : kLowest, 0.f, 0};
    bool odd = false;  // greedy: NaN or +inf seen
    constexpr int U = kFlight<T>;
    for (uint32_t p = lo + lane; p < hi; p += 32 * U) {
      Elements<T> v[U];
#pragma unroll
      for (int f = 0; f < U; ++f) {
        if (p + 32 * f < hi) {
          row.load(p + 32 * f, v[f]);
        } else {
#pragma unroll
          for (int c = 0; c < kPack; ++c) v[f].v[c] = from_f<T>(-INFINITY);
        }
      }
      float m = st.m;
#pragma unroll
      for (int f = 0; f < U; ++f) m = fmaxf(m, largest(v[f]));
      if (a.greedy) {
#pragma unroll
        for (int f = 0; f < U; ++f)
#pragma unroll
          for (int c = 0; c < kPack; ++c) {
            const float x = to_f(v[f].v[c]);
            odd |= !(x < INFINITY);
            if (x == m && m > st.m) st.key = max(st.key, key_of(m, (uint32_t)(row.first(p + 32 * f) + c)));
          }
        if (m > st.m) st.m = m;
        continue;
      }
      if (m > st.m) {
        st.s *= ex2(fmaxf((st.m - m) * a.k2, -1e4f));
        st.m = m;
      }
      float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (int f = 0; f < U; ++f)
#pragma unroll
        for (int c = 0; c < kPack; c += 2) {
          const float2 y = mul2(add2(make_float2(to_f(v[f].v[c]), to_f(v[f].v[c + 1])), both(-m)), both(a.k2));
          sum[f & 1] = add2(sum[f & 1], make_float2(ex2(y.x), ex2(y.y)));
        }
      sum[0] = add2(sum[0], sum[1]);
      st.s += sum[0].x + sum[0].y;
    }
    if (a.greedy) {
      st.key = max_warp(st.key);
      st.s = __any_sync(~0u, odd) ? NAN : 0.f;
    } else {
      st = join_warp(st, a.k2);
    }
    if (lane == 0) sh.part[i][warp % of_row] = st;
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < rows; i += kThreads) {
    Stat st = sh.part[i][0];
    for (uint32_t w = 1; w < of_row; ++w) join(st, sh.part[i][w], a.greedy ? 0.f : a.k2);
    sh.mine[i] = st;
  }
  cluster.sync();
  for (uint32_t i = threadIdx.x; i < rows; i += kThreads) {
    Stat st = *cluster.map_shared_rank(&sh.mine[i], 0);
    for (uint32_t c = 1; c < parts; ++c) join(st, *cluster.map_shared_rank(&sh.mine[i], c), a.greedy ? 0.f : a.k2);
    sh.all[i] = st;
  }
  __syncthreads();

  // From here on all threads of the cluster take the same way.
  uint32_t turn = 0;
  // the sum over the cluster of what the warps have; where this warp's share begins and ends in it (an end
  // is exactly the next one's beginning)
  auto sum_all = [&](double v, double& begin, double& end) {
    if (lane == 0) sh.warp[warp] = v;
    __syncthreads();
    double mine = 0.0, ahead = 0.0, until = 0.0;
#pragma unroll
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w == warp) ahead = mine;
      mine += sh.warp[w];
      if (w == warp) until = mine;
    }
    if (threadIdx.x == 0) sh.sum[turn & 1] = mine;
    cluster.sync();
    const double part = lane < parts ? *cluster.map_shared_rank(&sh.sum[turn & 1], lane) : 0.0;
    double total = 0.0, before = 0.0;
#pragma unroll
    for (uint32_t c = 0; c < kCluster; ++c) {
      if (c == rank) before = total;
      total += __shfl_sync(~0u, part, c);
    }
    begin = before + ahead;
    end = before + until;
    ++turn;
    return total;
  };
  auto weight = [&](float v, float m) {
    // a masked token, and one whose weight would leave 64 bits, has none
    const double w = power_of((double)v - m, a.k64, sh.power);
    return (double)(v - m) * a.k64 >= -64.0 * 1020.0 ? w : 0.0;
  };
  auto whole_sum = [&](uint32_t i) {
    const Row<T> row(x0 + i * a.xr, a.cols);
    uint32_t lo, hi;
    share(row, lo, hi);
    const float m = sh.all[i].m;
    double s = 0.0, unused;
    for (uint32_t p = lo + lane; p < hi; p += 32) {
      float v[kPack];
      row.load(p, v);
#pragma unroll
      for (int c = 0; c < kPack; ++c) s += weight(v[c], m);
    }
    return sum_all(sum_warp(s), unused, unused);
  };
  auto draft = [&](uint32_t i) { return load_index(a.drafts, a.draft_wide, seq * a.ds + i * a.di); };
  auto valid = [&](uint32_t i) {
    const Stat& st = sh.all[i];
    return a.greedy ? st.s == 0.f && st.key != 0 : st.s > 0.f && st.s < INFINITY && st.m < INFINITY;
  };

  // 2. drafts from the first on, until one is refused or there is none
  uint32_t at = 0;
  bool refused = false;
  for (; at < a.n; ++at) {
    const int64_t d = draft(at);
    if (d < 0 || d >= a.cols) break;  // the drafts end here
    if (!valid(at)) {
      refused = true;
      break;
    }
    if (a.greedy) {
      refused = d != (uint32_t)~(uint32_t)sh.all[at].key;
    } else {
      const double w = exp(((double)to_f(x0[at * a.xr + d]) - sh.all[at].m) * (a.k64 / (64.0 * 1.44269504088896340736)));
      const double q = a.q ? (double)prob(a.q, a.q_type, seq * a.qs + at * a.qr + d) : 1.0;
      const double uq = (double)__ldg(a.u + seq * a.us + at * a.ui) * q;
      double bound = uq * sh.all[at].s;
      // the sum's error, in roundings (2^-24): at most 8 + 256 additions in a thread, whose maximum may rise as often as it
      // takes packs, 256 times, of 5 each (an exponential of 2^-22 and a product), 29 joins of 6, an exponential of 4, and of the
      // exponents' arguments 1.8 times the sum of w |log2 w| / S, at most log2 of the tokens (those of the rises add up to one
      // argument): 1770 together, below 2^-13
      if (fabs(bound - w) <= 0x1p-12 * w && w > 0.0) bound = uq * whole_sum(at);
      refused = !(bound < w);
    }
    if (refused) break;
  }

  // 3. the next token
  int64_t* out = a.tokens + seq * rows;
  if (rank == 0) {
    for (uint32_t i = threadIdx.x; i < rows; i += kThreads)
      if (i != at || !valid(at) || a.greedy)
        out[i] = i < at ? draft(i) : i == at && valid(at) ? (int64_t)(uint32_t)~(uint32_t)sh.all[at].key : -1;
    if (threadIdx.x == 0) a.accepted[seq] = at;
  }
  if (a.greedy || !valid(at)) {
    cluster.sync();  // no CTA leaves while another reads its `mine`
    return;
  }
  const Row<T> row(x0 + at * a.xr, a.cols);
  uint32_t lo, hi;
  share(row, lo, hi);
  const float m = sh.all[at].m;
  const int64_t gone = refused && !a.q ? draft(at) : -1;   // the draft itself, where it had all
  const double total_w = refused && a.q ? whole_sum(at) : 0.0;
  bool less = refused;
  auto weights = [&](uint32_t p, double (&r)[kPack]) {
    float v[kPack], q[kPack];
    const int64_t e = row.first(p);
    if (less && a.q) {
#pragma unroll
      for (int c = 0; c < kPack; ++c)
        q[c] = e + c >= 0 && e + c < a.cols ? prob(a.q, a.q_type, seq * a.qs + at * a.qr + e + c) : 0.f;
    }
    row.load(p, v);
#pragma unroll
    for (int c = 0; c < kPack; ++c) {
      r[c] = weight(v[c], m);
      if (!less) continue;
      if (!a.q) {
        if (e + c == gone) r[c] = 0.0;
      } else {
        const double rest = r[c] - (double)q[c] * total_w;
        r[c] = rest > 0.0 ? rest : 0.0;  // (a NaN leaves nothing)
      }
    }
  };
  const bool kept = hi - lo <= 32 * kKept;
  double begin, end, total;
  for (;;) {
    double s = 0.0;
    uint32_t k = 0;
    for (uint32_t p = lo + lane; p < hi; p += 32, ++k) {
      double r[kPack], one = 0.0;
      weights(p, r);
#pragma unroll
      for (int c = 0; c < kPack; ++c) one += r[c];
      if (kept) sh.kept[warp][k][lane] = one;
      s += one;
    }
    total = sum_all(sum_warp(s), begin, end);
    if (total > 0.0 || !less) break;
    less = false;
  }
  double u = (double)__ldg(a.u + seq * a.us + a.n * a.ui);
  u = u > 0.0 ? u : 0.0;
  double goal = u * total;
  if (!(goal < total)) goal = __longlong_as_double(__double_as_longlong(total) - 1);
  if (begin <= goal && goal < end) {  // one warp of the cluster
    double run = begin;
    int64_t found = -1, last = -1;
    uint32_t k = 0;
    for (uint32_t p0 = lo; p0 < hi && found < 0; p0 += 32, ++k) {
      const uint32_t p = p0 + lane;
      double r[kPack], s = 0.0;
      if (p < hi) {
        if (kept) {
          s = sh.kept[warp][k][lane];
        } else {
          weights(p, r);
#pragma unroll
          for (int c = 0; c < kPack; ++c) s += r[c];
        }
      }
      double sum = s;
#pragma unroll
      for (uint32_t d = 1; d < 32; d <<= 1) {
        const double o = __shfl_up_sync(~0u, sum, d);
        if (lane >= d) sum += o;
      }
      // the first lane whose sum passes the goal (else the last with any: the sums of step 3 rounded in another
      // order); of its elements the first that does, or the last with any weight
      const uint32_t past = __ballot_sync(~0u, run + sum > goal && s > 0.0);
      const uint32_t some = __ballot_sync(~0u, s > 0.0);
      const double ahead = run + (sum - s);
      run += __shfl_sync(~0u, sum, 31);
      if (!past && (!some || p0 + 32 < hi)) {
        if (some) last = p0 + 31 - __clz(some);  // (a pack)
        continue;
      }
      const uint32_t who = past ? __ffs(past) - 1 : 31 - __clz(some);
      found = p0 + who;
      double acc = __shfl_sync(~0u, ahead, who);
      weights((uint32_t)found, r);
      int64_t pick = -1, high = -1;
#pragma unroll
      for (int c = 0; c < kPack; ++c) {
        acc += r[c];
        if (r[c] > 0.0) high = row.first((uint32_t)found) + c;
        if (r[c] > 0.0 && pick < 0 && acc > goal) pick = high;
      }
      if (lane == 0) out[at] = pick >= 0 ? pick : high;
    }
    if (found < 0) {  // the last steps had nothing: the last weight of the warp's share
      double r[kPack];
      weights((uint32_t)last, r);
      int64_t high = -1;
#pragma unroll
      for (int c = 0; c < kPack; ++c)
        if (r[c] > 0.0) high = row.first((uint32_t)last) + c;
      if (lane == 0) out[at] = high;
    }
  }
  cluster.sync();  // no CTA leaves while another reads its sums
}

}  // namespace
}  // namespace rowops
}  // namespace gpuos

using namespace gpuos::rowops;

extern "C" int32_t gpuos_verify(const gpuos_tensor* logits, const gpuos_tensor* drafts, const gpuos_tensor* uniforms,
                                const gpuos_tensor* probs, const gpuos_tensor* tokens, const gpuos_tensor* accepted,
                                double temperature, void* stream) {
  return entry("gpuos_verify", [&] {
    check_tensor(logits, 3, "logits");
    need(is_real(logits->dtype), "logits must be float32, float16 or bfloat16");
    const int64_t b = logits->sizes[0], rows = logits->sizes[1], v = logits->sizes[2];
    need(rows >= 1 && rows <= (int64_t)kMaxDrafts + 1, "logits must be (sequence, draft + 1, token) with at most 63 drafts");
    need(v >= 1 && v < kMaxTokens, "logits must have between 1 and 2^24 - 1 tokens a row");
    need(v == 1 || logits->strides[2] == 1, "logits: the last dim must be contiguous");
    // (k2 stays a 32-bit number)
    need(temperature == 0.0 || (temperature >= 1e-30 && temperature <= 1e30), "temperature must be 0, or in [1e-30, 1e30]");
    check_tensor(drafts, 2, "drafts");
    need(is_index(drafts->dtype), "drafts must be int32 or int64");
    need(drafts->sizes[0] == b && drafts->sizes[1] == rows - 1, "drafts must be (sequence, draft), one less than logits has rows");
    const bool greedy = temperature == 0.0;
    if (!greedy) need(uniforms != nullptr, "uniforms are needed (but for temperature 0)");
    if (uniforms) {
      check_tensor(uniforms, 2, "uniforms");
      need(uniforms->dtype == GPUOS_F32, "uniforms must be float32");
      need(uniforms->sizes[0] == b && uniforms->sizes[1] == rows, "uniforms must be (sequence, draft + 1)");
    }
    if (probs) {
      check_tensor(probs, 3, "probs");
      need(is_real(probs->dtype), "probs must be float32, float16 or bfloat16");
      need(probs->sizes[0] == b && probs->sizes[1] == rows - 1 && probs->sizes[2] == v, "probs must be (sequence, draft, token)");
      need(v == 1 || probs->sizes[1] == 0 || probs->strides[2] == 1, "probs: the last dim must be contiguous");
    }
    check_tensor(tokens, 2, "tokens");
    check_tensor(accepted, 1, "accepted");
    need(tokens->dtype == GPUOS_I64 && accepted->dtype == GPUOS_I64, "tokens and accepted must be int64");
    need(tokens->sizes[0] == b && tokens->sizes[1] == rows, "tokens must be (sequence, draft + 1)");
    need(accepted->sizes[0] == b, "accepted must be [sequence]");
    need((rows == 1 || tokens->strides[1] == 1) && (b <= 1 || tokens->strides[0] == rows), "tokens must be contiguous");
    need(b <= 1 || accepted->strides[0] == 1, "accepted must be contiguous");
    for (const gpuos_tensor* o : {tokens, accepted})
      for (const gpuos_tensor* i : {logits, drafts, uniforms, probs})
        if (i) no_overlap(*o, *i, "an output must not overlap an input");
    no_overlap(*tokens, *accepted, "outputs overlap");
    need(b < (1ll << 27), "too many sequences");
    if (b == 0) return;
    VerifyArgs a{};
    a.x = logits->data;
    a.xs = logits->strides[0];
    a.xr = logits->strides[1];
    a.drafts = drafts->data;
    a.draft_wide = drafts->dtype == GPUOS_I64;
    a.ds = drafts->strides[0];
    a.di = drafts->strides[1];
    if (!greedy) {
      a.u = static_cast<const float*>(uniforms->data);
      a.us = uniforms->strides[0];
      a.ui = uniforms->strides[1];
      a.k64 = 64.0 * 1.44269504088896340736 / temperature;
      a.k2 = (float)(1.44269504088896340736 / temperature);
    }
    if (probs && rows > 1 && !greedy) {
      a.q = probs->data;
      a.q_type = probs->dtype;
      a.qs = probs->strides[0];
      a.qr = probs->strides[1];
    }
    a.tokens = static_cast<int64_t*>(tokens->data);
    a.accepted = static_cast<int64_t*>(accepted->data);
    a.n = (uint32_t)rows - 1;
    a.cols = (uint32_t)v;
    a.greedy = greedy;
    // CTAs of a sequence: as few as keep their lanes' sums (and the bound on sums in 32 bits); of few sequences
    // more, with a pack for every thread at least, as long as all run at once (64 x 50257 fp32 drawn: 19 us, 25 with twice as many)
    uint32_t parts = 1;
    while (parts < kCluster && (uint64_t)parts * kThreads * kPack < (uint64_t)v &&
           (2 * (uint64_t)b * parts <= 3u * (uint32_t)sm_count() || (uint64_t)parts * kWarps * kKept * 32 * kPack < (uint64_t)v + kPack))
      parts *= 2;
    // so many that a warp's share of a row fills what it has in flight
    const uint32_t flight = 32 * (logits->dtype == GPUOS_F32 ? kFlight<float> : kFlight<__half>) * kPack;
    a.groups = 1;
    while (a.groups < kWarps && a.groups < rows && 2 * a.groups * (uint64_t)v <= (uint64_t)flight * parts * kWarps) a.groups *= 2;
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((uint32_t)b * parts);
    c.blockDim = dim3(kThreads);
    c.dynamicSmemBytes = sizeof(Shared);
    c.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim = {parts, 1, 1};
    c.attrs = at;
    c.numAttrs = 1;
    const VerifyArgs args = a;
    auto go = [&](auto* kernel) {
      static_assert(sizeof(Shared) <= 48 << 10);
      cuda_ok(cudaLaunchKernelEx(&c, kernel, args), "launch");
    };
    if (logits->dtype == GPUOS_F32) go(gpuos_verify_kernel<float>);
    else if (logits->dtype == GPUOS_F16) go(gpuos_verify_kernel<__half>);
    else go(gpuos_verify_kernel<__nv_bfloat16>);
  });
}
