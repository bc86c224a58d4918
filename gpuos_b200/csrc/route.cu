// gpuos_route / gpuos_route_grad: routing of tokens to experts.
//
//   s    = softmax(x) or sigmoid(x)          over a token's E logits
//   key  = s + bias                          (without a bias: x, which orders as s does)
//   groups of E / groups neighbours: a group is worth its largest key, or the sum of its two
//   largest; the best `top_groups` stay open
//   top_k largest keys of the open groups; of equal ones the lowest index
//   w    = s of the chosen (/ their sum) * scale
//
// The chosen experts are those of exact arithmetic.  Keys are computed in 32
// bits with a known error bound; where two keys whose order matters are closer
// than the bound (and not of equal inputs), the token is done again in 64 bits.
//
// A token belongs to LPT lanes of a warp, each holding NPL neighbouring experts
// in registers: up to 256 experts take 8 a lane and as many lanes as needed, so
// that one warp serves up to 8 tokens of few experts.  Rounds of maximum over
// the lanes pick the experts; a lane's experts are neighbours, so the first
// lane that holds the maximum holds the lowest index.
#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 64;
constexpr int kMaxGroups = 64;

struct RouteArgs {
  const void* x;
  const float* bias;
  float* weights;
  void* experts;
  const float* gw;     // gradient: of the weights
  void* gx;            // gradient: of the logits
  int64_t xs, ws, wk, es, ek, bs, gs, gk, os;  // strides: row of x; row and rank of weights, experts, gw; bias; row of gx
  int64_t tokens;
  uint32_t n;          // experts
  uint32_t top_k, groups, top_groups;
  FastDiv per_group;
  float scale;
  int sigmoid, renorm, top2, wide, vec;
};

template <typename R> struct Num;
template <> struct Num<float> {
  using Key = uint32_t;
  static __device__ __forceinline__ float exp_(float x) { return expf(x); }
  // An unsigned integer that orders as x does; NaN as -inf; never 0.
  static __device__ __forceinline__ Key key(float x) {
    if (x != x) x = -INFINITY;
    const uint32_t b = __float_as_uint(x + 0.f);
    return (b >> 31) ? ~b : b | 0x80000000u;
  }
  static __device__ __forceinline__ float value(Key k) {
    return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
  }
};
template <> struct Num<double> {
  using Key = unsigned long long;
  static __device__ __forceinline__ double exp_(double x) { return exp(x); }
  static __device__ __forceinline__ Key key(double x) {
    if (x != x) x = -INFINITY;
    const Key b = (Key)__double_as_longlong(x + 0.0);
    return (b >> 63) ? ~b : b | (1ull << 63);
  }
  static __device__ __forceinline__ double value(Key k) {
    return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k));
  }
};

template <int LPT, typename V>
__device__ __forceinline__ V lanes_max(V v) {
#pragma unroll
  for (int d = LPT / 2; d; d >>= 1) {
    const V o = __shfl_xor_sync(~0u, v, d);
    v = o > v ? o : v;
  }
  return v;
}

template <int LPT, typename V>
__device__ __forceinline__ V lanes_sum(V v) {
#pragma unroll
  for (int d = LPT / 2; d; d >>= 1) v += __shfl_xor_sync(~0u, v, d);
  return v;
}

// A lane's NPL logits from `at` on; those from n on are -inf.
template <typename T, int NPL>
__device__ __forceinline__ void load_logits(const T* row, uint32_t at, uint32_t n, bool vec, bool live,
                                            float (&x)[NPL]) {
  constexpr int W = 16 / sizeof(T) < NPL ? 16 / sizeof(T) : NPL;
  if (vec) {
#pragma unroll
    for (int k = 0; k < NPL; k += W) {
      Pack<T, W> q;
      const bool in = live && at + k < n;
      if (in) q = load_pack<T, W>(row + at + k);
#pragma unroll
      for (int i = 0; i < W; ++i) x[k + i] = in ? to_f(q.v[i]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) x[i] = live && at + i < n ? to_f(row[at + i]) : -INFINITY;
  }
}

// Scores of a lane's experts in R; a row without a finite maximum below NaN
// has scores 0 (nothing is left by its mask).
template <typename R, int NPL, int LPT>
__device__ __forceinline__ void score(const float (&x)[NPL], uint32_t at, uint32_t n, bool sigmoid, R (&s)[NPL],
                                      float* top, R* total) {
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) s[i] = at + i < n ? R(1) / (R(1) + Num<R>::exp_(-(R)x[i])) : R(0);
    return;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NPL; ++i) m = fmaxf(m, x[i]);
  m = lanes_max<LPT>(m);
  R sum = 0;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    // NaN stays: one makes the whole row's scores NaN
    s[i] = (m == -INFINITY && x[i] == -INFINITY) ? R(0) : Num<R>::exp_((R)x[i] - (R)m);
    sum += s[i];
  }
  sum = lanes_sum<LPT>(sum);
  const R inv = sum == R(0) ? R(0) : R(1) / sum;
#pragma unroll
  for (int i = 0; i < NPL; ++i) s[i] *= inv;
  *top = m;
  *total = sum;
}

template <int LPT> constexpr uint32_t kLanes = LPT == 32 ? ~0u : (1u << (LPT & 31)) - 1;

struct Chosen {
  float score;
  uint32_t expert;
};

// One token's selection in R.  Returns whether 32-bit keys leave the order in
// doubt (always false in 64 bits).
template <typename R, int NPL, int LPT>
__device__ __forceinline__ bool select(const RouteArgs& a, const float (&x)[NPL], const float (&bias)[NPL],
                                       uint32_t lane, uint32_t base_lane, R (&s)[NPL], double* worth,
                                       Chosen* chosen) {
  using Key = typename Num<R>::Key;
  constexpr bool kWide = sizeof(R) == 8;
  const uint32_t at = lane * NPL;
  float m = 0.f;
  R total = 0;
  score<R, NPL, LPT>(x, at, a.n, a.sigmoid, s, &m, &total);
  Key key[NPL];
  const bool keyed = a.bias != nullptr;
#pragma unroll
  for (int i = 0; i < NPL; ++i)
    key[i] = at + i < a.n ? Num<R>::key(keyed ? s[i] + (R)bias[i] : (R)x[i]) : Key(0);
  bool doubt = false;

  if (a.groups > 1) {
    // with the sum of two the scores themselves count, not the logits
    for (uint32_t g = 0; g < a.groups; ++g) {
      const uint32_t lo = g * a.per_group.d, hi = lo + a.per_group.d;
      Key k1 = 0;
      uint32_t first = ~0u;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (at + i >= lo && at + i < hi && key[i] > k1) {
          k1 = key[i];
          first = i;
        }
      const Key best = lanes_max<LPT>(k1);
      R v = keyed || !a.top2 ? Num<R>::value(best) : R(0);
      if (a.top2) {
        const uint32_t has = __ballot_sync(~0u, k1 == best && first != ~0u) >> base_lane;
        const uint32_t owner = __ffs(has & kLanes<LPT>) - 1;
        Key k2 = 0;
        R s1 = 0, s2 = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (at + i >= lo && at + i < hi) {
            if (lane == owner && i == (int)first) s1 = s[i];
            else if (key[i] > k2) {
              k2 = key[i];
              s2 = s[i];
            }
          }
        const Key second = lanes_max<LPT>(k2);
        if (keyed) {
          v += second ? Num<R>::value(second) : R(0);
        } else {
          // the scores of the two (equal keys have equal scores)
          s2 = second && k2 == second ? s2 : R(0);
          v = lanes_max<LPT>(s1) + lanes_max<LPT>(s2);
        }
      }
      if (lane == 0) worth[g] = (double)v;
    }
    __syncwarp();
    // a group stays open where fewer than top_groups are better, or as good and before it
    double in = INFINITY, out = -INFINITY;  // the worst open one and the best closed one
    unsigned long long open = 0;
    for (uint32_t g = lane; g < a.groups; g += LPT) {
      const auto mine = Num<double>::key(worth[g]);
      uint32_t before = 0;
      for (uint32_t h = 0; h < a.groups; ++h) {
        const auto other = Num<double>::key(worth[h]);
        before += other > mine || (other == mine && h < g);
      }
      if (before < a.top_groups) {
        open |= 1ull << g;
        in = fmin(in, worth[g]);
      } else {
        out = fmax(out, worth[g]);
      }
    }
#pragma unroll
    for (int d = LPT / 2; d; d >>= 1) open |= __shfl_xor_sync(~0u, open, d);
    if (!kWide && (keyed || a.top2)) {
      in = -lanes_max<LPT>(-in);
      out = lanes_max<LPT>(out);
      // each worth is off by at most 20 * 2^-24 of its scores (at most 2) and 2 * 2^-24 of itself
      if (!(in - out > 5e-6 + 5e-7 * fabs(in))) doubt = true;
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (!((open >> a.per_group.div(at + i)) & 1)) key[i] = 0;
    __syncwarp();
  }

  Key mine = 0;
#pragma unroll
  for (int i = 0; i < NPL; ++i) mine = key[i] > mine ? key[i] : mine;
  float before_key = INFINITY, before_s = 0.f, before_x = 0.f, before_b = 0.f;
  const bool check = !kWide && keyed;
  for (uint32_t r = 0; r <= a.top_k; ++r) {
    if (r == a.top_k && !check) break;
    const Key best = lanes_max<LPT>(mine);
    const uint32_t has = __ballot_sync(~0u, mine == best) >> base_lane;
    const uint32_t owner = __ffs(has & kLanes<LPT>) - 1;
    float sc = 0.f, xx = 0.f, bb = 0.f;
    uint32_t e = 0;
    if (lane == owner) {
      bool found = false;
      Key next = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        if (!found && key[i] == best) {
          found = true;
          sc = (float)s[i];
          xx = x[i];
          bb = bias[i];
          e = at + i;
          key[i] = 0;
        }
        next = key[i] > next ? key[i] : next;
      }
      mine = next;
      if (r < a.top_k) chosen[r] = Chosen{sc, e};
    }
    if (check) {
      const uint32_t from = base_lane + owner;
      sc = __shfl_sync(~0u, sc, from);
      xx = __shfl_sync(~0u, xx, from);
      bb = __shfl_sync(~0u, bb, from);
      const float k = Num<float>::value((uint32_t)best);
      // each key is off by at most 10 * 2^-24 of its score and 2^-24 of itself; equal inputs tie exactly
      if (best != 0 && r > 0 && !(before_key - k > 1.25e-6f * fmaxf(sc, before_s) + 2.5e-7f * fabsf(k)) &&
          !(xx == before_x && bb == before_b))
        doubt = true;
      before_key = k;
      before_s = sc;
      before_x = xx;
      before_b = bb;
    }
  }
  __syncwarp();
  return doubt;
}

template <typename T, int NPL, int LPT>
__global__ void __launch_bounds__(kThreads)
gpuos_route_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr uint32_t kTokens = kThreads / LPT;  // tokens a CTA handles at once
  const uint32_t sub = threadIdx.x / LPT, lane = threadIdx.x % LPT, base_lane = (threadIdx.x & 31) - lane;
  double* worth = reinterpret_cast<double*>(smem) + sub * (a.groups > 1 ? a.groups : 0);
  Chosen* chosen = reinterpret_cast<Chosen*>(reinterpret_cast<double*>(smem) +
                                             kTokens * (a.groups > 1 ? a.groups : 0)) + sub * a.top_k;
  const uint32_t at = lane * NPL;
  float bias[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i) bias[i] = a.bias && at + i < a.n ? __ldg(a.bias + (at + i) * a.bs) : 0.f;
  for (int64_t t0 = (int64_t)blockIdx.x * kTokens; t0 < a.tokens; t0 += (int64_t)gridDim.x * kTokens) {
    const int64_t t = t0 + sub;
    const bool live = t < a.tokens;
    float x[NPL];
    load_logits<T, NPL>(static_cast<const T*>(a.x) + (live ? t * a.xs : 0), at, a.n, a.vec, live, x);
    bool doubt;
    {
      float s[NPL];
      doubt = select<float, NPL, LPT>(a, x, bias, lane, base_lane, s, worth, chosen);
    }
    if (__any_sync(~0u, doubt)) {
      double s[NPL];
      select<double, NPL, LPT>(a, x, bias, lane, base_lane, s, worth, chosen);
    }
    float total = 1.f;
    if (a.renorm) {
      total = 0.f;
      for (uint32_t r = 0; r < a.top_k; ++r) total += chosen[r].score;
    }
    const float by = total == 0.f ? 0.f : a.scale / total;
    if (live)
      for (uint32_t r = lane; r < a.top_k; r += LPT) {
        a.weights[t * a.ws + r * a.wk] = a.renorm ? chosen[r].score * by : chosen[r].score * a.scale;
        if (a.wide) static_cast<int64_t*>(a.experts)[t * a.es + r * a.ek] = chosen[r].expert;
        else static_cast<int32_t*>(a.experts)[t * a.es + r * a.ek] = (int32_t)chosen[r].expert;
      }
    __syncwarp();
  }
}

// The gradient of the weights through the chosen scores:
//   renormalised, S the sum of the chosen:  ds_j = scale (g_j - sum_i g_i s_i / S) / S,  else scale g_j
//   sigmoid:  dx_j = ds_j s_j (1 - s_j)
//   softmax:  dx_e = s_e (ds_e - sum_i ds_i s_i)        (ds = 0 where not chosen)
template <typename T, int NPL, int LPT>
__global__ void __launch_bounds__(kThreads)
gpuos_route_grad_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr uint32_t kTokens = kThreads / LPT;
  const uint32_t sub = threadIdx.x / LPT, lane = threadIdx.x % LPT;
  float* dense = reinterpret_cast<float*>(smem) + sub * (LPT * NPL);
  Chosen* chosen = reinterpret_cast<Chosen*>(reinterpret_cast<float*>(smem) + kThreads * NPL) + sub * a.top_k;
  const uint32_t at = lane * NPL;
  for (int64_t t0 = (int64_t)blockIdx.x * kTokens; t0 < a.tokens; t0 += (int64_t)gridDim.x * kTokens) {
    const int64_t t = t0 + sub;
    const bool live = t < a.tokens;
    const T* row = static_cast<const T*>(a.x) + (live ? t * a.xs : 0);
    float x[NPL], s[NPL];
    load_logits<T, NPL>(row, at, a.n, a.vec, live, x);
    float m = 0.f, total = 1.f;
    score<float, NPL, LPT>(x, at, a.n, a.sigmoid, s, &m, &total);
    // the chosen ones' scores and gradients, a lane each
    float sum = 0.f, dot = 0.f;
    for (uint32_t r = lane; r < a.top_k; r += LPT) {
      int64_t e = -1;
      if (live)
        e = a.wide ? static_cast<const int64_t*>(a.experts)[t * a.es + r * a.ek]
                   : (int64_t)static_cast<const int32_t*>(a.experts)[t * a.es + r * a.ek];
      const bool in = e >= 0 && e < a.n;
      const float g = in ? a.gw[t * a.gs + r * a.gk] : 0.f;
      float sc = 0.f;
      if (in) {
        const float v = to_f(row[e]);
        sc = a.sigmoid ? 1.f / (1.f + expf(-v)) : total == 0.f ? 0.f : expf(v - m) / total;
      }
      sum += sc;
      dot += g * sc;
      chosen[r] = Chosen{g, in ? (uint32_t)e : ~0u};
    }
    sum = lanes_sum<LPT>(sum);
    dot = lanes_sum<LPT>(dot);
    float mul = a.scale, sub_ = 0.f, all;
    if (a.renorm) {
      mul = sum == 0.f ? 0.f : a.scale / sum;
      sub_ = sum == 0.f ? 0.f : dot / sum;
      all = 0.f;  // sum of ds_i s_i = scale (dot - dot) / S
    } else {
      all = a.scale * dot;
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < NPL; ++i) dense[at + i] = 0.f;
    // in order of rank, so that an expert named twice adds up the same way each time
    for (uint32_t r = 0; r < a.top_k; ++r) {
      const Chosen c = chosen[r];
      if (c.expert / NPL == lane) dense[c.expert] += mul * (c.score - sub_);
    }
    float d[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      const float ds = dense[at + i];
      d[i] = a.sigmoid ? ds * s[i] * (1.f - s[i]) : s[i] * (ds - all);
      if (s[i] == 0.f) d[i] = 0.f;
    }
    if (live) {
      T* o = static_cast<T*>(a.gx) + t * a.os;
      if (a.vec) {
        constexpr int W = 16 / sizeof(T) < NPL ? 16 / sizeof(T) : NPL;
#pragma unroll
        for (int k = 0; k < NPL; k += W) {
          Pack<T, W> q;
#pragma unroll
          for (int i = 0; i < W; ++i) q.v[i] = from_f<T>(d[k + i]);
          if (at + k < a.n) store_pack<T, W>(o + at + k, q);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (at + i < a.n) o[at + i] = from_f<T>(d[i]);
      }
    }
    __syncwarp();
  }
}

template <typename T, int NPL, int LPT>
void launch(const RouteArgs& a, bool grad, cudaStream_t s) {
  constexpr uint32_t kTokens = kThreads / LPT;
  const uint64_t ctas = ((uint64_t)a.tokens + kTokens - 1) / kTokens;
  const unsigned grid = (unsigned)std::min<uint64_t>(ctas, (uint64_t)sm_count() * 8);
  if (grad) {
    const size_t smem = kThreads * NPL * sizeof(float) + kTokens * a.top_k * sizeof(Chosen);
    if (smem > 48 * 1024)
      cuda_ok(cudaFuncSetAttribute(gpuos_route_grad_kernel<T, NPL, LPT>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "shared memory");
    gpuos_route_grad_kernel<T, NPL, LPT><<<grid, kThreads, smem, s>>>(a);
  } else {
    const size_t smem = kTokens * ((a.groups > 1 ? a.groups : 0) * sizeof(double) + a.top_k * sizeof(Chosen));
    if (smem > 48 * 1024)
      cuda_ok(cudaFuncSetAttribute(gpuos_route_kernel<T, NPL, LPT>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "shared memory");
    gpuos_route_kernel<T, NPL, LPT><<<grid, kThreads, smem, s>>>(a);
  }
  cuda_ok(cudaGetLastError(), "launch");
}

template <typename T>
void by_size(const RouteArgs& a, bool grad, cudaStream_t s) {
  if (a.n <= 32) launch<T, 8, 4>(a, grad, s);
  else if (a.n <= 64) launch<T, 8, 8>(a, grad, s);
  else if (a.n <= 128) launch<T, 8, 16>(a, grad, s);
  else if (a.n <= 256) launch<T, 8, 32>(a, grad, s);
  else if (a.n <= 512) launch<T, 16, 32>(a, grad, s);
  else launch<T, 32, 32>(a, grad, s);
}

void start(const RouteArgs& a, int32_t dt, bool grad, cudaStream_t s) {
  if (a.tokens == 0 || a.n == 0) return;
  if (dt == GPUOS_F32) by_size<float>(a, grad, s);
  else if (dt == GPUOS_F16) by_size<__half>(a, grad, s);
  else by_size<__nv_bfloat16>(a, grad, s);
}

// What the two entry points check alike.
RouteArgs prepare(const gpuos_tensor* x, const gpuos_tensor* weights, const char* weights_name,
                  const gpuos_tensor* experts, int32_t score, int32_t renorm, float scale) {
  check_tensor(x, 2, "logits");
  check_tensor(weights, 2, weights_name);
  check_tensor(experts, 2, "experts");
  need(is_real(x->dtype), "logits must be float32, float16 or bfloat16");
  need(weights->dtype == GPUOS_F32, "weights must be float32");
  need(is_index(experts->dtype), "experts must be int32 or int64");
  need(score == GPUOS_SCORE_SOFTMAX || score == GPUOS_SCORE_SIGMOID, "unknown score");
  need(std::abs(scale) <= 3.4028234e38f, "scale must be finite");
  const int64_t tokens = x->sizes[0], n = x->sizes[1];
  need(n >= 1 && n <= 1024, "the number of experts must be in [1, 1024]");
  need(tokens < (1ll << 40), "too many tokens");
  need(weights->sizes[0] == tokens && experts->sizes[0] == tokens, "weights and experts must have a row for each token");
  const int64_t k = weights->sizes[1];
  need(experts->sizes[1] == k, "weights and experts must have the same columns");
  need(k >= 1 && k <= kMaxTop && k <= n, "top_k must be in [1, min(64, experts)]");
  if (numel(*x)) need(n == 1 || x->strides[1] == 1, "the last dim of logits must be contiguous");
  RouteArgs a{};
  a.x = x->data;
  a.experts = experts->data;
  a.xs = x->strides[0];
  a.es = experts->strides[0];
  a.ek = experts->strides[1];
  a.tokens = tokens;
  a.n = (uint32_t)n;
  a.top_k = (uint32_t)k;
  a.scale = scale;
  a.sigmoid = score == GPUOS_SCORE_SIGMOID;
  a.renorm = renorm != 0;
  a.wide = experts->dtype == GPUOS_I64;
  a.groups = a.top_groups = 1;
  a.per_group = FastDiv((uint32_t)n);
  const int w = 16 / esize(x->dtype);
  a.vec = n % w == 0 && rows_aligned(*x, w);
  return a;
}

void route(const gpuos_tensor* x, const gpuos_tensor* bias, const gpuos_tensor* weights, const gpuos_tensor* experts,
           int32_t score, int32_t groups, int32_t top_groups, int32_t group_score, int32_t renorm, float scale,
           cudaStream_t stream) {
  RouteArgs a = prepare(x, weights, "weights", experts, score, renorm, scale);
  need(groups >= 1 && groups <= kMaxGroups && a.n % groups == 0, "groups must divide the experts, at most 64");
  need(top_groups >= 1 && top_groups <= groups, "top_groups must be in [1, groups]");
  need(group_score == GPUOS_GROUP_MAX || group_score == GPUOS_GROUP_TOP2, "unknown group score");
  need(a.top_k <= a.n / groups * top_groups, "top_k must not exceed the experts of the open groups");
  a.weights = static_cast<float*>(weights->data);
  a.ws = weights->strides[0];
  a.wk = weights->strides[1];
  a.groups = (uint32_t)groups;
  a.top_groups = (uint32_t)top_groups;
  a.per_group = FastDiv(a.n / groups);
  a.top2 = group_score == GPUOS_GROUP_TOP2;
  if (bias) {
    check_tensor(bias, 1, "bias");
    need(bias->dtype == GPUOS_F32 && bias->sizes[0] == a.n, "bias must be float32, one for each expert");
    a.bias = static_cast<const float*>(bias->data);
    a.bs = bias->strides[0];
    no_overlap(*weights, *bias, "weights overlap bias");
    no_overlap(*experts, *bias, "experts overlap bias");
  }
  if (groups == top_groups) a.groups = 1;  // every group is open
  check_output(*weights, "weights");
  check_output(*experts, "experts");
  no_overlap(*weights, *experts, "weights overlap experts");
  no_overlap(*weights, *x, "weights overlap logits");
  no_overlap(*experts, *x, "experts overlap logits");
  start(a, x->dtype, false, stream);
}

void route_grad(const gpuos_tensor* x, const gpuos_tensor* experts, const gpuos_tensor* gw, const gpuos_tensor* gx,
                int32_t score, int32_t renorm, float scale, cudaStream_t stream) {
  RouteArgs a = prepare(x, gw, "grad_weights", experts, score, renorm, scale);
  check_tensor(gx, 2, "grad_logits");
  need(gx->dtype == x->dtype, "grad_logits must have the dtype of logits");
  same_sizes(*gx, *x, "grad_logits must have the sizes of logits");
  if (numel(*gx)) need(a.n == 1 || gx->strides[1] == 1, "the last dim of grad_logits must be contiguous");
  check_output(*gx, "grad_logits");
  no_overlap(*gx, *x, "grad_logits overlap logits");
  no_overlap(*gx, *experts, "grad_logits overlap experts");
  no_overlap(*gx, *gw, "grad_logits overlap grad_weights");
  a.gw = static_cast<const float*>(gw->data);
  a.gs = gw->strides[0];
  a.gk = gw->strides[1];
  a.gx = gx->data;
  a.os = gx->strides[0];
  a.vec = a.vec && rows_aligned(*gx, 16 / esize(x->dtype));
  start(a, x->dtype, true, stream);
}

}  // namespace
}  // namespace rowops
}  // namespace gpuos

extern "C" int32_t gpuos_route(const gpuos_tensor* logits, const gpuos_tensor* bias, const gpuos_tensor* weights,
                               const gpuos_tensor* experts, int32_t score, int32_t groups, int32_t top_groups,
                               int32_t group_score, int32_t renormalize, float scale, void* stream) {
  return gpuos::rowops::entry("gpuos_route", [&] {
    gpuos::rowops::route(logits, bias, weights, experts, score, groups, top_groups, group_score, renormalize, scale,
                         static_cast<cudaStream_t>(stream));
  });
}

extern "C" int32_t gpuos_route_grad(const gpuos_tensor* logits, const gpuos_tensor* experts,
                                    const gpuos_tensor* grad_weights, const gpuos_tensor* grad_logits, int32_t score,
                                    int32_t renormalize, float scale, void* stream) {
  return gpuos::rowops::entry("gpuos_route_grad", [&] {
    gpuos::rowops::route_grad(logits, experts, grad_weights, grad_logits, score, renormalize, scale,
                              static_cast<cudaStream_t>(stream));
  });
}
