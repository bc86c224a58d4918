// gpuos_route / gpuos_route_grad: routing of tokens to experts.
//
//   s    = softmax(x) or sigmoid(x)          over a token's E logits
//   key  = s + bias                          (without a bias: x, which orders as s does)
//   groups of E / groups neighbours: a group is worth its largest key, or the sum of its two
//   largest; the best `top_groups` stay open
//   top_k largest keys of the open groups; of equal ones the lowest index
//   w    = s of the chosen (/ their sum) * scale
//
// The chosen experts are those of exact arithmetic, at the price of a fast
// selection: every key becomes one unsigned integer, the key's place in the
// row's range above the expert's slot, so that a maximum over lanes gives key and
// expert at once and of equal keys the lowest index.  16-bit logits without a
// bias fit whole; other keys are computed in 32 bits, with a known error bound, and rounded
// to 22 to 24 bits of the range that the largest ones span.  Where two keys whose
// order matters come out closer than the error, the token is done again in 64 bits
// (about one in a thousand of random logits).
//
// A token belongs to LPT lanes of a warp, each holding NPL neighbouring experts
// of one group in registers: up to 256 experts take 8 a lane and as many lanes as
// needed, so that one warp serves up to 8 tokens of few experts.  A lane sorts its
// keys once; a round of the selection is then a maximum over the lanes' first ones.
// Few experts make the kernel a matter of instructions, not of bytes: 16384
// tokens of 256 take 18 MB, 2.8 us.
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
  uint32_t per_group;  // experts of a group
  // How a token's experts are seated: by groups, so that no lane has experts of two, or, where
  // the groups are too many for the lanes of a warp, all in a row.
  uint32_t seat_groups, seat_per_group;
  FastDiv lanes;       // lanes of a group
  float scale;
  int sigmoid, renorm, top2, wide, vec;
};

template <typename R> struct Num;
template <> struct Num<float> {
  static __device__ __forceinline__ float exp_(float x) { return expf(x); }
};
template <> struct Num<double> {
  using Key = unsigned long long;
  static __device__ __forceinline__ double exp_(double x) { return exp(x); }
  // An unsigned integer that orders as x does; NaN as -inf; never 0.
  static __device__ __forceinline__ Key key(double x) {
    if (x != x) x = -INFINITY;
    const Key b = (Key)__double_as_longlong(x + 0.0);
    return (b >> 63) ? ~b : b | (1ull << 63);
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

// A lane's n of NPL logits from `at` on; the others are -inf.
template <typename T, int NPL>
__device__ __forceinline__ void load_logits(const T* row, uint32_t at, uint32_t n, bool vec, bool live,
                                            float (&x)[NPL]) {
  constexpr int W = 16 / sizeof(T) < NPL ? 16 / sizeof(T) : NPL;
  if (vec) {
#pragma unroll
    for (int k = 0; k < NPL; k += W) {
      Pack<T, W> q;
      const bool in = live && k < (int)n;
      if (in) q = load_pack<T, W, false>(row + at + k);
#pragma unroll
      for (int i = 0; i < W; ++i) x[k + i] = in ? to_f(q.v[i]) : -INFINITY;
    }
  } else {
#pragma unroll
    for (int i = 0; i < NPL; ++i) x[i] = live && i < (int)n ? to_f(row[at + i]) : -INFINITY;
  }
}

// Scores of a lane's n of NPL experts in R; a row of -inf has softmax scores 0
// (nothing is left by its mask).  NaN stays: one makes the whole row's scores NaN.
template <typename R, int NPL, int LPT>
__device__ __forceinline__ void score(const float (&x)[NPL], uint32_t n, bool sigmoid, R (&s)[NPL],
                                      float* top = nullptr, R* total = nullptr) {
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) s[i] = i < (int)n ? R(1) / (R(1) + Num<R>::exp_(-(R)x[i])) : R(0);
    return;
  }
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NPL; ++i) m = fmaxf(m, x[i]);
  m = lanes_max<LPT>(m);
  R sum = 0;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    s[i] = (m == -INFINITY && x[i] == -INFINITY) ? R(0) : Num<R>::exp_((R)x[i] - (R)m);
    sum += s[i];
  }
  sum = lanes_sum<LPT>(sum);
  const R inv = sum == R(0) ? R(0) : R(1) / sum;
#pragma unroll
  for (int i = 0; i < NPL; ++i) s[i] *= inv;
  if (top) *top = m;
  if (total) *total = sum;
}

// The 16 bits of a value that came from T, -0 as 0.
template <typename T>
__device__ __forceinline__ uint32_t half_bits(float x) {
  x += 0.f;
  if constexpr (std::is_same_v<T, __half>) return __half_as_ushort(__float2half_rn(x));
  else return __float_as_uint(x) >> 16;
}

template <int LPT> constexpr uint32_t kLanes = LPT == 32 ? ~0u : (1u << (LPT & 31)) - 1;

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2e = 1.44269504088896341f;

template <int LPT>
__device__ __forceinline__ uint32_t lanes_max_u32(uint32_t v) {
  if constexpr (LPT == 32) return __reduce_max_sync(~0u, v);
  else return lanes_max<LPT>(v);
}

// Where a lane's experts are.
struct Seat {
  uint32_t lane, base;  // in the token; of the token in the warp
  uint32_t group, first_lane;  // the lane's group, and that group's first lane in the token
  uint32_t at, n;       // first expert and how many of the lane's NPL
};

// The expert of slot lane * NPL + i.
template <int NPL>
__device__ __forceinline__ uint32_t expert_of(const RouteArgs& a, uint32_t slot) {
  const uint32_t lane = slot / NPL, g = a.lanes.div(lane);
  return g * a.seat_per_group + (lane - g * a.lanes.d) * NPL + slot % NPL;
}

// One token's selection in 64 bits: chosen[r] is the slot of rank r.
template <int NPL, int LPT>
__device__ __noinline__ void select_exact(const RouteArgs& a, const float (&x)[NPL], const float (&bias)[NPL],
                                          const Seat seat, bool keyed, double* worth, uint16_t* chosen) {
  using Key = Num<double>::Key;
  double s[NPL];
  score<double, NPL, LPT>(x, seat.n, a.sigmoid, s);
  Key key[NPL];
#pragma unroll
  for (int i = 0; i < NPL; ++i)
    key[i] = i < (int)seat.n ? Num<double>::key(keyed ? s[i] + (double)bias[i] : (double)x[i]) : Key(0);
  if (a.groups > 1) {
    // what counts for a group: the keys, or the scores where two of them add up
    double v[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      v[i] = keyed ? s[i] + (double)bias[i] : a.top2 ? s[i] : (double)x[i];
      if (!(v[i] >= -INFINITY)) v[i] = -INFINITY;  // NaN
    }
    for (uint32_t g = 0; g < a.groups; ++g) {
      const uint32_t lo = g * a.per_group, hi = lo + a.per_group;
      double w1 = -INFINITY, w2 = -INFINITY;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (i < (int)seat.n && seat.at + i >= lo && seat.at + i < hi) {
          w2 = fmax(w2, fmin(w1, v[i]));
          w1 = fmax(w1, v[i]);
        }
#pragma unroll
      for (int d = LPT / 2; d; d >>= 1) {
        const double o1 = __shfl_xor_sync(~0u, w1, d), o2 = __shfl_xor_sync(~0u, w2, d);
        w2 = fmax(fmin(w1, o1), fmax(w2, o2));
        w1 = fmax(w1, o1);
      }
      if (seat.lane == 0) worth[g] = a.top2 && a.per_group > 1 ? w1 + w2 : w1;
    }
    __syncwarp();
    // a group stays open where fewer than top_groups are better, or as good and before it
    unsigned long long open = 0;
    for (uint32_t g = seat.lane; g < a.groups; g += LPT) {
      const Key mine = Num<double>::key(worth[g]);
      uint32_t before = 0;
      for (uint32_t h = 0; h < a.groups; ++h) {
        const Key other = Num<double>::key(worth[h]);
        before += other > mine || (other == mine && h < g);
      }
      if (before < a.top_groups) open |= 1ull << g;
    }
#pragma unroll
    for (int d = LPT / 2; d; d >>= 1) open |= __shfl_xor_sync(~0u, open, d);
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (i < (int)seat.n && !((open >> ((seat.at + i) / a.per_group)) & 1)) key[i] = 0;
  }
  Key mine = 0;
#pragma unroll
  for (int i = 0; i < NPL; ++i) mine = key[i] > mine ? key[i] : mine;
  for (uint32_t r = 0; r < a.top_k; ++r) {
    const Key best = lanes_max<LPT>(mine);
    const uint32_t has = __ballot_sync(~0u, mine == best) >> seat.base;
    if (seat.lane == (uint32_t)(__ffs(has & kLanes<LPT>) - 1)) {
      bool found = false;
      Key next = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        if (!found && key[i] == best) {
          found = true;
          chosen[r] = (uint16_t)(seat.lane * NPL + i);
          key[i] = 0;
        }
        next = key[i] > next ? key[i] : next;
      }
      mine = next;
    }
  }
  __syncwarp();
}

// Sorts a lane's keys, the largest first (compare-exchanges of Batcher's merge).
template <int N>
__device__ __forceinline__ void sort_down(uint32_t (&k)[N]) {
#pragma unroll
  for (int p = 1; p < N; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int j = q % p; j + q < N; j += 2 * q)
#pragma unroll
        for (int i = 0; i < q; ++i)
          if (i + j + q < N && (i + j) / (2 * p) == (i + j + q) / (2 * p)) {
            const uint32_t hi = max(k[i + j], k[i + j + q]), lo = min(k[i + j], k[i + j + q]);
            k[i + j] = hi;
            k[i + j + q] = lo;
          }
}

template <typename T, int NPL, int LPT>
__global__ void __launch_bounds__(kThreads)
gpuos_route_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr uint32_t kTokens = kThreads / LPT;  // tokens a CTA handles at once
  constexpr uint32_t kSlots = LPT * NPL;
  constexpr int kBits = kSlots <= 256 ? 24 : 22;  // of a key, above the slot's
  constexpr bool kHalf = sizeof(T) == 2;
  const uint32_t sub = threadIdx.x / LPT;
  double* worth = reinterpret_cast<double*>(smem) + sub * (a.groups > 1 ? a.groups : 0);
  uint16_t* chosen = reinterpret_cast<uint16_t*>(reinterpret_cast<double*>(smem) +
                                                 kTokens * (a.groups > 1 ? a.groups : 0)) + sub * a.top_k;
  Seat seat;
  seat.lane = threadIdx.x % LPT;
  seat.base = (threadIdx.x & 31) - seat.lane;
  seat.group = a.lanes.div(seat.lane);
  seat.first_lane = seat.group * a.lanes.d;
  const uint32_t in_group = (seat.lane - seat.first_lane) * NPL;
  seat.at = seat.group * a.seat_per_group + in_group;
  seat.n = seat.group < a.seat_groups && in_group < a.seat_per_group
               ? min((uint32_t)NPL, a.seat_per_group - in_group) : 0;
  float bias[NPL];
  bool keyed = a.bias != nullptr;
  if (keyed) {
    // a bias that is the same for all does not change the order
    const float b0 = __ldg(a.bias);
    bool same = b0 - b0 == 0.f;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      bias[i] = i < (int)seat.n ? __ldg(a.bias + (seat.at + i) * a.bs) : b0;
      same = same && bias[i] == b0;
    }
    keyed = !__syncthreads_and(same);
  }

  for (int64_t t0 = (int64_t)blockIdx.x * kTokens; t0 < a.tokens; t0 += (int64_t)gridDim.x * kTokens) {
    const int64_t t = t0 + sub;
    const bool live = t < a.tokens;
    const T* row = static_cast<const T*>(a.x) + (live ? t * a.xs : 0);
    float x[NPL];
    load_logits<T, NPL>(row, seat.at, seat.n, a.vec, live, x);
    // scores, as far as the order or the weights need all of them
    float s[NPL], m = 0.f, total = 1.f;
    const bool scored = keyed || (a.groups > 1 && a.top2);
    if (!a.sigmoid) {
      m = -INFINITY;
#pragma unroll
      for (int i = 0; i < NPL; ++i) m = fmaxf(m, x[i]);
      m = lanes_max<LPT>(m);
      total = 0.f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        s[i] = m == -INFINITY && x[i] == -INFINITY ? 0.f : ex2((x[i] - m) * kLog2e);
        total += s[i];
      }
      total = lanes_sum<LPT>(total);
      const float by = total == 0.f ? 0.f : rcp(total);
      if (scored) {
#pragma unroll
        for (int i = 0; i < NPL; ++i) s[i] *= by;
      }
    } else if (scored) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) s[i] = rcp(1.f + ex2(x[i] * -kLog2e));
    }
    // A score is off by at most 10 * 2^-24 of the largest one (1 for a sigmoid), a
    // key by 2^-24 of itself more; two of them by twice that.
    const float s_max = a.sigmoid ? 1.f : rcp(total);
    bool doubt = a.top_k > LPT || a.groups != a.seat_groups;
    bool open = seat.n > 0;
    if (a.groups > 1 && a.groups == a.seat_groups) {
      float v1 = -INFINITY, v2 = -INFINITY;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (i < (int)seat.n) {
          const float v = keyed ? s[i] + bias[i] : a.top2 ? s[i] : x[i];
          if (v != v) doubt = true;
          v2 = fmaxf(v2, fminf(v1, v));
          v1 = fmaxf(v1, v);
        }
      float w1 = v1, w2 = v2;
      for (uint32_t i = 1; i < a.lanes.d; ++i) {
        uint32_t from = seat.lane + i;
        if (from >= seat.first_lane + a.lanes.d) from -= a.lanes.d;
        const float o1 = __shfl_sync(~0u, v1, seat.base + from), o2 = __shfl_sync(~0u, v2, seat.base + from);
        w2 = fmaxf(fminf(w1, o1), fmaxf(w2, o2));
        w1 = fmaxf(w1, o1);
      }
      const bool two = a.top2 && a.per_group > 1;
      const float w = two ? w1 + w2 : w1;
      // two keys: twice the error; without scores the largest logits are exact
      const float error = keyed || a.top2 ? (two ? 2.f : 1.f) * 1.25e-6f * s_max + 5e-7f * fabsf(w) : 0.f;
      uint32_t before = 0, maybe = 0;
      for (uint32_t h = 0; h < a.groups; ++h) {
        const float o = __shfl_sync(~0u, w, seat.base + h * a.lanes.d);
        before += o > w || (o == w && h < seat.group);
        // Another group within the error: its order is in doubt.  A NaN or two infinities too.
        maybe += h != seat.group && error > 0.f && !(fabsf(o - w) > error);
      }
      open = open && before < a.top_groups;
      // it matters where it could open this group or close it
      if (seat.n && maybe && before < a.top_groups + maybe && before + maybe >= a.top_groups) doubt = true;
    }

    uint32_t key[NPL];
    bool exact = false;
    uint32_t slack = 0;  // keys this close are in doubt
    if (kHalf && !keyed) {
      exact = true;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const uint32_t b = half_bits<T>(x[i]);
        key[i] = (((b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u) << 16) | (kSlots - 1 - (seat.lane * NPL + i));
        if (x[i] != x[i]) doubt = true;
      }
    } else {
      // the range from the largest key down to one that top_k + 1 others reach
      float k[NPL], hi = -INFINITY, lo = INFINITY;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        k[i] = keyed ? s[i] + bias[i] : x[i];
        if (i < (int)seat.n) {
          hi = fmaxf(hi, k[i]);
          lo = fminf(lo, k[i]);
        }
      }
      const uint32_t lanes = __popc(__ballot_sync(~0u, open) >> seat.base & kLanes<LPT>);
      const float top = lanes_max<LPT>(open ? hi : -INFINITY);
      lo = -lanes_max<LPT>(open ? -(a.top_k < lanes ? hi : lo) : -INFINITY);
      lo = fmaxf(lo, top - 64.f);
      const float range = fmaxf(top - lo, 1e-30f);
      const float by = (float)((1 << kBits) - 64) / range;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const uint32_t f = (uint32_t)fminf(fmaxf(fmaf(k[i] - lo, by, 16.f), 1.f), (float)((1 << kBits) - 1));
        key[i] = f << (32 - kBits) | (kSlots - 1 - (seat.lane * NPL + i));
      }
      // Rounding to places keeps the order of exact keys, or makes them equal; for the others
      // their error counts, and the roundings of the difference, below 4 places.
      if (keyed) {
        const float error = 1.25e-6f * s_max + 2.5e-7f * fmaxf(fabsf(top), fabsf(lo));
        slack = 4 + (uint32_t)fminf(error * by, 4e9f);
      }
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (!open || i >= (int)seat.n) key[i] = 0;

    uint32_t won = 0;  // of rank `lane`
    if (NPL <= 8) {
      sort_down<NPL>(key);
    } else {
#pragma unroll
      for (int i = 1; i < NPL; ++i) {  // the largest first
        const uint32_t hi = max(key[0], key[i]);
        key[i] = min(key[0], key[i]);
        key[0] = hi;
      }
    }
    uint32_t last = ~0u;
    for (uint32_t r = 0; r < a.top_k + (exact ? 0 : 1); ++r) {
      const uint32_t best = lanes_max_u32<LPT>(key[0]);
      if (!exact) {
        const uint32_t f = best >> (32 - kBits);
        if (best != 0 && (last - f <= slack || (r < a.top_k && f < 8))) doubt = true;
        last = f;
      }
      if (seat.lane == r) won = best;
      if (key[0] == best) {
        if (NPL <= 8) {
#pragma unroll
          for (int i = 0; i + 1 < NPL; ++i) key[i] = key[i + 1];
          key[NPL - 1] = 0;
        } else {
          key[0] = 0;
#pragma unroll
          for (int i = 1; i < NPL; ++i) {
            const uint32_t hi = max(key[0], key[i]);
            key[i] = min(key[0], key[i]);
            key[0] = hi;
          }
        }
      }
    }
    const bool redo = __any_sync(~0u, doubt && live);
    if (redo) select_exact<NPL, LPT>(a, x, bias, seat, keyed, worth, chosen);

    // weights from the chosen logits, a lane each
    float sum = 0.f;
    for (uint32_t r = seat.lane; r < a.top_k; r += LPT) {
      const uint32_t slot = redo ? chosen[r] : kSlots - 1 - (won & ((1u << (exact ? 16 : 32 - kBits)) - 1));
      const uint32_t e = expert_of<NPL>(a, slot);
      const float v = live ? to_f(row[e]) : 0.f;
      float sc;
      if (a.sigmoid) sc = 1.f / (1.f + expf(-v));
      else sc = total == 0.f ? 0.f : expf(v - m) / total;
      sum += sc;
      if (live) {
        if (!a.renorm) a.weights[t * a.ws + r * a.wk] = sc * a.scale;
        if (a.wide) static_cast<int64_t*>(a.experts)[t * a.es + r * a.ek] = e;
        else static_cast<int32_t*>(a.experts)[t * a.es + r * a.ek] = (int32_t)e;
      }
      won = __float_as_uint(sc);  // the only one of a lane where it is needed below
    }
    if (a.renorm) {
      sum = lanes_sum<LPT>(sum);
      const float by = sum == 0.f ? 0.f : a.scale / sum;
      for (uint32_t r = seat.lane; r < a.top_k; r += LPT) {
        float sc = __uint_as_float(won);
        if (a.top_k > LPT) {  // several ranks a lane: again
          const float v = live ? to_f(row[expert_of<NPL>(a, chosen[r])]) : 0.f;
          sc = a.sigmoid ? 1.f / (1.f + expf(-v)) : total == 0.f ? 0.f : expf(v - m) / total;
        }
        if (live) a.weights[t * a.ws + r * a.wk] = sc * by;
      }
    }
    __syncwarp();
  }
}

struct Chosen {
  float score;
  uint32_t expert;
};

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
    load_logits<T, NPL>(row, at, at < a.n ? min((uint32_t)NPL, a.n - at) : 0u, a.vec, live, x);
    float m = 0.f, total = 1.f;
    score<float, NPL, LPT>(x, at < a.n ? min((uint32_t)NPL, a.n - at) : 0u, a.sigmoid, s, &m, &total);
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
void launch(RouteArgs a, bool grad, cudaStream_t s) {
  constexpr uint32_t kTokens = kThreads / LPT;
  const uint64_t ctas = ((uint64_t)a.tokens + kTokens - 1) / kTokens;
  const unsigned grid = (unsigned)std::min<uint64_t>(ctas, (uint64_t)sm_count() * 8);
  a.seat_groups = a.groups;
  a.seat_per_group = a.per_group;
  if (a.groups * ((a.per_group + NPL - 1) / NPL) > LPT) {
    a.seat_groups = 1;
    a.seat_per_group = a.n;
  }
  a.lanes = FastDiv((a.seat_per_group + NPL - 1) / NPL);
  if (grad) {
    const size_t smem = kThreads * NPL * sizeof(float) + kTokens * a.top_k * sizeof(Chosen);
    if (smem > 48 * 1024)
      cuda_ok(cudaFuncSetAttribute(gpuos_route_grad_kernel<T, NPL, LPT>,
                                   cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem), "shared memory");
    gpuos_route_grad_kernel<T, NPL, LPT><<<grid, kThreads, smem, s>>>(a);
  } else {
    const size_t smem = kTokens * ((a.groups > 1 ? a.groups : 0) * sizeof(double) + a.top_k * sizeof(uint16_t));
    gpuos_route_kernel<T, NPL, LPT><<<grid, kThreads, smem, s>>>(a);
  }
  cuda_ok(cudaGetLastError(), "launch");
}

// Lanes a token needs with NPL experts a lane, none of two groups.
uint32_t lanes_for(const RouteArgs& a, uint32_t npl) { return a.groups * ((a.per_group + npl - 1) / npl); }

template <typename T>
void by_size(const RouteArgs& a, bool grad, cudaStream_t s) {
  const uint32_t lanes = lanes_for(a, 8);
  if (lanes <= 4) launch<T, 8, 4>(a, grad, s);
  else if (lanes <= 8) launch<T, 8, 8>(a, grad, s);
  else if (lanes <= 16) launch<T, 8, 16>(a, grad, s);
  else if (lanes <= 32) launch<T, 8, 32>(a, grad, s);
  else if (lanes_for(a, 16) <= 32) launch<T, 16, 32>(a, grad, s);
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
  a.per_group = (uint32_t)n;
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
  a.per_group = a.n / groups;
  a.top2 = group_score == GPUOS_GROUP_TOP2;
  if (bias) {
    check_tensor(bias, 1, "bias");
    need(bias->dtype == GPUOS_F32 && bias->sizes[0] == a.n, "bias must be float32, one for each expert");
    a.bias = static_cast<const float*>(bias->data);
    a.bs = bias->strides[0];
    no_overlap(*weights, *bias, "weights overlap bias");
    no_overlap(*experts, *bias, "experts overlap bias");
  }
  if (groups == top_groups) {  // every group is open
    a.groups = 1;
    a.per_group = a.n;
  }
  a.vec = a.vec && a.per_group % (16 / esize(x->dtype)) == 0;
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
