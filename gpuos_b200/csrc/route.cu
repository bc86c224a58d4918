// gpuos_route / gpuos_route_grad: routing of tokens to experts.
//
//   s    = softmax(x) or sigmoid(x)          over a token's E logits
//   key  = s + bias                          (without one, or with one number for all: x, which orders as s does)
//   groups of E / groups neighbours: a group is worth its largest key, or the sum of its two
//   largest; the best `top_groups` stay open
//   top_k largest keys of the open groups; of equal ones the lowest index
//   w    = s of the chosen (/ their sum) * scale
//
// The chosen experts are those of 64-bit arithmetic, by a selection in 32-bit integers, so that a
// maximum over lanes is one or a few instructions.  16-bit logits without a bias fit whole above the
// expert's slot; 32-bit logits become their place among 2^24 (2^22) of the range that the row's
// largest ones span.  Scores are computed in 64 bits (the exponential as a series,
// to 2^-32: the half-rate pipe has room beside the integers) and become places among 2^29
// of the range that scores and bias can take; groups add places.
// Where places whose order matters are equal, or for scores next to each other, the
// token's lanes do it again with 64-bit keys.  (Scores in 32 bits put one token in two
// thousand in doubt, and the few that waited for those set the time.)  What that does not settle (keys within 2^-38, NaN, more
// ranks than lanes, groups that fit no seats) is left for the CTA's second part, a warp to a token.
//
// A token belongs to LPT lanes of a warp, each holding NPL neighbouring experts
// of one group in registers: up to 256 experts take 8 a lane and as many lanes as
// needed, so that one warp serves up to 8 tokens of few experts.  A lane sorts its
// keys once; a round of the selection is then a maximum over the lanes' first ones.
// Few experts make the kernel a matter of instructions, not of bytes: 16384
// tokens of 256 fp32 logits in 8 groups are 18 MB, 2.8 us, and 1236 instructions of a warp each, 23.8 us
// at three quarters of the issue slots; 32749 of 128 bf16 without groups take 14.7 us, the gradient 10.0.
// Tokens that all go to the second part cost several times that: 8192 x 64 with 40 ranks 59 us.
#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 64;
constexpr uint32_t kCtaTokens = 1024;  // a CTA takes at most
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
  uint32_t exact_warps;  // of a CTA, that do tokens in doubt
  float scale;
  int sigmoid, renorm, top2, wide, vec;
};

using Key64 = unsigned long long;

// An unsigned integer that orders as x does; NaN as -inf; never 0.
__device__ __forceinline__ Key64 key64(double x) {
  if (x != x) x = -INFINITY;
  const Key64 b = (Key64)__double_as_longlong(x + 0.0);
  return (b >> 63) ? ~b : b | (1ull << 63);
}

// Maxima over a token's lanes; over a whole warp in one instruction.
template <int LPT>
__device__ __forceinline__ uint32_t lanes_top(uint32_t v) {
  if constexpr (LPT == 32) {
    return __reduce_max_sync(~0u, v);
  } else {
#pragma unroll
    for (int d = LPT / 2; d; d >>= 1) v = max(v, __shfl_xor_sync(~0u, v, d));
    return v;
  }
}
template <int LPT>
__device__ __forceinline__ Key64 lanes_top(Key64 v) {
  if constexpr (LPT == 32) {
    const uint32_t hi = __reduce_max_sync(~0u, (uint32_t)(v >> 32));
    const uint32_t lo = __reduce_max_sync(~0u, (uint32_t)(v >> 32) == hi ? (uint32_t)v : 0u);
    return (Key64)hi << 32 | lo;
  } else {
#pragma unroll
    for (int d = LPT / 2; d; d >>= 1) v = max(v, __shfl_xor_sync(~0u, v, d));
    return v;
  }
}
template <int LPT>
__device__ __forceinline__ float lanes_top(float v) {
  if constexpr (LPT == 32) {
    float r;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
  } else {
#pragma unroll
    for (int d = LPT / 2; d; d >>= 1) v = fmaxf(v, __shfl_xor_sync(~0u, v, d));
    return v;
  }
}

__device__ __forceinline__ double value64(Key64 k) {
  return __longlong_as_double((long long)((k >> 63) ? k & ~(1ull << 63) : ~k));
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

__device__ __forceinline__ float sigmoid(float v) {
  const float a = expf(-fabsf(v)), q = rcp(1.f + a);
  return v > 0.f ? q : a * q;
}
// The sigmoid of a chosen logit over e^top, top the smaller of 0 and the largest chosen logit: of a
// sum of those, sigmoids too small for 32 bits keep their shares.  e^-v leaves 64 bits at the limit: the
// sigmoid is 0 from there on.
__device__ __forceinline__ float sigmoid_over(float v, float top) {
  if (v <= -709.78271484375f) return 0.f;
  return v > 0.f ? sigmoid(v) : expf(v - top) * rcp(1.f + expf(v));
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

// One token's selection in 64 bits, by a warp: keys are held as ordered integers in
// `key` (a.n of them, 0 for those of closed groups), the groups' worths in `worth`.
template <typename T>
__device__ __forceinline__ void route_exact(const RouteArgs& a, bool keyed, int64_t t, Key64* key, Key64* worth) {
  const uint32_t lane = threadIdx.x & 31;
  const T* row = static_cast<const T*>(a.x) + t * a.xs;
  float m = -INFINITY;
  double total = 0;
  if (!a.sigmoid) {
    for (uint32_t e = lane; e < a.n; e += 32) m = fmaxf(m, to_f(row[e]));
    m = lanes_top<32>(m);
#pragma unroll 1
    for (uint32_t e = lane; e < a.n; e += 32) {
      const float v = to_f(row[e]);
      if (v != -INFINITY || m != -INFINITY) total += exp((double)v - (double)m);
    }
    total = lanes_sum<32>(total);
  }
  auto score = [&](float v) {
    if (a.sigmoid) return 1.0 / (1.0 + exp(-(double)v));
    return total == 0.0 ? 0.0 : exp((double)v - (double)m) / total;
  };
#pragma unroll 1
  for (uint32_t e = lane; e < a.n; e += 32) {
    // without a bias the order is the logits', but of two scores that add up
    const float v = to_f(row[e]);
    key[e] = key64(keyed ? score(v) + (double)a.bias[e * a.bs] : a.groups > 1 && a.top2 ? score(v) : (double)v);
  }
  __syncwarp();
  if (a.groups > 1) {
    const bool two = a.top2 && a.per_group > 1;
#pragma unroll 1
    for (uint32_t g = lane; g < a.groups; g += 32) {
      Key64 k1 = 0, k2 = 0;
#pragma unroll 4
      for (uint32_t i = 0; i < a.per_group; ++i) {
        const Key64 k = key[g * a.per_group + i];
        k2 = max(k2, min(k1, k));
        k1 = max(k1, k);
      }
      worth[g] = two ? key64(value64(k1) + value64(k2)) : k1;
    }
    __syncwarp();
    unsigned long long open = 0;
#pragma unroll 1
    for (uint32_t g = lane; g < a.groups; g += 32) {
      const Key64 w = worth[g];
      uint32_t before = 0;
#pragma unroll 4
      for (uint32_t h = 0; h < a.groups; ++h) before += worth[h] > w || (worth[h] == w && h < g);
      if (before < a.top_groups) open |= 1ull << g;
    }
    open = (unsigned long long)__reduce_or_sync(~0u, (uint32_t)(open >> 32)) << 32 | __reduce_or_sync(~0u, (uint32_t)open);
#pragma unroll 1
    for (uint32_t e = lane; e < a.n; e += 32) {
      if (!((open >> (e / a.per_group)) & 1)) key[e] = 0;
      else if (!keyed) key[e] = key64(to_f(row[e]));
    }
    __syncwarp();
  }
  // rounds: the largest key, of equal ones the lowest index
  Key64 mine = 0;
  uint32_t at = 0;
  auto again = [&] {
    mine = 0;
#pragma unroll 8
    for (uint32_t e = lane; e < a.n; e += 32)
      if (key[e] > mine) {
        mine = key[e];
        at = e;
      }
  };
  again();
  float low = -INFINITY, high = -INFINITY;  // the logits of ranks lane and lane + 32
#pragma unroll 1
  for (uint32_t r = 0; r < a.top_k; ++r) {
    const Key64 best = lanes_top<32>(mine);
    const uint32_t e = __reduce_min_sync(~0u, mine == best ? at : ~0u);
    if (mine == best && at == e) {
      key[e] = 0;
      again();
    }
    if (lane == r % 32) (r < 32 ? low : high) = to_f(row[e]);
    if (lane == 0) {
      if (a.wide) static_cast<int64_t*>(a.experts)[t * a.es + r * a.ek] = e;
      else static_cast<int32_t*>(a.experts)[t * a.es + r * a.ek] = (int32_t)e;
    }
  }
  const float top = lanes_top<32>(fmaxf(low, high));
  auto weight = [&](float v) {
    // (as in the lanes' part)
    if (a.sigmoid) return a.renorm ? sigmoid_over(v, fminf(top, 0.f)) : sigmoid(v);
    if (!a.renorm || total != total) return (float)score(v);
    return top == -INFINITY ? 0.f : expf(v - top);
  };
  low = lane < a.top_k ? weight(low) : 0.f;
  high = lane + 32 < a.top_k ? weight(high) : 0.f;
  const float sum = a.renorm ? lanes_sum<32>(low + high) : 1.f;
  auto put = [&](uint32_t r, float s) {
    if (r < a.top_k) a.weights[t * a.ws + r * a.wk] = sum == 0.f ? 0.f : s / sum * a.scale;
  };
  put(lane, low);
  put(lane + 32, high);
  __syncwarp();
}

// 2^y to 2^-41; beyond 1000 either way that of the limit: the exponential series of the fraction, to t^10 (the rest is
// below 0.35^11 / 11!).
__device__ __forceinline__ double exp2_series(double y) {
  y = fmin(fmax(y, -1000.0), 1000.0);
  const int n = __double2int_rn(y);
  const double t = (y - (double)n) * 0.69314718055994530942;
  double p = 1.0 / 3628800.0;
  p = fma(p, t, 1.0 / 362880.0);
  p = fma(p, t, 1.0 / 40320.0);
  p = fma(p, t, 1.0 / 5040.0);
  p = fma(p, t, 1.0 / 720.0);
  p = fma(p, t, 1.0 / 120.0);
  p = fma(p, t, 1.0 / 24.0);
  p = fma(p, t, 1.0 / 6.0);
  p = fma(p, t, 0.5);
  p = fma(p, t, 1.0);
  p = fma(p, t, 1.0);
  return __longlong_as_double(__double_as_longlong(p) + ((long long)n << 52));
}

// 1 / d by one Newton step from 23 bits; 0 where that is below 2^-126.
__device__ __forceinline__ double inverse(double d) {
  const double r = (double)rcp((float)d);
  return r * fma(-d, r, 2.0);
}

// Conversions by the bits, for finite values within 2^-126..2^127 and 0 (which becomes 2^-127): a
// conversion instruction between 32 and 64 bits takes eight times an integer one's time.
__device__ __forceinline__ double widen(float x) {
  const int b = __float_as_int(x);
  return __hiloint2double(((b >> 3) & 0x8fffffff) + 0x38000000, b << 29);
}
__device__ __forceinline__ float narrow(double x) {  // x > 0; cut, not rounded
  return __uint_as_float(__funnelshift_l(__double2loint(x), __double2hiint(x) - 0x38000000, 3));
}

// e^a for |a| at most 60 to 2^-32: the exponential series of what is left of a without multiples
// of ln 2, to r^8 (the rest is below 0.35^9 / 9!).
__device__ __forceinline__ double exp_series(double a) {
  const double whole = 6755399441055744.0;  // 3 * 2^51: a sum's low word is its integer
  const double t = fma(a, 1.44269504088896340736, whole);
  const double r = fma(t - whole, -0.69314718055994530942, a);
  double p = 1.0 / 40320.0;
  p = fma(p, r, 1.0 / 5040.0);
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return __hiloint2double(__double2hiint(p) + (__double2loint(t) << 20), __double2loint(p));
}

// 1 / d for d of 1 to 2^100, by one Newton step from 20 bits: to 2^-39.
__device__ __forceinline__ double inverse_of_sum(double d) {
  const double r = widen(rcp(narrow(d)));
  return r * fma(-d, r, 2.0);
}

// One token's selection in 64 bits by its own lanes: lane r gets the slot of rank r.
// Returns whether two keys whose order matters are still too close, or a score is too small for the series.
template <typename T, int NPL, int LPT, bool GROUPED>
__device__ __forceinline__ bool resolve(const RouteArgs& a, const T* row, bool live, const Seat& seat, bool keyed,
                                        uint32_t* slot) {
  constexpr double kClose = 0x1p-38, kLog2eD = 1.44269504088896340736;
  float x[NPL];
  load_logits<T, NPL>(row, seat.at, seat.n, a.vec, live, x);
  double v[NPL];
  bool close = false, open = seat.n > 0;
  // e^d for d at most 0.  Between kLeast and `gone`, from where on the score is 0 in 64 bits (masked
  // logits, most of all), the series' limit would make different scores equal.
  constexpr double kLeast = -690.0;
  auto power = [&](double d, double gone) {
    close = close || (d < kLeast && d > gone);
    return d <= gone ? 0.0 : exp2_series(d * kLog2eD);
  };
  if (!keyed && !(GROUPED && a.top2)) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) v[i] = (double)x[i];
  } else if (a.sigmoid) {
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      // e^x / (1 + e^x) of a negative logit, whose e^-x would have no inverse from 2^126 on
      const double e = x[i] < 0.f ? power((double)x[i], -710.0) : exp2_series((double)x[i] * -kLog2eD);
      const double r = inverse(1.0 + e);
      v[i] = x[i] < 0.f ? e * r : r;
    }
  } else {
    float m = x[0];
#pragma unroll
    for (int i = 1; i < NPL; ++i) m = fmaxf(m, x[i]);
    m = lanes_top<LPT>(m);
    double total = 0;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      v[i] = x[i] == -INFINITY ? 0.0 : power((double)x[i] - (double)m, -746.0);
      total += v[i];
    }
    total = lanes_sum<LPT>(total);
    const double by = total == 0.0 ? 0.0 : inverse(total);  // nothing is left of a row of -inf
#pragma unroll
    for (int i = 0; i < NPL; ++i) v[i] *= by;
  }
  if (keyed) {
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (i < (int)seat.n) v[i] += (double)__ldg(a.bias + (seat.at + i) * a.bs);
  }
  if (GROUPED) {
    double l1 = -INFINITY, l2 = -INFINITY;
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (i < (int)seat.n) {
        l2 = fmax(l2, fmin(l1, v[i]));
        l1 = fmax(l1, v[i]);
      }
    double w1 = l1, w2 = l2;
#pragma unroll 1
    for (uint32_t i = 1; i < a.lanes.d; ++i) {
      uint32_t from = seat.lane + i;
      if (from >= seat.first_lane + a.lanes.d) from -= a.lanes.d;
      const double o1 = __shfl_sync(~0u, l1, seat.base + from), o2 = __shfl_sync(~0u, l2, seat.base + from);
      w2 = fmax(fmin(w1, o1), fmax(w2, o2));
      w1 = fmax(w1, o1);
    }
    const double w = a.top2 && a.per_group > 1 ? w1 + w2 : w1;
    uint32_t before = 0, near = 0;
#pragma unroll 1
    for (uint32_t h = 0; h < a.groups; ++h) {
      const double o = __shfl_sync(~0u, w, seat.base + h * a.lanes.d);
      before += o > w || (o == w && h < seat.group);
      near += o != w && fabs(o - w) < kClose;
    }
    close = close || (seat.n && near != 0);
    open = open && before < a.top_groups;
    if (!keyed && a.top2) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) v[i] = (double)x[i];
    }
  }
  Key64 key[NPL], mine = 0;
#pragma unroll
  for (int i = 0; i < NPL; ++i) {
    key[i] = open && i < (int)seat.n ? key64(v[i]) : Key64(0);
    mine = max(mine, key[i]);
  }
  double last = INFINITY;
#pragma unroll 1
  for (uint32_t r = 0; r <= a.top_k; ++r) {
    const Key64 best = lanes_top<LPT>(mine);
    const uint32_t has = __ballot_sync(~0u, mine == best) >> seat.base;
    const uint32_t owner = __ffs(has & kLanes<LPT>) - 1;
    uint32_t at = 0;
    if (seat.lane == owner) {
      bool found = false;
      mine = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        if (!found && key[i] == best) {
          found = true;
          at = seat.lane * NPL + i;
          key[i] = 0;
        }
        mine = max(mine, key[i]);
      }
    }
    at = __shfl_sync(~0u, at, seat.base + owner);
    if (seat.lane == r) *slot = at;
    if (best != 0) {
      const double k = value64(best);
      if (keyed && k != last && last - k < kClose) close = true;
      last = k;
    }
  }
  return close;
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

template <typename T, int NPL, int LPT, bool GROUPED, bool SIGMOID>
__global__ void __launch_bounds__(kThreads, NPL <= 8 ? 4 : 1)
gpuos_route_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr uint32_t kTokens = kThreads / LPT;  // tokens a CTA handles at once
  constexpr uint32_t kSlots = LPT * NPL;
  constexpr int kShift = kSlots <= 256 ? 8 : 10;  // bits of a slot, below the key's
  constexpr float kPlaces = (float)((1u << (32 - kShift)) - 1);
  constexpr bool kHalf = sizeof(T) == 2;
  constexpr int kLow = NPL <= 8 ? 3 : NPL <= 16 ? 4 : 5;  // bits of a place in the lane, below a score's place
  constexpr float kScorePlaces = (float)(1u << (32 - kLow)) - 64.f;
  __shared__ double shift[kSlots];       // the place of a slot's bias; lane l's i-th at [i][l]
  __shared__ uint32_t left;              // tokens in doubt,
  __shared__ uint16_t which[kCtaTokens];  // and which of this CTA's
  const uint32_t sub = threadIdx.x / LPT;
  if (threadIdx.x == 0) left = 0;
  __syncthreads();
  Seat seat;
  seat.lane = threadIdx.x % LPT;
  seat.base = (threadIdx.x & 31) - seat.lane;
  seat.group = a.lanes.div(seat.lane);
  seat.first_lane = seat.group * a.lanes.d;
  const uint32_t in_group = (seat.lane - seat.first_lane) * NPL;
  seat.at = seat.group * a.seat_per_group + in_group;
  seat.n = seat.group < a.seat_groups && in_group < a.seat_per_group
               ? min((uint32_t)NPL, a.seat_per_group - in_group) : 0;
  bool keyed = a.bias != nullptr, lost = false;
  double times = kScorePlaces;  // places of a score of 1
  if (keyed) {
    float bias[NPL], hi = -INFINITY, lo = INFINITY;
    // A bias that is the same for all (zeros, before balancing starts) counts as none: the order is the
    // logits', as without it.
    const float b0 = __ldg(a.bias);
    bool same = b0 - b0 == 0.f;
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      bias[i] = i < (int)seat.n ? __ldg(a.bias + (seat.at + i) * a.bs) : b0;
      same = same && bias[i] == b0;
      hi = fmaxf(hi, bias[i]);
      lo = fminf(lo, bias[i]);
      lost = lost || bias[i] - bias[i] != 0.f;  // infinities and NaN have no places
    }
    keyed = !__syncthreads_and(same);
    lost = __syncthreads_or(lost);
    hi = lanes_top<LPT>(hi);
    lo = -lanes_top<LPT>(-lo);
    times = (double)kScorePlaces / (1.0 + (double)hi - (double)lo);
    if (sub == 0) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) shift[i * LPT + seat.lane] = ((double)bias[i] - (double)lo) * times;
    }
    __syncthreads();
  }
  const bool scored = keyed || (GROUPED && a.top2);

  for (uint32_t step = 0;; ++step) {
    const int64_t t0 = ((int64_t)step * gridDim.x + blockIdx.x) * kTokens;
    if (t0 >= a.tokens) break;
    const int64_t t = t0 + sub;
    const bool live = t < a.tokens;
    const T* row = static_cast<const T*>(a.x) + (live ? t * a.xs : 0);
    float x[NPL];
    load_logits<T, NPL>(row, seat.at, seat.n, a.vec, live, x);
    // a NaN (or infinities of both signs) shows in the sum and goes the exact way
    float check = x[0];
#pragma unroll
    for (int i = 1; i < NPL; ++i) check += x[i];
    bool later = a.top_k >= LPT || (GROUPED && a.groups != a.seat_groups) || lost, doubt = false;

    float m = 0.f, total = 1.f;  // of a softmax
    if (!SIGMOID) {
      m = x[0];
#pragma unroll
      for (int i = 1; i < NPL; ++i) m = fmaxf(m, x[i]);
      m = lanes_top<LPT>(m);
    }
    // a row of -inf: every difference is -inf, not NaN
    const float top_x = m == -INFINITY ? 0.f : m;
    const bool odd = check != check || m == INFINITY;
    uint32_t key[NPL];
    if (scored) {
      double e[NPL], by = 1.0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        // beyond 60 a score is 0 or 1 as far as its place goes
        const float v = SIGMOID ? fminf(fmaxf(-x[i], -60.f), 60.f) : x[i] - top_x;
        e[i] = exp_series(SIGMOID ? widen(v) : v < -60.f ? -60.0 : (double)x[i] - (double)top_x);
      }
      if (!SIGMOID) {
        double sum = 0;
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (x[i] != -INFINITY) sum += e[i];
        sum = lanes_sum<LPT>(sum);
        total = (float)sum;
        by = sum == 0.0 ? 0.0 : inverse_of_sum(sum);
      }
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const double sc = SIGMOID ? inverse_of_sum(1.0 + e[i]) : e[i] * by;
        // an integer in the low word: below 2^52 a double's last bit is one place
        const double place = fma(sc, times, keyed ? shift[i * LPT + seat.lane] : 0.0) + (4503599627370496.0 + 16.0);
        key[i] = (uint32_t)__double2loint(place);
      }
    } else if (!SIGMOID) {
      total = 0.f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) total += ex2((x[i] - top_x) * kLog2e);
      total = lanes_sum<LPT>(total);
    }
    bool open = seat.n > 0;
    if (GROUPED && a.groups == a.seat_groups) {
      // the group's two largest, of places or (without scores) of logits in their order
      uint32_t v1 = 0, v2 = 0;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        uint32_t v = key[i];
        if (!scored) {
          const uint32_t b = __float_as_uint(x[i] + 0.f);
          v = (b >> 31) ? ~b : b | 0x80000000u;
        }
        if (i >= (int)seat.n) v = 0;
        v2 = max(v2, min(v1, v));
        v1 = max(v1, v);
      }
      uint32_t w1 = v1, w2 = v2;
      for (uint32_t i = 1; i < a.lanes.d; ++i) {
        uint32_t from = seat.lane + i;
        if (from >= seat.first_lane + a.lanes.d) from -= a.lanes.d;
        const uint32_t o1 = __shfl_sync(~0u, v1, seat.base + from), o2 = __shfl_sync(~0u, v2, seat.base + from);
        w2 = max(min(w1, o1), max(w2, o2));
        w1 = max(w1, o1);
      }
      const uint32_t w = a.top2 && a.per_group > 1 ? w1 + w2 : w1;
      uint32_t before = 0;  // groups that are better, or as good and before it
#pragma unroll 4
      for (uint32_t h = 0; h < a.groups; ++h) {
        const uint32_t o = __shfl_sync(~0u, w, seat.base + h * a.lanes.d);
        before += o > w || (o == w && h < seat.group);
      }
      open = open && before < a.top_groups;
      if (scored) {
        // A place is off by 0.8 at most: its rounding, and the series' 2.8e-10 of a score (twice of a
        // softmax) times 2^29; two sums of two places are in doubt within 4.
        const uint32_t in = ~lanes_top<LPT>(open ? ~w : 0u), out = lanes_top<LPT>(seat.n && !open ? w : 0u);
        if (in <= out + 4) doubt = true;
      }
    }

    const bool exact = kHalf && !keyed;
    if (keyed) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) key[i] = key[i] << kLow | (NPL - 1 - i);
    } else if (exact) {
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const uint32_t b = half_bits<T>(x[i]);
        key[i] = (((b & 0x8000u) ? ~b & 0xffffu : b | 0x8000u) << 16) | (kSlots - 1 - (seat.lane * NPL + i));
      }
    } else {
      // the range from the largest logit down to one that top_k + 1 others reach
      float hi = -INFINITY, lo = INFINITY;
#pragma unroll
      for (int i = 0; i < NPL; ++i)
        if (i < (int)seat.n) {
          hi = fmaxf(hi, x[i]);
          lo = fminf(lo, x[i]);
        }
      const uint32_t lanes = __popc(__ballot_sync(~0u, open) >> seat.base & kLanes<LPT>);
      const float top = lanes_top<LPT>(open ? hi : -INFINITY);
      lo = -lanes_top<LPT>(open ? -(a.top_k < lanes ? hi : lo) : -INFINITY);
      lo = fmaxf(lo, top - 64.f);
      const float by = (kPlaces - 64.f) * rcp(fmaxf(top - lo, 1e-30f));
      // rounding to places keeps the order, or makes logits equal
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        const uint32_t f = (uint32_t)fminf(fmaxf(fmaf(x[i] - lo, by, 16.f), 1.f), kPlaces);
        key[i] = f << kShift | (kSlots - 1 - (seat.lane * NPL + i));
      }
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i)
      if (!open || i >= (int)seat.n) key[i] = 0;

    uint32_t won = 0;  // of rank `lane`; and of the first one not chosen
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
    uint32_t from = 0;  // the lane it is from
    for (uint32_t r = 0; r <= a.top_k; ++r) {
      const uint32_t best = lanes_top<LPT>(key[0]);
      // (scores' places of several lanes may be equal: the lowest lane's counts)
      const uint32_t owner = __ffs(__ballot_sync(~0u, key[0] == best) >> seat.base) - 1;
      if (seat.lane == r) {
        won = best;
        from = owner;
      }
      if (seat.lane == owner) {
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
    if (!exact) {
      const int down = keyed ? kLow : kShift;
      const uint32_t f = won >> down, next = __shfl_down_sync(~0u, f, 1);
      if (seat.lane < a.top_k && (f < 8 || (next != 0 && f - next <= (keyed ? 2u : 0u)))) doubt = true;
    }
    uint32_t slot = keyed ? from * NPL + (NPL - 1 - (won & ((1u << kLow) - 1)))
                          : kSlots - 1 - (won & ((1u << (exact ? 16 : kShift)) - 1));
    // (the whole warp takes part; a token that is not in doubt keeps what it has, whatever is beside it)
    if (__any_sync(~0u, (doubt || odd) && live && !later)) {
      uint32_t again = slot;
      const bool close = resolve<T, NPL, LPT, GROUPED>(a, row, live, seat, keyed, &again);
      const uint32_t asked = __ballot_sync(~0u, doubt || odd), open_still = __ballot_sync(~0u, odd || close);
      if ((asked >> seat.base & kLanes<LPT>) != 0) {
        slot = again;
        later = later || (open_still >> seat.base & kLanes<LPT>) != 0;
      }
    }
    if (later && live && seat.lane == 0) which[atomicAdd(&left, 1u)] = (uint16_t)(step * kTokens + sub);

    // weights from the chosen logits, a lane each
    const bool mine = seat.lane < a.top_k && live && !later;
    float v = -INFINITY, sc = 0.f;
    if (mine) {
      const uint32_t e = expert_of<NPL>(a, slot);
      v = to_f(row[e]);
      if (a.wide) static_cast<int64_t*>(a.experts)[t * a.es + seat.lane * a.ek] = e;
      else static_cast<int32_t*>(a.experts)[t * a.es + seat.lane * a.ek] = (int32_t)e;
    }
    if (SIGMOID) {
      sc = mine ? rcp(1.f + expf(-v)) : 0.f;
      // below -60, on the way out of 32 bits, by e^v, and shares over the largest chosen
      const uint32_t low = __ballot_sync(~0u, mine && v < -60.f);
      if (low != 0) {
        const float over = sigmoid_over(v, a.renorm ? fminf(lanes_top<LPT>(v), 0.f) : 0.f);
        if ((low >> seat.base & kLanes<LPT>) != 0) sc = over;  // (other tokens of the warp keep theirs)
      }
    } else if (a.renorm) {
      // The chosen may lie far below the row's largest logit, where scores leave 32 bits: their shares
      // are the softmax of the chosen alone.  (Ordered by logits, the chosen have the largest.)
      const float top = scored ? lanes_top<LPT>(v) : m;
      if (mine && top != -INFINITY) sc = expf(v - top);
    } else if (mine && m != -INFINITY) {
      sc = expf(v - m) * rcp(total);
    }
    if (a.renorm) {
      // the share first: the scale over the sum may leave 32 bits.  The sum is 0 or at least e^-60, so
      // it has an inverse.
      const float sum = lanes_sum<LPT>(sc);
      sc = sum == 0.f ? 0.f : sc * __frcp_rn(sum);
    }
    if (mine) a.weights[t * a.ws + seat.lane * a.wk] = sc * a.scale;
  }

  __syncthreads();
  Key64* key = reinterpret_cast<Key64*>(smem) + (threadIdx.x / 32) * (a.n + a.groups);
  for (uint32_t i = threadIdx.x / 32; i < left && threadIdx.x / 32 < a.exact_warps; i += a.exact_warps) {
    const uint32_t step = which[i] / kTokens, token = which[i] - step * kTokens;
    route_exact<T>(a, keyed, ((int64_t)step * gridDim.x + blockIdx.x) * kTokens + token, key, key + a.n);
  }
}

struct Chosen {
  float value;
  uint32_t expert;
};

// The gradient of the weights through the chosen scores:
//   renormalised, S the sum of the chosen:  ds_j = scale (g_j - sum_i g_i s_i / S) / S,  else scale g_j
//   sigmoid:  dx_j = ds_j s_j (1 - s_j)
//   softmax:  dx_e = s_e (ds_e - sum_i ds_i s_i)        (ds = 0 where not chosen)
// Of a renormalised softmax the last sum is 0 and s / S is the softmax of the
// chosen logits alone; so only a plain softmax needs the whole row.
template <typename T, int NPL, int LPT>
__global__ void __launch_bounds__(kThreads, NPL <= 8 ? 4 : 1)
gpuos_route_grad_kernel(const __grid_constant__ RouteArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];
  constexpr uint32_t kTokens = kThreads / LPT;
  constexpr int NR = LPT == 32 ? kMaxTop / 32 : 1;
  const uint32_t sub = threadIdx.x / LPT, lane = threadIdx.x % LPT;
  float* dense = reinterpret_cast<float*>(smem) + sub * (LPT * NPL);
  Chosen* chosen = reinterpret_cast<Chosen*>(reinterpret_cast<float*>(smem) + kThreads * NPL) + sub * a.top_k;
  const uint32_t at = lane * NPL, n = at < a.n ? min((uint32_t)NPL, a.n - at) : 0u;
  const bool whole = !a.sigmoid && !a.renorm;
  for (int64_t t0 = (int64_t)blockIdx.x * kTokens; t0 < a.tokens; t0 += (int64_t)gridDim.x * kTokens) {
    const int64_t t = t0 + sub;
    const bool live = t < a.tokens;
    const T* row = static_cast<const T*>(a.x) + (live ? t * a.xs : 0);
    // the chosen ones, a lane each
    float g[NR], v[NR];
    uint32_t e[NR];
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const uint32_t r = lane + i * LPT;
      g[i] = 0.f;
      v[i] = -INFINITY;
      e[i] = ~0u;
      if (r >= a.top_k || !live) continue;
      const int64_t w = a.wide ? static_cast<const int64_t*>(a.experts)[t * a.es + r * a.ek]
                               : (int64_t)static_cast<const int32_t*>(a.experts)[t * a.es + r * a.ek];
      if (w < 0 || w >= a.n) continue;
      e[i] = (uint32_t)w;
      g[i] = a.gw[t * a.gs + r * a.gk];
      v[i] = to_f(row[w]);
    }
    float p[NPL], m = -INFINITY, by = 1.f;
    if (whole) {
      load_logits<T, NPL>(row, at, n, a.vec, live, p);
#pragma unroll
      for (int i = 0; i < NPL; ++i) m = fmaxf(m, p[i]);
      m = lanes_top<LPT>(m);
      const float shift = m == -INFINITY ? 0.f : m;
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < NPL; ++i) {
        p[i] = ex2((p[i] - shift) * kLog2e);
        total += p[i];
      }
      total = lanes_sum<LPT>(total);
      by = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
      for (int i = 0; i < NPL; ++i) p[i] *= by;
    } else {
#pragma unroll
      for (int i = 0; i < NR; ++i) m = fmaxf(m, v[i]);
      m = lanes_top<LPT>(m);
      if (a.sigmoid) m = fminf(m, 0.f);
    }
    float sc[NR], sum = 0.f, dot = 0.f;
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      if (a.sigmoid) sc[i] = a.renorm ? sigmoid_over(v[i], m) : sigmoid(v[i]);
      else sc[i] = m == -INFINITY || e[i] == ~0u ? 0.f : expf(v[i] - m) * by;
      sum += sc[i];
      dot += g[i] * sc[i];
    }
    sum = lanes_sum<LPT>(sum);
    dot = lanes_sum<LPT>(dot);
    // (as in the forward: the sum is 0 or at least a half)
    const float over = !a.renorm || sum == 0.f ? 0.f : __frcp_rn(sum), less = dot * over;
    const float all = a.scale * dot;  // of a plain softmax: the sum of ds_i s_i
#pragma unroll
    for (int i = 0; i < NR; ++i) {
      const uint32_t r = lane + i * LPT;
      float d = a.scale * (g[i] - less);
      if (a.renorm) d *= sc[i] * over;
      else if (a.sigmoid) d *= sc[i];
      if (a.sigmoid) {
        const float x = expf(-fabsf(v[i])), q = 1.f / (1.f + x);
        d *= v[i] > 0.f ? x * q : q;  // 1 - s
      }
      if (r < a.top_k) chosen[r] = Chosen{d, e[i]};
    }
#pragma unroll
    for (int i = 0; i < NPL; ++i) dense[at + i] = 0.f;
    __syncwarp();
    // in order of rank, so that an expert named twice adds up the same way each time
    for (uint32_t r = 0; r < a.top_k; ++r) {
      const Chosen c = chosen[r];
      if (c.expert / NPL == lane) dense[c.expert] += c.value;
    }
    float d[NPL];
#pragma unroll
    for (int i = 0; i < NPL; ++i) {
      d[i] = dense[at + i];
      if (whole) d[i] = p[i] == 0.f ? 0.f : p[i] * (d[i] - all);
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
          if (k < (int)n) store_pack<T, W>(o + at + k, q);
        }
      } else {
#pragma unroll
        for (int i = 0; i < NPL; ++i)
          if (i < (int)n) o[at + i] = from_f<T>(d[i]);
      }
    }
    __syncwarp();
  }
}

template <typename T, int NPL, int LPT>
void launch(RouteArgs a, bool grad, cudaStream_t s) {
  constexpr uint32_t kTokens = kThreads / LPT;
  const uint64_t ctas = ((uint64_t)a.tokens + kTokens - 1) / kTokens;
  // weights: CTAs that stay, as each first looks at the bias, but take at most kCtaTokens
  // (16384 x 256 with one: 17.8 us, 19.6 with a CTA for each step; without one 32749 x 128: 14.6 and 15.6);
  // their gradient has nothing to set up (8.9 us of CTAs of a step, 9.5 of CTAs that stay)
  uint64_t wanted = ctas;
  if (!grad) {
    const uint64_t most = kCtaTokens / kTokens;
    wanted = std::max<uint64_t>(std::min<uint64_t>(ctas, (uint64_t)sm_count() * 8), (ctas + most - 1) / most);
  }
  need(wanted < 0x7fffffffull, "too many tokens");
  const unsigned grid = (unsigned)wanted;
  a.seat_groups = a.groups;
  a.seat_per_group = a.per_group;
  if (a.groups * ((a.per_group + NPL - 1) / NPL) > LPT) {
    a.seat_groups = 1;
    a.seat_per_group = a.n;
  }
  a.lanes = FastDiv((a.seat_per_group + NPL - 1) / NPL);
  if (grad) {
    // (36 KB at most)
    const size_t smem = kThreads * NPL * sizeof(float) + kTokens * a.top_k * sizeof(Chosen);
    run(gpuos_route_grad_kernel<T, NPL, LPT>, grid, kThreads, smem, s, a);
  } else {
    // 18 KB of keys: 8 warps of 256 experts, fewer of more
    const size_t keys = (a.n + a.groups) * sizeof(Key64);
    a.exact_warps = (uint32_t)std::max<size_t>(1, std::min<size_t>(kThreads / 32, 18 * 1024 / keys));
    const size_t smem = a.exact_warps * keys;
    if (a.groups > 1 && a.sigmoid) run(gpuos_route_kernel<T, NPL, LPT, true, true>, grid, kThreads, smem, s, a);
    else if (a.groups > 1) run(gpuos_route_kernel<T, NPL, LPT, true, false>, grid, kThreads, smem, s, a);
    else if (a.sigmoid) run(gpuos_route_kernel<T, NPL, LPT, false, true>, grid, kThreads, smem, s, a);
    else run(gpuos_route_kernel<T, NPL, LPT, false, false>, grid, kThreads, smem, s, a);
  }
}

// Lanes a token needs with NPL experts a lane, none of two groups.
uint32_t lanes_for(const RouteArgs& a, uint32_t npl) { return a.groups * ((a.per_group + npl - 1) / npl); }

template <typename T>
void by_size(const RouteArgs& a, bool grad, cudaStream_t s) {
  // a lane for each rank and the first one not chosen; as few lanes as hold the experts, so that a warp
  // serves several tokens
  const uint32_t lanes = std::max(lanes_for(a, 8), std::min<uint32_t>(a.top_k + 1, 32));
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
