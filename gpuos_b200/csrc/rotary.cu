// gpuos_rotary: rotary positions on one or two tensors (queries and keys) of
// the same tokens, in one launch.
//
//   angle a = p * f_i,  c = scale * cos a,  d = scale * sin a
//   (x1, x2) -> (x1 c - x2 d, x2 c + x1 d)      pair i of the first R elements
//
// and the elements from R on are copied.  The inverse takes -d: the rotation
// is orthogonal (up to scale), so that is the gradient too.
//
// Angles are p * f_i in 64 bits, reduced to turns there: p reaches millions,
// where a 32-bit product is off by whole radians.  What is left, at most half
// a turn, is rounded to 32 bits (2^-25 turns) for sincospif.
//
// One CTA takes whole tokens: it computes the tokens' (c, d) once into shared
// memory and every head reads them there, so the sines cost R/2 evaluations a
// token, not R/2 a head, and the kernel is left with its bytes: x once in, once
// out.  The first items' loads are in flight while the sines are computed.
#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

constexpr int kThreads = 256;
constexpr int kItems = 4;           // items a thread has in flight
constexpr int kTablePairs = 2048;   // (c, d) pairs a CTA holds: 16 KB

struct RotTensor {
  const void* x;
  void* o;
  int64_t xs0, xs1, xh, os0, os1, oh;  // element strides: outer token, inner token, head
  uint32_t items;                      // per token: heads * per_head
  FastDiv per_head;
  uint32_t copies;                     // items of a head from `turned` on are copied
};

struct RotArgs {
  RotTensor t[2];
  const void* pos;
  const void* freq;
  int64_t ps0, ps1, fs;
  int64_t tokens;
  int64_t inner;        // tokens of the inner token dim
  uint32_t half;        // pairs
  uint32_t turned;      // items of a head that are rotated
  uint32_t tile;        // tokens a CTA takes
  uint32_t split;       // CTAs that share a tile's items
  FastDiv token_items;
  FastDiv half_div;
  float scale;
  int pos_wide, freq_wide;
};

// V elements of x1 and of x2 (half layout), or V interleaved elements.  VL is
// what one access moves.
template <typename T, int V, int VL>
__device__ __forceinline__ void fetch(const T* p, Pack<T, V>& r) {
#pragma unroll
  for (int k = 0; k < V; k += VL) {
    const Pack<T, VL> q = load_pack<T, VL>(p + k);
#pragma unroll
    for (int i = 0; i < VL; ++i) r.v[k + i] = q.v[i];
  }
}

template <typename T, int V, int VL>
__device__ __forceinline__ void put(T* p, const Pack<T, V>& r) {
#pragma unroll
  for (int k = 0; k < V; k += VL) {
    Pack<T, VL> q;
#pragma unroll
    for (int i = 0; i < VL; ++i) q.v[i] = r.v[k + i];
    store_pack<T, VL>(p + k, q);
  }
}

struct Item {
  uint32_t token;  // of the tile
  uint32_t j;      // of the head
  int64_t xo, oo;  // element offsets of the item's first element
  int which;
  bool turn;
};

template <int V, bool INTER>
__device__ __forceinline__ Item locate(const RotArgs& a, uint32_t it, int64_t tok0) {
  Item r;
  r.token = a.token_items.div(it);
  uint32_t m = it - r.token * a.token_items.d;
  r.which = m >= a.t[0].items;
  if (r.which) m -= a.t[0].items;
  const RotTensor& t = a.t[r.which];
  const uint32_t head = t.per_head.div(m);
  r.j = m - head * t.per_head.d;
  r.turn = r.j < a.turned;
  const int64_t token = tok0 + r.token;
  int64_t outer = 0, inner = token;
  if (a.inner != a.tokens) {
    outer = token / a.inner;
    inner = token - outer * a.inner;
  }
  // rotated items step by V; the copied part starts behind all R elements
  const int64_t e = r.turn ? (int64_t)r.j * V
                           : 2 * (int64_t)a.half + (int64_t)(r.j - a.turned) * V;
  r.xo = outer * t.xs0 + inner * t.xs1 + head * t.xh + e;
  r.oo = outer * t.os0 + inner * t.os1 + head * t.oh + e;
  return r;
}

// The table holds for item j of a head the V (half layout) or V/2 pairs it
// needs, chunk k of two pairs at [k][j], so that neighbouring lanes read
// neighbouring 16 bytes.
template <int P>
__device__ __forceinline__ uint32_t table_at(uint32_t token, uint32_t pair, uint32_t half) {
  if constexpr (P == 1) return token * half + pair;
  const uint32_t j = pair / P, i = pair % P;
  return token * half + (i / 2) * (half / P) * 2 + j * 2 + (i & 1);
}

template <typename T, int V, int VL, bool INTER>
__global__ void __launch_bounds__(kThreads)
gpuos_rotary_kernel(const __grid_constant__ RotArgs a) {
  constexpr int P = INTER ? V / 2 : V;  // pairs an item rotates
  __shared__ __align__(16) float2 table[kTablePairs];
  const uint32_t tile = blockIdx.x / a.split, part = blockIdx.x - tile * a.split;
  const int64_t tok0 = (int64_t)tile * a.tile;
  const uint32_t ntok = (uint32_t)min((int64_t)a.tile, a.tokens - tok0);
  const uint32_t all = ntok * a.token_items.d;
  const uint32_t lo = (uint32_t)((uint64_t)all * part / a.split);
  const uint32_t hi = (uint32_t)((uint64_t)all * (part + 1) / a.split);

  Item item[kItems];
  Pack<T, V> x1[kItems], x2[kItems];
  auto load = [&](uint32_t base) {
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const uint32_t it = base + u * kThreads + threadIdx.x;
      if (it >= hi) break;
      item[u] = locate<V, INTER>(a, it, tok0);
      const T* p = static_cast<const T*>(a.t[item[u].which].x) + item[u].xo;
      fetch<T, V, VL>(p, x1[u]);
      if (!INTER && item[u].turn) fetch<T, V, VL>(p + a.half, x2[u]);
    }
  };
  load(lo);

  for (uint32_t k = threadIdx.x; k < ntok * a.half; k += kThreads) {
    const uint32_t tok = a.half_div.div(k), pair = k - tok * a.half;
    const int64_t token = tok0 + tok;
    int64_t outer = 0, inner = token;
    if (a.inner != a.tokens) {
      outer = token / a.inner;
      inner = token - outer * a.inner;
    }
    const int64_t p = load_index(a.pos, a.pos_wide, outer * a.ps0 + inner * a.ps1);
    const double f = a.freq_wide ? static_cast<const double*>(a.freq)[pair * a.fs]
                                 : (double)static_cast<const float*>(a.freq)[pair * a.fs];
    const double turns = (double)p * f * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    table[table_at<P>(tok, pair, a.half)] = make_float2(c * fabsf(a.scale), s * a.scale);
  }
  __syncthreads();

  for (uint32_t base = lo; base < hi; base += kItems * kThreads) {
    if (base != lo) load(base);
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const uint32_t it = base + u * kThreads + threadIdx.x;
      if (it >= hi) break;
      T* o = static_cast<T*>(a.t[item[u].which].o) + item[u].oo;
      if (!item[u].turn) {
        put<T, V, VL>(o, x1[u]);
        continue;
      }
      const float2* tab = table + item[u].token * a.half;
      float2 cd[P];
      if constexpr (P == 1) {
        cd[0] = tab[item[u].j];
      } else {
#pragma unroll
        for (int k = 0; k < P / 2; ++k) {
          const float4 q = *reinterpret_cast<const float4*>(tab + (k * (a.half / P) + item[u].j) * 2);
          cd[2 * k] = make_float2(q.x, q.y);
          cd[2 * k + 1] = make_float2(q.z, q.w);
        }
      }
      Pack<T, V> y1, y2;
#pragma unroll
      for (int i = 0; i < P; ++i) {
        const float p = to_f(INTER ? x1[u].v[2 * i] : x1[u].v[i]);
        const float q = to_f(INTER ? x1[u].v[2 * i + 1] : x2[u].v[i]);
        const T r = from_f<T>(p * cd[i].x - q * cd[i].y), w = from_f<T>(q * cd[i].x + p * cd[i].y);
        if (INTER) {
          y1.v[2 * i] = r;
          y1.v[2 * i + 1] = w;
        } else {
          y1.v[i] = r;
          y2.v[i] = w;
        }
      }
      put<T, V, VL>(o, y1);
      if (!INTER) put<T, V, VL>(o + a.half, y2);
    }
  }
}

template <typename T>
void launch(const RotArgs& a, int v, int vl, bool inter, unsigned grid, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);
#define GPUOS_ROT(V, VL, I) gpuos_rotary_kernel<T, V, VL, I><<<grid, kThreads, 0, s>>>(a)
  if (inter) {
    if (v == W) GPUOS_ROT(W, W, true);
    else if (vl == 2) GPUOS_ROT(2, 2, true);
    else GPUOS_ROT(2, 1, true);
  } else {
    if (v == W) GPUOS_ROT(W, W, false);
    else if (v == 2) GPUOS_ROT(2, 2, false);
    else GPUOS_ROT(1, 1, false);
  }
#undef GPUOS_ROT
}

void rotary(int32_t n, const gpuos_tensor* x, const gpuos_tensor* out, const gpuos_tensor* positions,
            const gpuos_tensor* inv_freq, float scale, int32_t flags, cudaStream_t stream) {
  need(n == 1 || n == 2, "takes one or two tensors");
  need(x && out && positions && inv_freq, "NULL tensor");
  need((flags & ~(GPUOS_ROTARY_INTERLEAVED | GPUOS_ROTARY_INVERSE)) == 0, "unknown flag");
  need(std::abs(scale) <= 3.4028234e38f && scale >= 0.f, "scale must be finite and not negative");
  const bool inter = flags & GPUOS_ROTARY_INTERLEAVED;
  check_tensor(inv_freq, 1, "inv_freq");
  need(inv_freq->dtype == GPUOS_F64 || inv_freq->dtype == GPUOS_F32, "inv_freq must be float64 or float32");
  need(is_index(positions->dtype), "positions must be int32 or int64");
  const int64_t half = inv_freq->sizes[0];
  const int nd = x[0].ndim;
  need(nd == 3 || nd == 4, "x must have 3 dims (token, head, element) or 4 (batch, token, head, element)");
  check_tensor(positions, nd - 2, "positions");
  RotArgs a{};
  int W = 16 / esize(x[0].dtype), vec = W, pair = 2;
  for (int i = 0; i < n; ++i) {
    check_tensor(&x[i], nd, "x");
    check_tensor(&out[i], nd, "out");
    need(is_real(x[i].dtype), "x must be float32, float16 or bfloat16");
    need(x[i].dtype == x[0].dtype && out[i].dtype == x[0].dtype, "x and out must have one dtype");
    same_sizes(x[i], out[i], "out must have the sizes of x");
    for (int d = 0; d < nd - 2; ++d) {
      need(x[i].sizes[d] == x[0].sizes[d], "the tensors must have the same tokens");
      need(x[i].sizes[d] == positions->sizes[d], "positions must have x's token sizes");
    }
    const int64_t head = x[i].sizes[nd - 1];
    need(head < (1 << 20) && x[i].sizes[nd - 2] < (1 << 20), "too many heads or elements");
    need(2 * half <= head, "inv_freq has more pairs than the head has elements");
    if (head > 1 && numel(x[i]))
      need(x[i].strides[nd - 1] == 1 && out[i].strides[nd - 1] == 1,
           "the last dim of x and out must be contiguous");
    check_output(out[i], "out");
  }
  need(half <= kTablePairs, "inv_freq has more than 2048 pairs");
  for (int i = 0; i < n; ++i) {
    need(same_view(x[i], out[i]) || !overlap(x[i], out[i]), "out must be x or not overlap it");
    need(!overlap(out[i], *positions) && !overlap(out[i], *inv_freq), "out overlaps an input");
    for (int k = 0; k < n; ++k)
      if (k != i) {
        need(!overlap(out[i], x[k]), "out overlaps another input");
        need(!overlap(out[i], out[k]), "the outputs overlap");
      }
  }
  // 16-byte items where pointers, strides, the rotated and the copied part
  // allow it, else two elements at a time, else one
  for (int i = 0; i < n; ++i) {
    if (numel(x[i]) == 0) continue;
    const int64_t rest = x[i].sizes[nd - 1] - 2 * half;
    auto fits = [&](int v) {
      return rows_aligned(x[i], v) && rows_aligned(out[i], v) && rest % v == 0 &&
             (inter ? 2 * half : half) % v == 0;
    };
    if (vec > 2 && !fits(vec)) vec = 2;
    if (!fits(2)) pair = 1;
  }
  int v = vec, vl = vec;
  if (vec == 2) {
    vl = pair;
    v = inter ? 2 : pair;
  }
  if (inter && v == 2 && vl == 1)  // scalar accesses still move two elements at a time
    for (int i = 0; i < n; ++i) need((x[i].sizes[nd - 1] - 2 * half) % 2 == 0, "interleaved pairs need an even head size");

  uint64_t per_token = 0;
  a.half = (uint32_t)half;
  a.turned = (uint32_t)(inter ? 2 * half / v : half / v);
  a.inner = x[0].sizes[nd - 3];
  a.tokens = nd == 4 ? x[0].sizes[0] * a.inner : a.inner;
  for (int i = 0; i < n; ++i) {
    RotTensor& t = a.t[i];
    const bool four = nd == 4;
    t.x = x[i].data;
    t.o = out[i].data;
    t.xs0 = four ? x[i].strides[0] : 0;
    t.os0 = four ? out[i].strides[0] : 0;
    t.xs1 = x[i].strides[nd - 3];
    t.os1 = out[i].strides[nd - 3];
    t.xh = x[i].strides[nd - 2];
    t.oh = out[i].strides[nd - 2];
    const int64_t rest = x[i].sizes[nd - 1] - 2 * half;
    // in place the part that is not rotated is there already
    const uint32_t per_head = a.turned + (same_view(x[i], out[i]) ? 0 : (uint32_t)(rest / v));
    t.per_head = FastDiv(std::max(per_head, 1u));
    t.items = (uint32_t)x[i].sizes[nd - 2] * per_head;
    per_token += (uint64_t)x[i].sizes[nd - 2] * per_head;
  }
  if (a.tokens == 0 || per_token == 0) return;
  need(per_token < (1u << 24), "a token has too many elements");
  a.pos = positions->data;
  a.ps0 = nd == 4 ? positions->strides[0] : 0;
  a.ps1 = positions->strides[nd - 3];
  a.pos_wide = positions->dtype == GPUOS_I64;
  a.freq = inv_freq->data;
  a.fs = half ? inv_freq->strides[0] : 0;
  a.freq_wide = inv_freq->dtype == GPUOS_F64;
  a.scale = (flags & GPUOS_ROTARY_INVERSE) ? -scale : scale;
  a.token_items = FastDiv((uint32_t)per_token);
  a.half_div = FastDiv(std::max<uint32_t>(a.half, 1));

  // A CTA takes the tokens that give each thread its items; few tokens are
  // split over more CTAs, one item a thread, so that a decode step's loads
  // start on many SMs at once.
  const int sms = sm_count();
  const uint64_t full = kItems * kThreads;
  uint64_t tile = std::max<uint64_t>(1, full / per_token);
  if (half) tile = std::min<uint64_t>(tile, kTablePairs / half);
  const uint64_t spread = std::max<uint64_t>(1, (uint64_t)a.tokens / (2 * sms));
  tile = std::min(tile, spread);
  const uint64_t tiles = ((uint64_t)a.tokens + tile - 1) / tile;
  uint64_t split = 1;
  if (tiles < (uint64_t)sms)
    split = std::max<uint64_t>(1, std::min<uint64_t>((tile * per_token + kThreads - 1) / kThreads,
                                                     2 * sms / tiles));
  need(tiles * split < 0x7fffffffull, "too many tokens");
  a.tile = (uint32_t)tile;
  a.split = (uint32_t)split;
  const unsigned grid = (unsigned)(tiles * split);
  if (x[0].dtype == GPUOS_F32) launch<float>(a, v, vl, inter, grid, stream);
  else if (x[0].dtype == GPUOS_F16) launch<__half>(a, v, vl, inter, grid, stream);
  else launch<__nv_bfloat16>(a, v, vl, inter, grid, stream);
  cuda_ok(cudaGetLastError(), "launch");
}

}  // namespace
}  // namespace rowops
}  // namespace gpuos

extern "C" int32_t gpuos_rotary(int32_t n, const gpuos_tensor* x, const gpuos_tensor* out,
                                const gpuos_tensor* positions, const gpuos_tensor* inv_freq,
                                float scale, int32_t flags, void* stream) {
  return gpuos::rowops::entry("gpuos_rotary", [&] {
    gpuos::rowops::rotary(n, x, out, positions, inv_freq, scale, flags, static_cast<cudaStream_t>(stream));
  });
}
