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
// A thread belongs to one token and one group of V elements (16 bytes where
// alignment allows) and walks over the heads in steps: its pairs' (c, d) stay in
// registers, and a head costs its loads, the arithmetic and its stores.  The
// CTA computes the (c, d) of its tokens once, into shared memory, while the first
// heads' loads are in flight: R/2 sines a token, not R/2 a head.  What is left are the
// bytes: x once in, once out.  16384 tokens x 64 heads x 128 bf16 take 93.5 us (5.7 TB/s), 9001 x 40 x
// 128 fp16 with half of it rotated 35 us (5.3 TB/s), a decode step of 8 tokens 2.4 us.
#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

constexpr int kThreads = 256;
constexpr int kTablePairs = 2048;   // (c, d) pairs a CTA holds: 16 KB

struct RotTensor {
  const void* x;
  void* o;
  int64_t xs0, xs1, xh, os0, os1, oh;  // element strides: outer token, inner token, head
  uint32_t heads;
  uint32_t copies;                     // groups of V elements behind the rotated ones
};

struct RotArgs {
  RotTensor t[2];
  const void* pos;
  const void* freq;
  int64_t ps0, ps1, fs;
  uint32_t tokens;
  FastDiv inner;        // tokens of the inner token dim
  FastDiv half;         // pairs
  uint32_t units;       // groups of V elements (of x1 in the half layout) that are rotated
  FastDiv lanes;        // threads side by side over a head's groups
  FastDiv per_token;    // threads of a token: lanes * head groups
  uint32_t head_step;   // head groups of all CTAs that share a token
  uint32_t tile;        // tokens a CTA takes
  uint32_t two;         // 1: two heads in flight (interleaved, nothing copied)
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

// The table holds for item j of a head the V (half layout) or V/2 pairs it
// needs, chunk k of two pairs at [k][j], so that neighbouring lanes read
// neighbouring 16 bytes.
template <int P>
__device__ __forceinline__ uint32_t table_at(uint32_t token, uint32_t pair, uint32_t half) {
  if constexpr (P == 1) return token * half + pair;
  const uint32_t j = pair / P, i = pair % P;
  return token * half + (i / 2) * (half / P) * 2 + j * 2 + (i & 1);
}

template <typename T>
__device__ __forceinline__ void turn(T& first, T& second, float2 cd) {
  const float v = to_f(first), w = to_f(second);
  first = from_f<T>(v * cd.x - w * cd.y);
  second = from_f<T>(w * cd.x + v * cd.y);
}

template <typename T, int V, int VL, bool INTER>
__global__ void __launch_bounds__(kThreads)
gpuos_rotary_kernel(const __grid_constant__ RotArgs a) {
  constexpr int P = INTER ? V / 2 : V;  // pairs of a group
  __shared__ __align__(16) float2 table[kTablePairs];
  const uint32_t half = a.half.d;
  const uint32_t tok0 = blockIdx.x * a.tile;
  const uint32_t ntok = min(a.tile, a.tokens - tok0);
  const uint32_t mine = a.per_token.div(threadIdx.x);  // token of the tile
  const uint32_t rest = threadIdx.x - mine * a.per_token.d;
  const uint32_t group = a.lanes.div(rest), j0 = rest - group * a.lanes.d;
  const uint32_t h0 = group + blockIdx.y * (a.per_token.d / a.lanes.d);
  const bool live = mine < ntok;
  const uint32_t heads = a.t[0].heads + a.t[1].heads;

  // the token's rows
  const T *x0 = nullptr, *x1 = nullptr;
  T *o0 = nullptr, *o1 = nullptr;
  if (live) {
    const uint32_t outer = a.inner.div(tok0 + mine), in = tok0 + mine - outer * a.inner.d;
    x0 = static_cast<const T*>(a.t[0].x) + outer * a.t[0].xs0 + in * a.t[0].xs1;
    x1 = static_cast<const T*>(a.t[1].x) + outer * a.t[1].xs0 + in * a.t[1].xs1;
    o0 = static_cast<T*>(a.t[0].o) + outer * a.t[0].os0 + in * a.t[0].os1;
    o1 = static_cast<T*>(a.t[1].o) + outer * a.t[1].os0 + in * a.t[1].os1;
  }
  auto from = [&](uint32_t h) {
    return h < a.t[0].heads ? x0 + h * a.t[0].xh : x1 + (h - a.t[0].heads) * a.t[1].xh;
  };
  auto to = [&](uint32_t h) {
    return h < a.t[0].heads ? o0 + h * a.t[0].oh : o1 + (h - a.t[0].heads) * a.t[1].oh;
  };

  // a rotated group (both halves), and the group of the copied part with its number
  Pack<T, V> p, q, r;
  auto load = [&](uint32_t h, uint32_t j) {
    const T* x = from(h) + j * V;
    fetch<T, V, VL>(x, p);
    if (!INTER) fetch<T, V, VL>(x + half, q);
    else if (a.two && h + a.head_step < heads) fetch<T, V, VL>(from(h + a.head_step) + j * V, q);
    if (j < a.t[h >= a.t[0].heads].copies) fetch<T, V, VL>(x + 2 * half, r);
  };
  if (live && j0 < a.units && h0 < heads) load(h0, j0);

  for (uint32_t k = threadIdx.x; k < ntok * half; k += kThreads) {
    const uint32_t tok = a.half.div(k), pair = k - tok * half;
    const uint32_t outer = a.inner.div(tok0 + tok), in = tok0 + tok - outer * a.inner.d;
    const int64_t at = load_index(a.pos, a.pos_wide, outer * a.ps0 + in * a.ps1);
    const double f = a.freq_wide ? static_cast<const double*>(a.freq)[pair * a.fs]
                                 : (double)static_cast<const float*>(a.freq)[pair * a.fs];
    const double turns = (double)at * f * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    table[table_at<P>(tok, pair, half)] = make_float2(c * fabsf(a.scale), s * a.scale);
  }
  __syncthreads();
  if (!live) return;

  for (uint32_t j = j0; j < a.units; j += a.lanes.d) {
    const float2* tab = table + mine * half;
    float2 cd[P];
    if constexpr (P == 1) {
      cd[0] = tab[j];
    } else {
#pragma unroll
      for (int k = 0; k < P / 2; ++k) {
        const float4 w = *reinterpret_cast<const float4*>(tab + (k * a.units + j) * 2);
        cd[2 * k] = make_float2(w.x, w.y);
        cd[2 * k + 1] = make_float2(w.z, w.w);
      }
    }
    for (uint32_t h = h0; h < heads; h += INTER ? a.head_step << a.two : a.head_step) {
      if (j != j0 || h != h0) load(h, j);
      T* o = to(h) + j * V;
#pragma unroll
      for (int i = 0; i < P; ++i) turn(p.v[INTER ? 2 * i : i], INTER ? p.v[2 * i + 1] : q.v[i], cd[i]);
      put<T, V, VL>(o, p);
      if (!INTER) put<T, V, VL>(o + half, q);
      if (j < a.t[h >= a.t[0].heads].copies) put<T, V, VL>(o + 2 * half, r);
      if constexpr (INTER) {
        if (a.two && h + a.head_step < heads) {
#pragma unroll
          for (int i = 0; i < P; ++i) turn(q.v[2 * i], q.v[2 * i + 1], cd[i]);
          put<T, V, VL>(to(h + a.head_step) + j * V, q);
        }
      }
    }
  }
  // where more is copied than rotated
  if (a.t[0].copies > a.units || a.t[1].copies > a.units) {
    uint32_t from_j = j0;
    while (from_j < a.units) from_j += a.lanes.d;
    for (uint32_t h = h0; h < heads; h += a.head_step) {
      const uint32_t copies = a.t[h >= a.t[0].heads].copies;
      for (uint32_t j = from_j; j < copies; j += a.lanes.d) {
        fetch<T, V, VL>(from(h) + 2 * half + j * V, r);
        put<T, V, VL>(to(h) + 2 * half + j * V, r);
      }
    }
  }
}

template <typename T>
void launch(const RotArgs& a, int v, int vl, bool inter, dim3 grid, cudaStream_t s) {
  constexpr int W = 16 / sizeof(T);
#define GPUOS_ROT(V, VL, I) run(gpuos_rotary_kernel<T, V, VL, I>, grid, kThreads, 0, s, a)
  if (inter) {
    if (v == W) GPUOS_ROT(W, W, true);
    else if (v == W / 2 && vl == W / 2) GPUOS_ROT(W / 2, W / 2, true);
    else if (vl == 2) GPUOS_ROT(2, 2, true);
    else GPUOS_ROT(2, 1, true);
  } else {
    if (v == W) GPUOS_ROT(W, W, false);
    else if (v == W / 2) GPUOS_ROT(W / 2, W / 2, false);
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
  need(half <= kTablePairs, "inv_freq has more than 2048 pairs");
  const int nd = x[0].ndim;
  need(nd == 3 || nd == 4, "x must have 3 dims (token, head, element) or 4 (batch, token, head, element)");
  check_tensor(positions, nd - 2, "positions");
  RotArgs a{};
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
  for (int i = 0; i < n; ++i) {
    need(same_view(x[i], out[i]) || !overlap(x[i], out[i]), "out must be x or not overlap it");
    need(!overlap(out[i], *positions) && !overlap(out[i], *inv_freq), "out overlaps an input");
    for (int k = 0; k < n; ++k)
      if (k != i) {
        need(!overlap(out[i], x[k]), "out overlaps another input");
        need(!overlap(out[i], out[k]), "the outputs overlap");
      }
  }
  // groups of 16 bytes where pointers, strides, the rotated and the copied
  // part allow it, else of 8, else of two elements, else single ones
  const int W = 16 / esize(x[0].dtype);
  int vl = W;
  for (int i = 0; i < n; ++i) {
    if (numel(x[i]) == 0) continue;
    const int64_t rest = x[i].sizes[nd - 1] - 2 * half;
    while (vl > 1 && !(rows_aligned(x[i], vl) && rows_aligned(out[i], vl) && rest % vl == 0 &&
                       (inter ? 2 * half : half) % vl == 0))
      vl = vl > 2 ? std::max(vl / 2, 2) : 1;
  }
  const int v = inter && vl == 1 ? 2 : vl;  // interleaved: single accesses still move a pair
  if (v != vl)
    for (int i = 0; i < n; ++i)
      need((x[i].sizes[nd - 1] - 2 * half) % 2 == 0, "interleaved pairs need an even head size");

  const bool four = nd == 4;
  const __int128 tokens = four ? (__int128)x[0].sizes[0] * x[0].sizes[1] : x[0].sizes[0];
  uint32_t heads = 0, copies = 0;
  for (int i = 0; i < n; ++i) {
    RotTensor& t = a.t[i];
    t.x = x[i].data;
    t.o = out[i].data;
    t.xs0 = four ? x[i].strides[0] : 0;
    t.os0 = four ? out[i].strides[0] : 0;
    t.xs1 = x[i].strides[nd - 3];
    t.os1 = out[i].strides[nd - 3];
    t.xh = x[i].strides[nd - 2];
    t.oh = out[i].strides[nd - 2];
    t.heads = (uint32_t)x[i].sizes[nd - 2];
    // in place the part that is not rotated is there already
    t.copies = same_view(x[i], out[i]) ? 0 : (uint32_t)((x[i].sizes[nd - 1] - 2 * half) / v);
    heads += t.heads;
    copies = std::max(copies, t.copies);
  }
  a.units = (uint32_t)((inter ? 2 * half : half) / v);
  if (tokens == 0 || heads == 0 || (a.units == 0 && copies == 0)) return;
  need(tokens < (__int128)0x7fffffff, "too many tokens");
  a.tokens = (uint32_t)tokens;
  a.inner = FastDiv((uint32_t)x[0].sizes[nd - 3]);
  a.half = FastDiv((uint32_t)half);
  a.pos = positions->data;
  a.ps0 = four ? positions->strides[0] : 0;
  a.ps1 = positions->strides[nd - 3];
  a.pos_wide = positions->dtype == GPUOS_I64;
  a.freq = inv_freq->data;
  a.fs = half ? inv_freq->strides[0] : 0;
  a.freq_wide = inv_freq->dtype == GPUOS_F64;
  a.scale = (flags & GPUOS_ROTARY_INVERSE) ? -scale : scale;

  const Spread sp = spread(a.tokens, a.units ? a.units : copies, heads, kThreads,
                           half ? kTablePairs / (uint32_t)half : kThreads);
  a.lanes = FastDiv(sp.lanes);
  a.per_token = FastDiv(sp.lanes * sp.groups);
  a.head_step = sp.groups * sp.split;
  a.tile = sp.tile;
  // An interleaved group is one load a head, half of what a split one keeps in flight: two heads at once
  // (15715 x 18 x 80 fp32: 37.0 us, 45.5 with one; 9001 x 40 x 128 bf16: 39.8 and 47.5).
  a.two = inter && copies == 0;
  const dim3 grid(sp.tiles, sp.split);
  if (x[0].dtype == GPUOS_F32) launch<float>(a, v, vl, inter, grid, stream);
  else if (x[0].dtype == GPUOS_F16) launch<__half>(a, v, vl, inter, grid, stream);
  else launch<__nv_bfloat16>(a, v, vl, inter, grid, stream);
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
