// gpuos_cache_write / gpuos_cache_read: a paged cache of keys and values held
// in 8 or 4 bits, one scale for each group of G elements of a head's row.
//
//   a     = max |x| over the group's finite elements
//   scale = a * fl(1/Q)            Q = 127 (int8), 448 (e4m3), 7 (int4)
//   inv   = fl(1/a) * Q
//   code  = x * inv rounded to the format, nearest even
//   x'    = code * scale, rounded once to the output type
//
// all in 32-bit arithmetic with a rounding after each step, so the codes are a
// function of the inputs alone: no step may be contracted or reordered.
// Groups below 2^-100 are stored as zeros (their reciprocal leaves the normal
// range), an infinity as the largest code of its sign, NaN as code 0 (int8,
// int4) or NaN (e4m3).
//
// Both kernels move every byte once, 8 elements a lane.  What could bound them
// above that are instructions, so each token's row of the cache is found once by the lanes that
// share the token, which then walk over its heads; a write holds a group in the
// registers of neighbouring lanes and joins its maximum by shuffles.
// 16000 tokens x 2 x 8 heads x 128 bf16 as e4m3: written in 20.4 us, read in 18.3 (99.5 MB each: 4.9 and
// 5.4 TB/s); 100003 tokens of 4 bits in groups of 32 to fp16: read in 96.8 us (5.6 TB/s).
#include <cuda_fp8.h>

#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace {

constexpr int kThreads = 256;
constexpr int kUnit = 8;        // elements a lane moves at once
constexpr int kGroupUnits = 4;  // of them a lane holds of a group

enum Format { kInt8, kE4M3, kInt4 };

struct CacheTensor {
  void* rows;                  // what is written (read only) or read into
  void* codes;
  float* scales;
  uint32_t rs, rh;             // rows: strides of token and head (elements)
  uint32_t cp, cr, ch;         // codes: strides of page, row, head (bytes)
  uint32_t sp, sr, sh, sg;     // scales: strides of page, row, head, group
  uint32_t heads;
  uint32_t head;               // elements
  uint32_t group;              // elements
  uint32_t items;              // write: groups of a token
  FastDiv groups;              // of a head
  FastDiv group_div;           // by `group`
  uint32_t lanes_log;          // write: lanes that share a group
};

struct CacheArgs {
  CacheTensor t[2];
  const void* slots;
  int64_t ss;
  int64_t rows;        // pages * page
  FastDiv page;
  uint32_t tokens;
  uint32_t token_log;  // write: lanes that share a token
  // read: how the threads are spread
  uint32_t tile, head_step;
  FastDiv lanes, per_token;
  int slot_wide;
};

__device__ __forceinline__ uint64_t wide(uint32_t a, uint32_t b) { return (uint64_t)a * b; }

__device__ __forceinline__ float q_max(int f) { return f == kInt8 ? 127.f : f == kE4M3 ? 448.f : 7.f; }

// Nearest-even rounding of |y| < 2^22 to an integer, left in the low bits: one
// addition at full rate where a conversion runs at a quarter of it.
__device__ __forceinline__ uint32_t round_bits(float y) { return __float_as_uint(__fadd_rn(y, 12582912.f)); }

// 8 values to the codes of their format, in order from the lowest bits.
template <int F>
__device__ __forceinline__ uint2 encode(const float (&y)[kUnit]) {
  uint2 r = make_uint2(0, 0);
  if constexpr (F == kInt8) {
    uint32_t b[kUnit];
#pragma unroll
    for (int i = 0; i < kUnit; ++i) b[i] = round_bits(y[i]);
    r.x = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
    r.y = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  } else if constexpr (F == kE4M3) {
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      h[i] = __nv_cvt_float2_to_fp8x2(make_float2(y[2 * i], y[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
    r.x = h[0] | (h[1] << 16);
    r.y = h[2] | (h[3] << 16);
  } else {
    // code + 8 in the low 4 bits: the magic sum's low bits are the code's two's complement
#pragma unroll
    for (int i = 0; i < kUnit; ++i) r.x |= ((round_bits(y[i]) + 8u) & 15u) << (4 * i);
  }
  return r;
}

// The values of 8 codes.  An integer k in the low bits of a float near 2^23
// makes it 2^23 + k exactly; a subtraction gives k back at full rate.
template <int F>
__device__ __forceinline__ void decode(uint2 r, float (&y)[kUnit]) {
  if constexpr (F == kInt8) {
#pragma unroll
    for (int i = 0; i < kUnit; ++i) {
      const uint32_t w = (i < 4 ? r.x : r.y) ^ 0x80808080u;  // code + 128
      y[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7440 | (i & 3))) - 8388736.f;
    }
  } else if constexpr (F == kE4M3) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = i < 2 ? r.x : r.y;
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> (16 * (i & 1))), __NV_E4M3);
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
      y[2 * i] = f.x;
      y[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < kUnit; ++i)
      y[i] = __uint_as_float(0x4b000000u | ((r.x >> (4 * i)) & 15u)) - 8388616.f;
  }
}

template <int F> constexpr int kCodeBits = F == kInt4 ? 4 : 8;

// Codes of the first n of 8 elements.
template <int F, bool VEC>
__device__ __forceinline__ void store_codes(uint8_t* p, uint2 r, int n) {
  if constexpr (VEC) {
    if constexpr (F == kInt4) *reinterpret_cast<uint32_t*>(p) = r.x;
    else *reinterpret_cast<uint2*>(p) = r;
  } else {
    const int bytes = n * kCodeBits<F> / 8;
    for (int i = 0; i < bytes; ++i) p[i] = (uint8_t)((i < 4 ? r.x : r.y) >> (8 * (i & 3)));
  }
}

template <int F, bool VEC>
__device__ __forceinline__ uint2 load_codes(const uint8_t* p, int n) {
  uint2 r = make_uint2(0, 0);
  if constexpr (VEC) {
    if constexpr (F == kInt4) r.x = __ldcs(reinterpret_cast<const uint32_t*>(p));
    else r = __ldcs(reinterpret_cast<const uint2*>(p));
  } else {
    const int bytes = n * kCodeBits<F> / 8;
    for (int i = 0; i < bytes; ++i) {
      if (i < 4) r.x |= (uint32_t)p[i] << (8 * i);
      else r.y |= (uint32_t)p[i] << (8 * (i - 4));
    }
  }
  return r;
}

// 8 elements as they are stored.
template <typename T, bool VEC>
__device__ __forceinline__ void load_unit(const T* p, int n, Pack<T, kUnit>& x) {
  if constexpr (VEC) {
    constexpr int W = 16 / sizeof(T);
#pragma unroll
    for (int k = 0; k < kUnit; k += W) {
      const Pack<T, W> q = load_pack<T, W>(p + k);
#pragma unroll
      for (int i = 0; i < W; ++i) x.v[k + i] = q.v[i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kUnit; ++i) x.v[i] = i < n ? p[i] : from_f<T>(0.f);
  }
}

// max that keeps a NaN: a group with one, or with an infinity, shows it in its
// maximum and takes the careful path below.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// max |x| of 8 elements (16-bit types two at a time).
template <typename T>
__device__ __forceinline__ float max_abs(const Pack<T, kUnit>& x) {
  if constexpr (sizeof(T) == 2) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    const T2* h = reinterpret_cast<const T2*>(&x);
    const T2 m = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
    return max_nan(to_f(m.x), to_f(m.y));
  } else {
    float m = fabsf(x.v[0]);
#pragma unroll
    for (int i = 1; i < kUnit; ++i) m = max_nan(m, fabsf(x.v[i]));
    return m;
  }
}

// A lane holds 4 units of a group, so that what a group costs besides (the
// shuffles of its maximum, its scale, its addresses) is shared by 32 elements: 16000 x 2 x
// 8 x 128 bf16 to e4m3 took 28.8 us with one unit a lane, 23.8 with two, 21.0 with four.
template <typename T, int F, bool VEC>
__global__ void __launch_bounds__(kThreads)
gpuos_cache_write_kernel(const __grid_constant__ CacheArgs a) {
  constexpr int NU = kGroupUnits;
  const CacheTensor& t = a.t[blockIdx.y];
  const uint32_t token = blockIdx.x * (kThreads >> a.token_log) + (threadIdx.x >> a.token_log);
  const uint32_t of_token = threadIdx.x & ((1u << a.token_log) - 1);
  const uint32_t lanes = 1u << t.lanes_log, lane = of_token & (lanes - 1);
  const uint32_t step = 1u << (a.token_log - t.lanes_log);
  const float inf = __int_as_float(0x7f800000), q = q_max(F);

  const bool live = token < a.tokens;
  bool has = false;
  const T* x0 = nullptr;
  uint8_t* codes = nullptr;
  float* scales = nullptr;
  if (live) {
    const int64_t slot = load_index(a.slots, a.slot_wide, token * a.ss);
    has = slot >= 0 && slot < a.rows;  // rows < 2^31
    const uint32_t page = a.page.div((uint32_t)slot), row = (uint32_t)slot - page * a.page.d;
    x0 = static_cast<const T*>(t.rows) + wide(token, t.rs);
    codes = static_cast<uint8_t*>(t.codes) + wide(page, t.cp) + wide(row, t.cr);
    scales = t.scales + wide(page, t.sp) + wide(row, t.sr);
  }
  for (uint32_t gi = of_token >> t.lanes_log; __any_sync(~0u, gi < t.items); gi += step) {
    const uint32_t head = t.groups.div(gi), g = gi - head * t.groups.d;
    const bool in = live && gi < t.items;
    // the rows are read without waiting for the token's slot
    const T* p = x0 + wide(head, t.rh) + g * t.group;
    Pack<T, kUnit> x[NU];
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      const uint32_t e = (lane + (k << t.lanes_log)) * kUnit;
#pragma unroll
      for (int i = 0; i < kUnit; ++i) x[k].v[i] = from_f<T>(0.f);
      if (in && e < t.group) load_unit<T, VEC>(p + e, (int)(t.group - e), x[k]);
    }
    float m = max_abs(x[0]);
#pragma unroll
    for (int k = 1; k < NU; ++k) m = max_nan(m, max_abs(x[k]));
#pragma unroll
    for (uint32_t d = 16; d; d >>= 1)
      if (d < lanes) m = max_nan(m, __shfl_xor_sync(~0u, m, d));
    const bool plain = m < inf;  // all elements finite
    if (!__all_sync(~0u, plain)) {
      float f = 0.f;
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
          const float v = fabsf(to_f(x[k].v[i]));
          if (v < inf) f = fmaxf(f, v);
        }
      for (uint32_t d = lanes >> 1; d; d >>= 1) f = fmaxf(f, __shfl_xor_sync(~0u, f, d));
      m = f;
    }
    if (!has || gi >= t.items) continue;
    const bool fits = m >= 0x1p-100f;
    const float inv = fits ? __fmul_rn(__frcp_rn(m), q) : 0.f;
    if (lane == 0) scales[wide(head, t.sh) + wide(g, t.sg)] = fits ? __fmul_rn(m, 1.f / q) : 0.f;
    uint8_t* c = codes + wide(head, t.ch) + g * t.group * kCodeBits<F> / 8;
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      const uint32_t e = (lane + (k << t.lanes_log)) * kUnit;
      if (e >= t.group) continue;
      float y[kUnit];
#pragma unroll
      for (int i = 0; i < kUnit; i += 2) {
        const float2 r = mul2(make_float2(to_f(x[k].v[i]), to_f(x[k].v[i + 1])), both(inv));
        y[i] = r.x;
        y[i + 1] = r.y;
      }
      if (!plain) {
#pragma unroll
        for (int i = 0; i < kUnit; ++i) {
          const float v = to_f(x[k].v[i]);
          if (fabsf(v) == inf) y[i] = copysignf(q, v);
          else if (v != v) y[i] = F == kE4M3 ? v : 0.f;
        }
      }
      store_codes<F, VEC>(c + e * kCodeBits<F> / 8, encode<F>(y), (int)min(t.group - e, (uint32_t)kUnit));
    }
  }
}

// Eight heads' codes in flight a thread (four where the results are 32 bits wide: 64 registers, four
// CTAs of an SM), since a code's load waits for the token's slot first.
template <typename T, int F, bool VEC>
__global__ void __launch_bounds__(kThreads, 4)
gpuos_cache_read_kernel(const __grid_constant__ CacheArgs a) {
  constexpr int IT = !VEC ? 1 : sizeof(T) == 4 ? 4 : 8;  // heads a thread has in flight
  constexpr int S = VEC ? 1 : kUnit;
  const CacheTensor& t = a.t[blockIdx.z];
  const uint32_t mine = a.per_token.div(threadIdx.x);
  const uint32_t token = blockIdx.x * a.tile + mine;
  if (mine >= a.tile || token >= a.tokens) return;
  const uint32_t rest = threadIdx.x - mine * a.per_token.d;
  const uint32_t group = a.lanes.div(rest), j0 = rest - group * a.lanes.d;
  const uint32_t h0 = group + blockIdx.y * (a.per_token.d / a.lanes.d);
  const int64_t slot = load_index(a.slots, a.slot_wide, token * a.ss);
  const bool has = slot >= 0 && slot < a.rows;
  const uint32_t page = a.page.div((uint32_t)slot), row = (uint32_t)slot - page * a.page.d;
  const uint8_t* codes = static_cast<const uint8_t*>(t.codes) + wide(page, t.cp) + wide(row, t.cr);
  const float* scales = t.scales + wide(page, t.sp) + wide(row, t.sr);
  T* o0 = static_cast<T*>(t.rows) + wide(token, t.rs);

  for (uint32_t j = j0; j * kUnit < t.head; j += a.lanes.d) {
    const uint32_t e = j * kUnit;
    const int n = (int)min(t.head - e, (uint32_t)kUnit);
    uint64_t sg[S];
#pragma unroll
    for (int i = 0; i < S; ++i) sg[i] = wide(t.group_div.div(e + i), t.sg);
    for (uint32_t h = h0; h < t.heads; h += IT * a.head_step) {
      uint2 code[IT];
      float scale[IT][S];
#pragma unroll
      for (int u = 0; u < IT; ++u) {
        const uint32_t hu = h + u * a.head_step;
        if (hu >= t.heads) break;
        code[u] = make_uint2(F == kInt4 ? 0x88888888u : 0u, 0u);  // no row: zeros
#pragma unroll
        for (int i = 0; i < S; ++i) scale[u][i] = 0.f;
        if (has) {
          code[u] = load_codes<F, VEC>(codes + wide(hu, t.ch) + e * kCodeBits<F> / 8, n);
#pragma unroll
          for (int i = 0; i < S; ++i)
            if (VEC || i < n) scale[u][i] = __ldg(scales + wide(hu, t.sh) + sg[i]);
        }
      }
#pragma unroll
      for (int u = 0; u < IT; ++u) {
        const uint32_t hu = h + u * a.head_step;
        if (hu >= t.heads) break;
        T* o = o0 + wide(hu, t.rh) + e;
        float y[kUnit];
        decode<F>(code[u], y);
        if constexpr (VEC) {
          constexpr int W = 16 / sizeof(T);
#pragma unroll
          for (int k = 0; k < kUnit; k += W) {
            Pack<T, W> w;
#pragma unroll
            for (int i = 0; i < W; i += 2) {
              const float2 r = mul2(make_float2(y[k + i], y[k + i + 1]), both(scale[u][0]));
              w.v[i] = from_f<T>(r.x);
              w.v[i + 1] = from_f<T>(r.y);
            }
            store_pack<T, W>(o + k, w);
          }
        } else {
#pragma unroll
          for (int i = 0; i < kUnit; ++i)
            if (i < n) o[i] = from_f<T>(__fmul_rn(y[i], scale[u][i]));
        }
      }
    }
  }
}

int format_of(int32_t dt) {
  switch (dt) {
    case GPUOS_I8: return kInt8;
    case GPUOS_E4M3: return kE4M3;
    case GPUOS_U8: return kInt4;
    default: invalid("codes must be int8, float8_e4m3fn or uint8 (two 4-bit codes a byte)");
  }
}

// An offset is then one 32 x 32 -> 64 bit product.  (The stride of a dim of one
// element is not used.)
uint32_t stride32(const gpuos_tensor& t, int d) {
  if (t.sizes[d] <= 1) return 0;
  need(t.strides[d] < (1ll << 32), "a stride is 2^32 elements or more");
  return (uint32_t)t.strides[d];
}

// The checks both directions share.  `rows` are the tensors of rows (x or out).
CacheArgs prepare(int32_t n, const gpuos_tensor* rows, const char* name, const gpuos_tensor* slots,
                  const gpuos_tensor* codes, const gpuos_tensor* scales, bool write, bool* vec) {
  need(n == 1 || n == 2, "takes one or two tensors");
  need(rows && slots && codes && scales, "NULL tensor");
  check_tensor(slots, 1, "slots");
  need(is_index(slots->dtype), "slots must be int32 or int64");
  CacheArgs a{};
  *vec = true;
  const int64_t tokens = slots->sizes[0];
  need(tokens < (1ll << 31), "too many tokens");
  for (int i = 0; i < n; ++i) {
    const gpuos_tensor &x = rows[i], &c = codes[i], &s = scales[i];
    check_tensor(&x, 3, name);
    check_tensor(&c, 4, "codes");
    check_tensor(&s, 4, "scales");
    need(is_real(x.dtype), write ? "x must be float32, float16 or bfloat16" : "out must be float32, float16 or bfloat16");
    need(x.dtype == rows[0].dtype, "the tensors of rows must have one dtype");
    const int f = format_of(c.dtype);
    need(c.dtype == codes[0].dtype, "the caches must have one format");
    need(s.dtype == GPUOS_F32, "scales must be float32");
    const int64_t head = x.sizes[2], bits = f == kInt4 ? 4 : 8;
    need(x.sizes[0] == tokens, "slots must name one row for each token");
    need(head > 0 && head < (1 << 20) && x.sizes[1] < (1 << 20), "heads or elements out of range");
    need(head * bits % 8 == 0, "4-bit codes need an even head size");
    need(c.sizes[2] == x.sizes[1] && c.sizes[3] == head * bits / 8,
         "codes must be (page, row, head, codes of a head)");
    for (int d = 0; d < 3; ++d) need(s.sizes[d] == c.sizes[d], "scales must have the pages, rows and heads of codes");
    need(c.sizes[0] == codes[0].sizes[0] && c.sizes[1] == codes[0].sizes[1], "the caches must have the same pages");
    need(s.sizes[3] > 0 && head % s.sizes[3] == 0, "the groups of scales must divide the head");
    const int64_t group = head / s.sizes[3];
    need(group <= 1024, "a group has at most 1024 elements");
    need(group * bits % 8 == 0, "a group of 4-bit codes must fill whole bytes");
    if (numel(x)) need(x.strides[2] == 1 || head == 1, "the last dim of the rows must be contiguous");
    if (numel(c)) need(c.strides[3] == 1 || c.sizes[3] == 1, "the last dim of codes must be contiguous");
    need((__int128)tokens * x.sizes[1] * std::max(s.sizes[3], (head + kUnit - 1) / kUnit) < (1ll << 31),
         "too many elements in one call");
    const bool fits = rows_aligned(x, 16 / esize(x.dtype)) && rows_aligned(c, f == kInt4 ? 4 : 8) &&
                      group % kUnit == 0;
    if (!fits) *vec = false;
    CacheTensor& t = a.t[i];
    t.rows = x.data;
    t.codes = c.data;
    t.scales = static_cast<float*>(s.data);
    t.rs = stride32(x, 0);
    t.rh = stride32(x, 1);
    t.cp = stride32(c, 0);
    t.cr = stride32(c, 1);
    t.ch = stride32(c, 2);
    t.sp = stride32(s, 0);
    t.sr = stride32(s, 1);
    t.sh = stride32(s, 2);
    t.sg = stride32(s, 3);
    t.heads = (uint32_t)x.sizes[1];
    t.head = (uint32_t)head;
    t.group = (uint32_t)group;
    t.group_div = FastDiv(t.group);
    t.groups = FastDiv((uint32_t)s.sizes[3]);
    t.items = t.heads * t.groups.d;
    while (t.lanes_log < 5 && (uint32_t)(kGroupUnits * kUnit << t.lanes_log) < t.group) ++t.lanes_log;
  }
  const __int128 cache_rows = (__int128)codes[0].sizes[0] * codes[0].sizes[1];
  need(cache_rows < ((__int128)1 << 31), "the cache has too many rows");
  a.rows = (int64_t)cache_rows;
  a.page = FastDiv((uint32_t)std::max<int64_t>(1, codes[0].sizes[1]));
  a.slots = slots->data;
  a.ss = slots->strides[0];
  a.slot_wide = slots->dtype == GPUOS_I64;
  a.tokens = (uint32_t)tokens;
  return a;
}

template <typename T, int F>
void launch_write(const CacheArgs& a, bool vec, int n, cudaStream_t s) {
  const uint32_t per_cta = kThreads >> a.token_log;
  const dim3 grid((a.tokens + per_cta - 1) / per_cta, n);
  if (vec) run(gpuos_cache_write_kernel<T, F, true>, grid, kThreads, 0, s, a);
  else run(gpuos_cache_write_kernel<T, F, false>, grid, kThreads, 0, s, a);
}

template <typename T, int F>
void launch_read(const CacheArgs& a, bool vec, dim3 grid, cudaStream_t s) {
  if (vec) run(gpuos_cache_read_kernel<T, F, true>, grid, kThreads, 0, s, a);
  else run(gpuos_cache_read_kernel<T, F, false>, grid, kThreads, 0, s, a);
}

template <typename L>
void by_type(int32_t dt, int32_t codes, L&& launch) {
  auto with = [&](auto type) {
    using T = decltype(type);
    switch (format_of(codes)) {
      case kInt8: launch(type, std::integral_constant<int, kInt8>()); break;
      case kE4M3: launch(type, std::integral_constant<int, kE4M3>()); break;
      default: launch(type, std::integral_constant<int, kInt4>()); break;
    }
    (void)sizeof(T);
  };
  if (dt == GPUOS_F32) with(float());
  else if (dt == GPUOS_F16) with(__half());
  else with(__nv_bfloat16());
}

void cache_write(int32_t n, const gpuos_tensor* x, const gpuos_tensor* slots, const gpuos_tensor* codes,
                 const gpuos_tensor* scales, cudaStream_t stream) {
  bool vec;
  CacheArgs a = prepare(n, x, "x", slots, codes, scales, true, &vec);
  for (int i = 0; i < n; ++i) {
    check_output(codes[i], "codes");
    check_output(scales[i], "scales");
    no_overlap(codes[i], scales[i], "codes overlap scales");
    for (int k = 0; k < n; ++k) {
      no_overlap(codes[i], x[k], "codes overlap x");
      no_overlap(scales[i], x[k], "scales overlap x");
      if (k == i) continue;
      no_overlap(codes[i], codes[k], "the caches overlap");
      no_overlap(scales[i], scales[k], "the caches overlap");
      no_overlap(codes[i], scales[k], "the caches overlap");
    }
    no_overlap(codes[i], *slots, "codes overlap slots");
    no_overlap(scales[i], *slots, "scales overlap slots");
  }
  if (a.tokens == 0 || a.rows == 0 || a.t[0].items + a.t[1].items == 0) return;
  // a warp serves a token, or several whose groups do not fill it
  uint32_t wanted = 1;
  for (int i = 0; i < n; ++i) {
    const CacheTensor& t = a.t[i];
    wanted = std::max(wanted, std::max(t.items, 1u) << t.lanes_log);
    a.token_log = std::max(a.token_log, t.lanes_log);
  }
  while (a.token_log < 5 && (1u << a.token_log) < wanted) ++a.token_log;
  by_type(x[0].dtype, codes[0].dtype, [&](auto type, auto f) {
    launch_write<decltype(type), decltype(f)::value>(a, vec, n, stream);
  });
}

void cache_read(int32_t n, const gpuos_tensor* slots, const gpuos_tensor* codes, const gpuos_tensor* scales,
                const gpuos_tensor* out, cudaStream_t stream) {
  bool vec;
  CacheArgs a = prepare(n, out, "out", slots, codes, scales, false, &vec);
  uint32_t heads = 0, head = 0;
  for (int i = 0; i < n; ++i) {
    check_output(out[i], "out");
    no_overlap(out[i], *slots, "out overlaps slots");
    for (int k = 0; k < n; ++k) {
      no_overlap(out[i], codes[k], "out overlaps codes");
      no_overlap(out[i], scales[k], "out overlaps scales");
      if (k != i) no_overlap(out[i], out[k], "the outputs overlap");
    }
    heads = std::max(heads, a.t[i].heads);
    head = std::max(head, a.t[i].head);
  }
  if (a.tokens == 0 || heads == 0) return;
  const Spread sp = spread(a.tokens, (head + kUnit - 1) / kUnit, heads, kThreads, kThreads);
  a.lanes = FastDiv(sp.lanes);
  a.per_token = FastDiv(sp.lanes * sp.groups);
  a.head_step = sp.groups * sp.split;
  a.tile = sp.tile;
  const dim3 grid(sp.tiles, sp.split, n);
  by_type(out[0].dtype, codes[0].dtype, [&](auto type, auto f) {
    launch_read<decltype(type), decltype(f)::value>(a, vec, grid, stream);
  });
}

}  // namespace
}  // namespace rowops
}  // namespace gpuos

extern "C" int32_t gpuos_cache_write(int32_t n, const gpuos_tensor* x, const gpuos_tensor* slots,
                                     const gpuos_tensor* codes, const gpuos_tensor* scales, void* stream) {
  return gpuos::rowops::entry("gpuos_cache_write", [&] {
    gpuos::rowops::cache_write(n, x, slots, codes, scales, static_cast<cudaStream_t>(stream));
  });
}

extern "C" int32_t gpuos_cache_read(int32_t n, const gpuos_tensor* slots, const gpuos_tensor* codes,
                                    const gpuos_tensor* scales, const gpuos_tensor* out, void* stream) {
  return gpuos::rowops::entry("gpuos_cache_read", [&] {
    gpuos::rowops::cache_read(n, slots, codes, scales, out, static_cast<cudaStream_t>(stream));
  });
}
