// What the attention's kernels share: the parameter block, and how the work of a
// call is cut into units, items and the CTAs' shares of them.
#pragma once
#include <atomic>

#include "rowops.cuh"

namespace gpuos {
namespace rowops {
namespace attend {

constexpr uint32_t kUnit = 128;      // positions a CTA takes at once, 32 a warp
constexpr uint32_t kWarps = 4, kThreads = 32 * kWarps;
// Units up to which an item is not split.  (1 sequence of 300, 700, 1000 positions, 32 heads over 8: 14.4, 19.4, 23.0 us with 8;
// 15.1, 15.0, 15.0 with 3.  16 sequences: 18.2, 21.6, 25.8 and 18.5, 20.0, 26.4.)
constexpr uint32_t kWhole = 8;
constexpr uint32_t kMaxHead = 256;
constexpr uint32_t kWideRows = 256;  // of a block of a prompt

// A slice of the cache.
struct Held {
  const uint8_t* codes;
  const float* scales;
  int64_t cp, cr, ch;      // strides of page, row, head (bytes)
  int64_t sp, sr, sh, sg;  // of the scales (elements)
};

struct Args {
  const void* q;
  int64_t qt, qh;          // strides of token and head
  void* out;
  int64_t ot, oh;
  float* lse;              // may be NULL
  int64_t lt, lh;
  Held k, v;
  const void* pages;
  int64_t ps, pp;
  const void* lengths;
  int64_t ls;
  const void* offsets;     // may be NULL: one query a sequence
  int64_t os;
  float* partial;          // of split items: 2 slots a CTA, each rows x (head + 2)
  int4* split;             // of each CTA: the item it begins and does not end, w: CTAs that go on with it; NULL: none can be
  int64_t pool;            // pages of the cache
  int64_t capacity;        // positions a row of the table has
  uint32_t tokens, sequences;
  uint32_t k_heads, each;  // query heads of a key head
  uint32_t head, groups;   // elements; scales of a head
  uint32_t group;          // elements of a scale
  uint32_t grid;           // CTAs over which the work is spread
  uint32_t few;            // sequences of more rows than this are the kernel's for prompts, the others the one's for few rows
  uint32_t wide_grid;      // blocks of the former there may be
  int q_vec, out_vec;      // rows of q and out lie on 16 bytes
  int64_t window;          // 0: none
  float scale2;            // scale * log2(e)
  FastDiv page, each_div;
  int causal, type;        // type: of q and out
  int page_wide, length_wide, offset_wide;
  int alike;               // keys and values have the same strides
  int vec;                 // bytes of codes loaded at once: 16, 4 or 1
  int split_q, split_p;    // 16-bit parts of q and p: one, or two
};

// The queries of a sequence and what is cached of it.
struct Sequence {
  int64_t first;   // token
  int64_t n;       // queries
  int64_t length;
};

__device__ __forceinline__ Sequence sequence(const Args& a, uint32_t s) {
  Sequence q;
  if (a.offsets) {
    const int64_t lo = load_index(a.offsets, a.offset_wide, s * a.os), hi = load_index(a.offsets, a.offset_wide, (s + 1) * a.os);
    q.first = min(max(lo, (int64_t)0), (int64_t)a.tokens);
    q.n = max(min(hi, (int64_t)a.tokens) - q.first, (int64_t)0);
  } else {
    q.first = s;
    q.n = 1;
  }
  const int64_t len = load_index(a.lengths, a.length_wide, s * a.ls);
  q.length = min(max(len, (int64_t)0), a.capacity);
  return q;
}

// The positions that queries [qa, qb] of a sequence see between them.
struct Range {
  int64_t lo, hi;
};

__device__ __forceinline__ int64_t last_seen(const Args& a, const Sequence& s, int64_t query) {
  return a.causal ? s.length - s.n + query : s.length - 1;
}
__device__ __forceinline__ int64_t first_seen(const Args& a, int64_t last) {
  return a.window ? max(last - a.window + 1, (int64_t)0) : 0;
}
__device__ __forceinline__ Range seen(const Args& a, const Sequence& s, int64_t qa, int64_t qb) {
  Range r;
  r.hi = max(last_seen(a, s, qb) + 1, (int64_t)0);
  r.lo = min(first_seen(a, last_seen(a, s, qa)), r.hi);
  return r;
}

// ---- e4m3 and int8 codes as 16-bit numbers, exactly ---------------------------------
enum Format { kInt8, kE4M3 };

// The two codes in the low (high) half of x.  The NaN code of e4m3 counts as 0.
template <int F>
__device__ __forceinline__ uint32_t pair_low(uint32_t x) {
  if constexpr (F == kInt8) {  // x holds code ^ 0x80; 0x6400 + u is 1024 + u
    const uint32_t w = __byte_perm(x, 0x64646464u, 0x4140);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    uint32_t r;
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l; }" : "=r"(r) : "r"(x));
    return r & __heq2_mask(*reinterpret_cast<const __half2*>(&r), *reinterpret_cast<const __half2*>(&r));
  }
}
template <int F>
__device__ __forceinline__ uint32_t pair_high(uint32_t x) {
  if constexpr (F == kInt8) {
    const uint32_t w = __byte_perm(x, 0x64646464u, 0x4342);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&r);
  } else {
    uint32_t r;
    asm("{ .reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h; }" : "=r"(r) : "r"(x));
    return r & __heq2_mask(*reinterpret_cast<const __half2*>(&r), *reinterpret_cast<const __half2*>(&r));
  }
}
template <int F>
__device__ __forceinline__ uint32_t raw(uint32_t codes) { return F == kInt8 ? codes ^ 0x80808080u : codes; }

__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

__device__ __forceinline__ float load_real(const void* p, int type, int64_t i) {
  if (type == GPUOS_F32) return __ldg(static_cast<const float*>(p) + i);
  if (type == GPUOS_F16) return to_f(static_cast<const __half*>(p)[i]);
  return to_f(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_real(void* p, int type, int64_t i, float v) {
  if (type == GPUOS_F32) static_cast<float*>(p)[i] = v;
  else if (type == GPUOS_F16) static_cast<__half*>(p)[i] = from_f<__half>(v);
  else static_cast<__nv_bfloat16*>(p)[i] = from_f<__nv_bfloat16>(v);
}

// CTAs of an SM: three leave 168 registers a thread, enough for 8 rows.  (64 sequences of 8000 e4m3 positions, 8 rows: 200 us
// with three and two stages of codes, 217 with two and three.)
__host__ __device__ constexpr uint32_t ctas(uint32_t padded, uint32_t tiles) { return padded == 256 ? 1 : tiles == 1 ? 3 : 2; }

// A kernel's shared memory beyond 48 KB, asked for once a device.
struct SharedMemory {
  std::atomic<bool> has[64] = {};
  void grant(const void* kernel, size_t bytes) {
    int dev = -1;
    cuda_ok(cudaGetDevice(&dev), "cudaGetDevice");
    if (dev < 0 || dev >= 64) invalid("device index out of range");
    if (has[dev].load(std::memory_order_relaxed)) return;
    cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes), "shared memory");
    has[dev].store(true, std::memory_order_relaxed);
  }
};

// Launches of one format (attend_int8.cu, attend_e4m3.cu).  `rows`: of a block.
struct Plan {
  uint32_t tiles;   // of 8 rows
  bool general;     // scales of a part of the head, or numbers in two parts
  uint32_t padded;  // head, as the kernel holds it
  uint32_t per_sm;  // CTAs
};
inline Plan plan(uint32_t head, uint32_t groups, bool split, int64_t rows) {
  Plan p;
  p.padded = head <= 64 ? 64 : head <= 128 ? 128 : 256;
  p.general = groups > 1 || split;
  p.tiles = p.general ? 2 : rows <= 8 ? 1 : p.padded == 256 ? 2 : 4;
  p.per_sm = ctas(p.padded, p.general ? 2 : p.tiles);
  return p;
}
template <int F> void launch(const Plan& p, const Args& a, cudaStream_t stream);
template <int F> void launch_wide(const Args& a, cudaStream_t stream);

constexpr uint32_t kAll = ~0u;        // `few` where there is no other kernel
// Rows of a key head of a sequence above which it is a prompt.  (16 sequences, 8 key heads of 128, 1000 and 8000 positions:
// 96 rows take 93 and 344 us by few rows, 67 and 368 as prompts; 128: 95 and 439, 60 and 311; 132 as prompts 58 and 378.  1
// sequence of 8000, which fills 8 CTAs as a prompt: 132 rows 296 us, 75 by few rows; from 512 on prompts are as fast.)
constexpr uint32_t kWideFrom = 128;

}  // namespace attend
}  // namespace rowops
}  // namespace gpuos
