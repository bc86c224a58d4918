// gpuos_attend for prompts: blocks of 256 query rows on the tensor cores.
//
// A CTA takes 256 rows (queries x query heads of one key head) as two tiles of 128
// and walks over their positions 128 at a time:
//   S = Q K^T (accumulators in TMEM)  ->  P = 2^(S kappa - M)  ->  O += P (nu V) (TMEM)
// Seven warps dequantise: codes become 16-bit floats exactly, once for both tiles,
// and go into shared memory as the tensor cores read them.  Four warps for each tile
// take S from TMEM, a row a thread, and put P in its place as 16-bit floats (in two parts for
// 16-bit floats of 11 bits); a thread issues the products.  While one tile's weights
// are computed the tensor cores work on the other's.  The scales of V, relative to a power of two, go into V for
// bf16 (three roundings of 2^-12 on average each, an eighth of the result's), into P in its two parts for fp16.
// Of a step that some rows of the block do not see all of, they go into P for both, relative to a power of two that is
// the row's own: a scale that a row does not see could else leave zeros of those that it does (prompts: 2 % of the time).
// The reference M of a row follows its maximum.  A step takes the last one's, and only where the weights' sum then
// says that one may be too large, or where the row does not see all positions, the maximum is looked for (and O rescaled).
// The bound are the products: 4 * 128 operations a (row, position) of a head of 128;
// beside it, an SM has 16 exponentials a cycle, 1024 cycles a tile and step, as many as the
// two products take, and shared memory feeds Q, K and V to the tensor cores in three quarters of that time.
// Measured: 2 prompts of up to 4096 queries behind up to 8192 positions, 32 heads of 128 over 8, bf16 from int8: 1007 us,
// 0.37 of the products' rate: a step takes 6000 cycles of the dequantising warps, whose chain of loads, conversions and
// stores is what bounds it, where the products take 2048 and the weights 2500.
// The warps of codes have 88 registers; what does not fit is spilled (180 bytes a thread for heads of 128 in bf16, 530 in fp16).
#pragma once
#include "attend.h"

namespace gpuos {
namespace rowops {
namespace attend {
namespace {

constexpr uint32_t kWideTile = 128, kWideThreads = 512;  // 8 warps of weights, 7 of codes, one that issues products
constexpr uint32_t kCodeWarps = 7;
// Of scales: the weights' warps read them after the products that K fed.  (They may be a step behind the warps of codes but
// not four, so that a phase cannot pass unseen; of the two stages of K it could.)
constexpr uint32_t kRings = 4;

template <int DT>
struct Wide {
  static constexpr uint32_t blocks = DT / 64;               // of 64 elements: 128 bytes, the swizzle's width
  static constexpr uint32_t block = kWideTile * 128;        // bytes
  static constexpr uint32_t tile = blocks * block;
  static constexpr uint32_t q = 0, k = 2 * tile, v = k + 2 * tile, total = v + 2 * tile + 1024;
};

struct WideShared {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], scales_full[kRings], done, where_full;
  uint32_t tmem;
  int dead, top, uniform;  // top: the largest exponent in the block's q
  uint32_t valid[kRings][4], odd[kRings][4];  // positions with a page; whose scale of V is not finite
  float unit[kRings];    // of a step: what V is relative to; 0: each row's own
  alignas(16) float kappa[kRings][kWideTile];
  alignas(16) float nu[kRings][kWideTile];   // relative to the step's unit (1 where rows have their own)
  alignas(16) float own[kRings][kWideTile];  // as it is
  alignas(16) float high[kRings][4];         // the largest that is finite, a warp's positions each
  uint32_t joint0, joint1;                   // the steps of which all rows see all positions
  int64_t where[2][2][kWideTile];  // of a step: where each position's codes are in K and in V, -1: nowhere
  int64_t units[kWideThreads + 1];
  uint32_t seq;
  int64_t at;
};

__device__ __forceinline__ uint32_t shared_at(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void barrier_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_at(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_at(b)) : "memory");
}
__device__ __forceinline__ uint64_t now_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}
// Waits for a phase; gives up after two seconds, or when another thread has.
__device__ __forceinline__ bool await(uint64_t* b, uint32_t parity, volatile int* dead) {
  uint64_t since = 0;
  for (uint32_t i = 0;; ++i) {
    uint32_t ok;
    // (asleep for 20 us at most: polls would take their part of shared memory's rate)
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(shared_at(b)), "r"(parity), "r"(20000) : "memory");
    if (ok) return true;
    if ((i & 15) == 15) {
      if (*dead) return false;
      const uint64_t t = now_ns();
      if (!since) since = t;
      if (t - since > 2000000000ull) {
        *dead = 1;
        return false;
      }
    }
  }
}

// A tile in shared memory: rows of 128 bytes, 8 of them a swizzled atom of 1024.
// K-major (Q, K): the next 8 rows 1024 bytes on.  V lies as K does, (position, element),
// which for its product is the other order: 8 positions 1024 bytes, 64 elements `block` bytes on.
__device__ __forceinline__ uint64_t descriptor(uint32_t at, uint32_t leading, uint32_t stride) {
  return (uint64_t)((at & 0x3ffff) >> 4) | ((uint64_t)(leading >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) | (1ull << 46) |
         (2ull << 61);
}
// 16-bit operands, 32-bit accumulators, M = 128.
__host__ __device__ constexpr uint32_t instruction(uint32_t n, bool b_turned) {
  return (1u << 4) | ((uint32_t)b_turned << 16) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
// Issued by one thread of a warp whose threads all come here with the same operands: those then stay in uniform
// registers (with operands of a single thread a product took 170 cycles to issue, and 64 to run).
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t what, uint32_t add) {
  asm volatile("{ .reg .pred p, q; elect.sync _|q, 0xffffffff; setp.ne.b32 p, %4, 0; "
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(what), "r"(add) : "memory");
}
__device__ __forceinline__ void product_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t what, uint32_t add) {
  asm volatile("{ .reg .pred p, q; elect.sync _|q, 0xffffffff; setp.ne.b32 p, %4, 0; "
               "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a), "l"(b), "r"(what), "r"(add) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* b) {
  asm volatile("{ .reg .pred q; elect.sync _|q, 0xffffffff; "
               "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(shared_at(b)) : "memory");
}
__device__ __forceinline__ void after_sync() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void before_sync() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void await_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void await_stores() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

#define GPUOS_TM_R8(r, i) "=f"(r[i]), "=f"(r[i + 1]), "=f"(r[i + 2]), "=f"(r[i + 3]), "=f"(r[i + 4]), "=f"(r[i + 5]), "=f"(r[i + 6]), "=f"(r[i + 7])
#define GPUOS_TM_U8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])

// 32 neighbouring columns of this thread's row.
__device__ __forceinline__ void tmem_load(uint32_t at, float (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : GPUOS_TM_R8(r, 0), GPUOS_TM_R8(r, 8), GPUOS_TM_R8(r, 16), GPUOS_TM_R8(r, 24)
      : "r"(at));
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t at, float (&r)[N], uint32_t first) {
  float (&part)[32] = *reinterpret_cast<float (*)[32]>(&r[first]);
  tmem_load(at, part);
}
__device__ __forceinline__ void tmem_load16(uint32_t at, float (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : GPUOS_TM_R8(r, 0), GPUOS_TM_R8(r, 8)
      : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::GPUOS_TM_U8(r, 0),
      GPUOS_TM_U8(r, 8), "r"(at)
      : "memory");
}

__device__ __forceinline__ uint32_t pack16(float2 x) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(x.y), "f"(x.x));
  return r;
}

// 8 elements of a row of q (16-bit floats; at once where rows lie on 16 bytes).
__device__ __forceinline__ void load_query(const Args& a, int64_t at, float (&v)[8]) {
  if (a.q_vec) {
    const Pack<uint16_t, 8> p = load_pack<uint16_t, 8, false>(static_cast<const uint16_t*>(a.q) + at);
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
      v[i] = a.type == GPUOS_F16 ? __half2float(__ushort_as_half(p.v[i])) : __bfloat162float(__ushort_as_bfloat16(p.v[i]));
  } else {
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) v[i] = load_real(a.q, a.type, at + i);
  }
}

// The exponent of a row's largest element (-127: zeros and what is smaller; 128: an infinity).
__device__ __forceinline__ int query_exponent(const Args& a, bool has, int64_t base) {
  float most = 0.f, v[8];
  if (has)
#pragma unroll 4
    for (uint32_t e = 0; e < a.head; e += 8) {
      load_query(a, base + e, v);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
    }
  return (int)(__float_as_uint(most) >> 23) - 127;
}

// Powers of two beyond the normal numbers, as two factors.
struct Power {
  float a, b;
  __device__ explicit Power(int e) {
    const int first = min(max(e, -126), 126);
    a = __uint_as_float((uint32_t)(first + 127) << 23);
    b = __uint_as_float((uint32_t)(min(max(e - first, -126), 126) + 127) << 23);
  }
};

// What scales of V are relative to: powers of two.
constexpr float kLeastUnit = 0x1p-90f;
__device__ __forceinline__ float unit_above(float most) {
  return fmaxf(__uint_as_float(min((__float_as_uint(most) & 0x7f800000u) + 0x00800000u, 0x7e800000u)), kLeastUnit);
}
__device__ __forceinline__ float inverse(float unit) { return __uint_as_float(0x7f000000u - __float_as_uint(unit)); }

// Row r of q times 2^shift, as 16-bit floats in a tile.
template <int DT>
__device__ __forceinline__ void stage_query(const Args& a, uint8_t* tile, uint32_t r, bool has, int64_t base, int shift) {
  const Power up(shift);
  const float by = a.scale2 < 0.f ? -up.b : up.b;
  float v[8];
#pragma unroll 4
  for (uint32_t x = 0; x < DT / 8; ++x) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (has && x * 8 < a.head) {
      load_query(a, base + x * 8, v);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) w[i] = pack16(make_float2(v[2 * i] * up.a * by, v[2 * i + 1] * up.a * by));
    }
    *reinterpret_cast<uint4*>(tile + (x >> 3) * Wide<DT>::block + r * 128 + (((x & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

__device__ __forceinline__ int64_t wide_blocks(const Args& a, const Sequence& s) {
  const int64_t rows = s.n * a.each;
  return rows > a.few ? (rows + kWideRows - 1) / kWideRows : 0;
}

template <int F, int DT, bool SPLIT>
__global__ void __launch_bounds__(kWideThreads, 1)
gpuos_attend_wide_kernel(const __grid_constant__ Args a) {
  using W = Wide<DT>;
  extern __shared__ uint8_t raw_smem[];
  __shared__ WideShared sh;
  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  uint8_t* const smem = raw_smem + (1024 - (shared_at(raw_smem) & 1023)) % 1024;

  // ---- the item: blocks of a sequence from the last (the longest) on, their heads side by side
  {
    const uint32_t per = (a.sequences + kWideThreads - 1) / kWideThreads;
    const uint32_t s0 = min(tid * per, a.sequences), s1 = min(s0 + per, a.sequences);
    int64_t n = 0;
    for (uint32_t s = s0; s < s1; ++s) n += wide_blocks(a, sequence(a, s)) * a.k_heads;
    sh.units[tid + 1] = n;
    if (tid == 0) sh.units[0] = 0, sh.seq = a.sequences, sh.dead = 0, sh.top = -127, sh.uniform = 1;
    __syncthreads();
    if (warp == 0) {
      int64_t run = 0;
      for (uint32_t i = 0; i < kWideThreads; i += 32) {
        int64_t v = sh.units[i + lane + 1];
        for (uint32_t d = 1; d < 32; d <<= 1) {
          const int64_t o = __shfl_up_sync(~0u, v, d);
          if (lane >= d) v += o;
        }
        sh.units[i + lane + 1] = run + v;
        run += __shfl_sync(~0u, v, 31);
      }
    }
    __syncthreads();
    const int64_t u = blockIdx.x;
    if (sh.units[tid] <= u && u < sh.units[tid + 1]) {
      int64_t at = sh.units[tid];
      for (uint32_t s = s0; s < s1; ++s) {
        const int64_t m = wide_blocks(a, sequence(a, s)) * a.k_heads;
        if (u < at + m) {
          sh.seq = s;
          sh.at = u - at;
          break;
        }
        at += m;
      }
    }
    __syncthreads();
  }
  if (sh.seq >= a.sequences) return;
  const Sequence s = sequence(a, sh.seq);
  const int64_t order = sh.at / a.k_heads;
  const uint32_t head = (uint32_t)(sh.at - order * a.k_heads);
  const int64_t row_base = (wide_blocks(a, s) - 1 - order) * kWideRows, row_all = s.n * a.each;
  const uint32_t query_a = a.each_div.div((uint32_t)row_base), query_b = a.each_div.div((uint32_t)(min(row_base + kWideRows, row_all) - 1));
  const Range range = seen(a, s, query_a, query_b);
  const uint32_t steps = (uint32_t)((range.hi - range.lo + kWideTile - 1) / kWideTile);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      barrier_init(&sh.k_full[i], 32 * kCodeWarps);
      barrier_init(&sh.v_full[i], 32 * kCodeWarps);
      barrier_init(&sh.k_empty[i], 1);
      barrier_init(&sh.v_empty[i], 1);
      barrier_init(&sh.s_full[i], 1);
      barrier_init(&sh.p_full[i], 128);
      
    }
    const int64_t lo = first_seen(a, last_seen(a, s, query_b)) - range.lo, hi = last_seen(a, s, query_a) + 1 - range.lo;
    sh.joint0 = (uint32_t)min((lo + kWideTile - 1) / kWideTile, (int64_t)steps);
    sh.joint1 = (uint32_t)(max(hi, (int64_t)0) / kWideTile);
    for (uint32_t i = 0; i < kRings; ++i) barrier_init(&sh.scales_full[i], 128);
    barrier_init(&sh.done, 1);
    barrier_init(&sh.where_full, 32 * kCodeWarps);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 15) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_at(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // The weights' warps bring the block's rows of q, times one power of two where the rows' largest elements are within
  // 2^10 of one another (16-bit floats then reach 2^-19 of each, 2^-29 of the largest score), else each its own.
  float scale = 1.f;
  int64_t lo = 1, hi = 0, token = 0;
  uint32_t q_head = 0;
  const uint32_t t = warp >> 2;  // the tile of a weights' warp
  const int64_t row = row_base + tid;
  const bool has_row = warp < 8 && row < row_all;
  int exponent = -127;
  if (has_row) {
    const uint32_t query = a.each_div.div((uint32_t)row);
    token = s.first + query;
    q_head = head * a.each + (uint32_t)row - query * a.each;
    const int64_t last = last_seen(a, s, query);
    lo = first_seen(a, last);
    hi = last + 1;
    exponent = query_exponent(a, true, token * a.qt + q_head * a.qh);
    atomicMax(&sh.top, exponent);
  }
  __syncthreads();
  if (has_row && exponent > -127 && exponent < sh.top - 10) sh.uniform = 0;
  __syncthreads();
  const bool uniform = sh.uniform;
  if (warp < 8) {
    const int shift = uniform ? (sh.top > -127 ? 14 - sh.top : 0) : exponent > -127 ? 14 - exponent : 0;
    stage_query<DT>(a, smem + W::q + t * W::tile, tid & 127, has_row, token * a.qt + q_head * a.qh, shift);
    if (!uniform) {
      const Power down(-shift);
      scale = fmaxf(fabsf(a.scale2) * down.a * down.b, 1e-38f);  // (a score of -inf stays one)
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = sh.tmem, t_s = tmem + t * 128, t_o = tmem + 256 + t * DT;

  // (256 * 168 + 256 * 88 registers: the 512 * 128 of the launch)
  if (warp >= 8) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
   if (warp < 8 + kCodeWarps) {
    // ---- codes: a thread finds a position; then 8 (heads up to 64: 4) threads load one, 16 bytes each
    const uint32_t j = tid - 256;
    constexpr uint32_t X = DT / 16;                                        // 16-byte pieces of a position
    constexpr uint32_t PASS = 32 * kCodeWarps / X, N = (kWideTile + PASS - 1) / PASS;  // positions at once, and how often
    static_assert(PASS % 4 == 0);
    const uint32_t piece = j % X, own = j / X;
    const bool in = piece * 16 < a.head;
    const int64_t table = sh.seq * a.ps;
    const uint8_t* const k_codes = a.k.codes + head * a.k.ch + piece * 16;
    const uint8_t* const v_codes = a.v.codes + head * a.v.ch + piece * 16;
    const Power down(uniform && sh.top > -127 ? sh.top - 14 : 0);
    const float by = uniform ? fabsf(a.scale2) * down.a : 1.f;
    // A position's page is read two steps ahead, its scales one (nothing waits for them).
    auto page_at = [&](uint32_t step) -> int64_t {  // as the table has it; -1 behind the range
      const int64_t p = range.lo + (int64_t)step * kWideTile + j;
      if (warp >= 12 || p >= range.hi) return -1;
      return load_index(a.pages, a.page_wide, table + a.page.div((uint32_t)p) * a.pp);
    };
    float kappa1 = 0.f, nu1 = 0.f;
    int64_t k_at = -1, v_at = -1, page2 = -1;
    auto ahead = [&](uint32_t step, int64_t page) {  // places of a step's codes, and its scales
      k_at = v_at = -1;
      kappa1 = nu1 = 0.f;
      if (warp >= 12 || page < 0 || page >= a.pool) return;
      const uint32_t p = (uint32_t)(range.lo + (int64_t)step * kWideTile + j), at = p - a.page.div(p) * a.page.d;
      k_at = page * a.k.cp + at * a.k.cr;
      v_at = page * a.v.cp + at * a.v.cr;
      kappa1 = __ldg(a.k.scales + page * a.k.sp + at * a.k.sr + head * a.k.sh);
      nu1 = __ldg(a.v.scales + page * a.v.sp + at * a.v.sr + head * a.v.sh);
    };
    // (a step's scales go where those of four steps before were, which have been read: `find` comes after the scores of two
    // steps before it were issued, and those wait for the weights of three)
    auto find = [&](uint32_t step) {
      if (warp < 12) {
        const uint32_t ring = step % kRings;
        sh.where[step & 1][0][j] = k_at;
        sh.where[step & 1][1][j] = v_at;
        sh.kappa[ring][j] = kappa1 * by * down.b;
        const uint32_t valid = __ballot_sync(~0u, k_at >= 0);
        // a scale that is not finite makes NaN of the rows that see it, and must not touch others: it is not multiplied
        const bool fine = fabsf(nu1) < INFINITY;
        const uint32_t odd = __ballot_sync(~0u, !fine);
        const float nu = fine ? nu1 : 0.f, high = warp_max(fabsf(nu));
        sh.own[ring][j] = nu;
        if (lane == 0) sh.valid[ring][warp - 8] = valid, sh.odd[ring][warp - 8] = odd, sh.high[ring][warp - 8] = high;
      }
      arrive(&sh.where_full);  // (who finds nothing has read what was there)
    };
    // Of a step that all rows see, V is brought in relative to a power of two that is raised when a scale passes it by 2^2.
    // Of the others the scales go into the weights, so that none changes a row that does not see it.
    float unit = kLeastUnit;
    auto joint = [&](uint32_t step) { return step >= sh.joint0 && step < sh.joint1; };
    auto raise = [&](uint32_t step) {
      const float4 w = *reinterpret_cast<const float4*>(sh.high[step % kRings]);
      const float most = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w));
      if (most > 4.f * unit && joint(step)) unit = unit_above(most);
    };
    auto load = [&](const uint8_t* codes, uint32_t step, uint32_t which, uint4 (&r)[N]) {
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        const uint32_t p = i * PASS + own;
        const int64_t at = N * PASS == kWideTile || p < kWideTile ? sh.where[step & 1][which][p] : -1;
        r[i] = at >= 0 && in ? __ldg(reinterpret_cast<const uint4*>(codes + at)) : make_uint4(0, 0, 0, 0);
      }
    };
    // (the two halves of 8 threads in turn: no two of them in a bank)
    const uint32_t flip = piece >> 2;
    const uint32_t put0 = (piece >> 2) * W::block + own * 128 + (((2 * (piece & 3) + flip) ^ (own & 7)) << 4);
    const uint32_t put1 = (piece >> 2) * W::block + own * 128 + (((2 * (piece & 3) + 1 - flip) ^ (own & 7)) << 4);
    auto put = [&](uint8_t* tile, const uint4 (&r)[N], [[maybe_unused]] const float* by_scale) {
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        if (N * PASS != kWideTile && i * PASS + own >= kWideTile) break;
        const uint32_t turn = (i * PASS & 4) << 4;  // of the swizzle, from a thread's first position to this one
        const uint32_t w0 = raw<F>(flip ? r[i].z : r[i].x), w1 = raw<F>(flip ? r[i].w : r[i].y);
        const uint32_t w2 = raw<F>(flip ? r[i].x : r[i].z), w3 = raw<F>(flip ? r[i].y : r[i].w);
        uint4 x = make_uint4(pair_low<F>(w0), pair_high<F>(w0), pair_low<F>(w1), pair_high<F>(w1));
        uint4 y = make_uint4(pair_low<F>(w2), pair_high<F>(w2), pair_low<F>(w3), pair_high<F>(w3));
        if (!SPLIT && by_scale) {
          const __half2 h = __float2half2_rn(by_scale[i * PASS + own]);
          __half2* const xs[2] = {reinterpret_cast<__half2*>(&x), reinterpret_cast<__half2*>(&y)};
#pragma unroll
          for (uint32_t k = 0; k < 8; ++k) xs[k >> 2][k & 3] = __hmul2(xs[k >> 2][k & 3], h);
        }
        *reinterpret_cast<uint4*>(tile + (put0 ^ turn) + i * PASS * 128) = x;
        *reinterpret_cast<uint4*>(tile + (put1 ^ turn) + i * PASS * 128) = y;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    uint4 rk[N], rv[N];
    bool ok = true;
    if (steps) {
      ahead(0, page_at(0));
      find(0);
      ahead(1, page_at(1));
      page2 = page_at(2);
      ok = await(&sh.where_full, 0, &sh.dead);
      if (ok) {
        raise(0);
        load(k_codes, 0, 0, rk);
      }
    }
    for (uint32_t i = 0; ok && i < steps; ++i) {
      const uint32_t st = i & 1, ring = i % kRings;
      load(v_codes, i, 1, rv);
      if (i >= 2 && !await(&sh.k_empty[st], (i / 2 - 1) & 1, &sh.dead)) break;
      put(smem + W::k + st * W::tile, rk, nullptr);
      if (warp < 12) {
        const bool all = joint(i);
        sh.nu[ring][j] = all ? sh.own[ring][j] * inverse(unit) : 1.f;
        if (tid == 256) sh.unit[ring] = all ? unit : 0.f;
        arrive(&sh.scales_full[ring]);
      }
      arrive(&sh.k_full[st]);
      if (i + 1 < steps) {
        __syncwarp();
        find(i + 1);
        ahead(i + 2, page2);
        page2 = page_at(i + 3);
        if (!await(&sh.where_full, (i + 1) & 1, &sh.dead)) break;  // (and this step's scales are there)
        raise(i + 1);
        load(k_codes, i + 1, 0, rk);
      } else if (!await(&sh.k_full[st], (i / 2) & 1, &sh.dead)) {
        break;
      }
      if (i >= 2 && !await(&sh.v_empty[st], (i / 2 - 1) & 1, &sh.dead)) break;
      put(smem + W::v + st * W::tile, rv, sh.nu[ring]);
      arrive(&sh.v_full[st]);
    }
   } else {
    // ---- products: a warp of its own issues them, since it waits while the tensor cores are busy
    if (steps) {
      constexpr uint32_t to_s = instruction(kWideTile, false), to_o = instruction(DT, true);
      const uint32_t at = shared_at(smem);
      const uint64_t q0 = descriptor(at + W::q, 16, 1024), k0 = descriptor(at + W::k, 16, 1024), v0 = descriptor(at + W::v, W::block, 1024);
      auto scores = [&](uint32_t tile, uint32_t st) {
        const uint64_t q = q0 + tile * (W::tile >> 4), k = k0 + st * (W::tile >> 4);
#pragma unroll
        for (uint32_t e = 0; e < DT / 16; ++e) {
          const uint32_t b = ((e >> 2) * W::block + (e & 3) * 32) >> 4;
          product(tmem + tile * 128, q + b, k + b, to_s, e > 0);
        }
        commit(&sh.s_full[tile]);
      };
      auto values = [&](uint32_t tile, uint32_t st, bool add) {
        const uint64_t v = v0 + st * (W::tile >> 4);
        const uint32_t p = tmem + tile * 128, o = tmem + 256 + tile * DT;
#pragma unroll
        for (uint32_t e = 0; e < kWideTile / 16; ++e) product_from_tmem(o, p + e * 8, v + e * 128, to_o, e > 0 || add);
        if constexpr (SPLIT) {
#pragma unroll
          for (uint32_t e = 0; e < kWideTile / 16; ++e) product_from_tmem(o, p + 64 + e * 8, v + e * 128, to_o, 1);
        }
      };
      bool ok = __all_sync(~0u, await(&sh.k_full[0], 0, &sh.dead));
      if (ok) {
        after_sync();
        scores(0, 0);
        scores(1, 0);
        commit(&sh.k_empty[0]);
      }
      for (uint32_t i = 0; ok && i < steps; ++i) {
        const uint32_t st = i & 1, next = st ^ 1;
        ok = __all_sync(~0u, await(&sh.v_full[st], (i / 2) & 1, &sh.dead));
#pragma unroll
        for (uint32_t tile = 0; tile < 2; ++tile) {
          ok = ok && __all_sync(~0u, await(&sh.p_full[tile], i & 1, &sh.dead));
          if (!ok) break;
          after_sync();
          values(tile, st, i > 0);
          if (tile == 1) commit(&sh.v_empty[st]);
          if (i + 1 == steps) continue;
          if (tile == 0) ok = __all_sync(~0u, await(&sh.k_full[next], ((i + 1) / 2) & 1, &sh.dead));
          if (!ok) break;
          after_sync();
          scores(tile, next);
          if (tile == 1) commit(&sh.k_empty[next]);
        }
      }
      commit(&sh.done);
      // (what was issued has to end before TMEM is given back, on a way out too)
      int alone = 0;
      await(&sh.done, 0, &alone);
    }
    __syncwarp();
   }
  } else {
    // ---- weights: a row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    const uint32_t lanes = (warp & 3) << 21;  // (32 lanes a warp, in the upper half of an address)
    float m = -INFINITY, ref = 0.f, unit = kLeastUnit, sum = 0.f;  // the row's maximum; what weights and O are relative to
    bool ok = true;
    // (room above for later maxima; for the lower parts, room below)
    constexpr int kUp = SPLIT ? 4 : 0, kSlack = SPLIT ? 2 : 8, kRoom = 5;
    // two weights times their scales, as 16-bit floats, and what those leave
    auto pair = [&](float2 y, uint32_t& w, uint32_t& low) {
      w = pack16(y);
      if constexpr (SPLIT) {
        const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&w));
        low = pack16(make_float2(y.x - h.x, y.y - h.y));
      }
    };
    // A step that the rows see all of: its weights in the units of the last one; whether they may be kept.
    auto quick = [&](uint32_t i, bool sure) {
      const uint32_t ring = i % kRings;
      const float* const kappa = sh.kappa[ring];
      const float* const nu = sh.nu[ring];
      // 16 scores at a time while the next ones are on their way (32 at a time left no registers for their scales ahead)
      float r[2][16];
      uint32_t w[64];
      [[maybe_unused]] uint32_t low[SPLIT ? 64 : 1];
      if (__any_sync(~0u, sh.unit[ring] != unit) && !sure) return false;
      tmem_load16(t_s + lanes, r[0]);
      float2 add[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (uint32_t c = 0; c < 8; ++c) {
        float4 k4[4];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) k4[e] = *reinterpret_cast<const float4*>(kappa + c * 16 + e * 4);
        await_loads();
        if (c < 7) tmem_load16(t_s + lanes + (c + 1) * 16, r[(c + 1) & 1]);
        const float (&x)[16] = r[c & 1];
        float2 y[8];
#pragma unroll
        for (uint32_t e = 0; e < 4; ++e) {
          y[2 * e] = fma2(make_float2(x[4 * e], x[4 * e + 1]), make_float2(k4[e].x, k4[e].y), both(-ref));
          y[2 * e + 1] = fma2(make_float2(x[4 * e + 2], x[4 * e + 3]), make_float2(k4[e].z, k4[e].w), both(-ref));
        }
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) y[e] = make_float2(ex2(y[e].x), ex2(y[e].y));
#pragma unroll
        for (uint32_t e = 0; e < 8; ++e) {
          add[e & 1] = add2(add[e & 1], y[e]);
          if constexpr (SPLIT) y[e] = mul2(y[e], *reinterpret_cast<const float2*>(nu + c * 16 + e * 2));
          pair(y[e], w[c * 8 + e], low[SPLIT ? c * 8 + e : 0]);
        }
      }
      add[0] = add2(add[0], add[1]);
      const float more = add[0].x + add[0].y;
      // no weight is larger than their sum (their scales, relative to the unit, are 4 at most)
      if (__any_sync(~0u, !(more <= (SPLIT ? 8192.f : 32768.f))) && !sure) return false;
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) {
        tmem_store16(t_s + lanes + c * 16, *reinterpret_cast<const uint32_t (*)[16]>(&w[c * 16]));
        if constexpr (SPLIT) tmem_store16(t_s + 64 + lanes + c * 16, *reinterpret_cast<const uint32_t (*)[16]>(&low[c * 16]));
      }
      sum += more;
      return true;
    };
    // O and the sum of weights in units of a higher maximum, or of another unit of V.
    auto rescale = [&](uint32_t i, float high, float unit_now) {
      const float before = ref;
      const bool none = m == -INFINITY;
      m = fmaxf(m, high);
      ref = (m > -INFINITY ? m : 0.f) - (float)kUp;
      float f = none ? 0.f : ex2(before - ref);
      sum *= f;
      f *= unit / unit_now;  // (at most 2^60)
      unit = unit_now;
      if (i == 0) return;
      float r[32];
#pragma unroll 1
      for (uint32_t c = 0; c < DT / 32; ++c) {
        tmem_load(t_o + lanes + c * 32, r);
        await_loads();
#pragma unroll
        for (uint32_t e = 0; e < 32; e += 2) *reinterpret_cast<float2*>(&r[e]) = mul2(*reinterpret_cast<float2*>(&r[e]), both(f));
        tmem_store16(t_o + lanes + c * 32, *reinterpret_cast<const uint32_t (*)[16]>(&r[0]));
        tmem_store16(t_o + lanes + c * 32 + 16, *reinterpret_cast<const uint32_t (*)[16]>(&r[16]));
      }
    };
    // The unit for a step that all rows see.  (One that is 2^60 below the row's takes nothing that O would keep.)
    auto joint_unit = [&](uint32_t i) {
      const float u = sh.unit[i % kRings];
      return unit > u * 0x1p60f ? unit : u;
    };
    auto raise = [&](uint32_t i) {
      const float* const kappa = sh.kappa[i % kRings];
      float r[32], high = -INFINITY;
#pragma unroll 1
      for (uint32_t c = 0; c < 4; ++c) {
        tmem_load(t_s + lanes + c * 32, r);
        await_loads();
#pragma unroll
        for (uint32_t e = 0; e < 32; e += 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(kappa + c * 32 + e);
          const float2 u = mul2(make_float2(r[e], r[e + 1]), make_float2(k4.x, k4.y)), v = mul2(make_float2(r[e + 2], r[e + 3]), make_float2(k4.z, k4.w));
          high = fmaxf(fmaxf(high, u.x), u.y);
          high = fmaxf(fmaxf(high, v.x), v.y);
        }
      }
      rescale(i, high, joint_unit(i));
    };
    // A step of which positions [from, to) are seen.  Seldom run, so small.
    auto careful = [&](uint32_t i, int from, int to) {
      const uint32_t ring = i % kRings;
      const float* const kappa = sh.kappa[ring];
      const bool joint = sh.unit[ring] > 0.f;
      const float* const nu = joint ? sh.nu[ring] : sh.own[ring];
      auto seen_of = [&](uint32_t c) {
        const int l = min(max(from - (int)c * 32, 0), 32), h = min(max(to - (int)c * 32, 0), 32);
        return (h >= 32 ? ~0u : (1u << h) - 1) & ~(l >= 32 ? ~0u : (1u << l) - 1) & sh.valid[ring][c];
      };
      float r[32], high = -INFINITY;
#pragma unroll 1
      for (uint32_t c = 0; c < 4; ++c) {
        tmem_load(t_s + lanes + c * 32, r);
        const uint32_t bits = seen_of(c);
        await_loads();
#pragma unroll
        for (uint32_t e = 0; e < 32; ++e) high = fmaxf(high, bits >> e & 1 ? r[e] * kappa[c * 32 + e] : -INFINITY);
      }
      if (high > -INFINITY) high *= scale;
      // a row's own unit: 2^kRoom below the largest scale it has seen (of those behind it, up to 2^(kRoom + 1) above it)
      float unit_now = unit;
      if (joint) {
        unit_now = joint_unit(i);
      } else {
        const float4 w = *reinterpret_cast<const float4*>(sh.high[ring]);
        if (fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w)) > (float)(2 << kRoom) * unit) {
          float most = 0.f;
#pragma unroll 1
          for (uint32_t c = 0; c < 4; ++c)
            for (uint32_t bits = seen_of(c); bits; bits &= bits - 1) most = fmaxf(most, fabsf(nu[c * 32 + __ffs(bits) - 1]));
          if (most > (float)(2 << kRoom) * unit) unit_now = unit_above(most) * (1.f / (1 << kRoom));
        }
      }
      // weights are at most 2^kUp at the maximum and 2^kSlack more from scores above it
      if (__any_sync(~0u, high > m + (float)kSlack || unit_now != unit)) rescale(i, high, unit_now);
      const float by = joint ? sh.unit[ring] * inverse(unit) : inverse(unit);
      // (the lower parts take the place of the last scores, once those have been read)
      [[maybe_unused]] uint32_t low[SPLIT ? 64 : 1];
#pragma unroll(SPLIT ? 4 : 1)
      for (uint32_t c = 0; c < 4; ++c) {
        uint32_t w[16];
        tmem_load(t_s + lanes + c * 32, r);
        const uint32_t bits = seen_of(c);
        if (bits & sh.odd[ring][c]) sum = NAN;
        await_loads();
#pragma unroll
        for (uint32_t e = 0; e < 32; e += 2) {
          float u = ex2(fmaf(r[e] * kappa[c * 32 + e], scale, -ref)), v = ex2(fmaf(r[e + 1] * kappa[c * 32 + e + 1], scale, -ref));
          u = bits >> e & 1 ? u : 0.f;
          v = bits >> e & 2 ? v : 0.f;
          sum += u + v;
          // (where it is not seen a scale may be anything)
          u = u == 0.f ? 0.f : u * ((SPLIT || !joint ? nu[c * 32 + e] : 1.f) * by);
          v = v == 0.f ? 0.f : v * ((SPLIT || !joint ? nu[c * 32 + e + 1] : 1.f) * by);
          pair(make_float2(u, v), w[e / 2], low[SPLIT ? c * 16 + e / 2 : 0]);
        }
        // (in the place of scores that have been read)
        tmem_store16(t_s + lanes + c * 16, w);
      }
      if constexpr (SPLIT) {
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) tmem_store16(t_s + 64 + lanes + c * 16, *reinterpret_cast<const uint32_t (*)[16]>(&low[c * 16]));
      }
    };
    for (uint32_t i = 0; i < steps; ++i) {
      ok = await(&sh.scales_full[i % kRings], (i / kRings) & 1, &sh.dead) && await(&sh.s_full[t], i & 1, &sh.dead);
      if (!__all_sync(~0u, ok)) break;
      after_sync();
      const int64_t p0 = range.lo + (int64_t)i * kWideTile;
      const uint32_t* const v = sh.valid[i % kRings];
      const uint32_t* const x = sh.odd[i % kRings];
      const bool plain = (v[0] & v[1] & v[2] & v[3]) == ~0u && !(x[0] | x[1] | x[2] | x[3]) && lo <= p0 && hi >= p0 + kWideTile;
      const int from = (int)max(min(lo - p0, (int64_t)kWideTile), (int64_t)0), to = (int)max(min(hi - p0, (int64_t)kWideTile), (int64_t)0);
      if (!(uniform && sh.unit[i % kRings] > 0.f && __all_sync(~0u, plain))) {
        careful(i, from, to);
      } else if (__any_sync(~0u, m == -INFINITY) || !quick(i, false)) {
        // (a row that has seen nothing yet, at the start or behind steps before its window or without pages, has no reference)
        raise(i);
        if (__all_sync(~0u, sh.unit[i % kRings] == unit)) quick(i, true);
        else careful(i, from, to);
      }
      await_stores();
      before_sync();
      arrive(&sh.p_full[t]);
    }
    if (steps) ok = await(&sh.done, 0, &sh.dead) && ok;
    // ---- the block's rows of the result
    if (!__all_sync(~0u, ok)) sum = NAN;  // given up: shows in the results
    after_sync();
    const float inv = sum == 0.f ? 0.f : unit / sum;
#pragma unroll
    for (uint32_t c = 0; c < DT / 32; ++c) {
      float r[32];
      __syncwarp();
      if (steps) {
        tmem_load(t_o + lanes + c * 32, r);
        await_loads();
      }
      if (row >= row_all) continue;
      const int64_t at = token * a.ot + q_head * a.oh + c * 32;
#pragma unroll
      for (uint32_t e = 0; e < 32; e += 8) {
        if (c * 32 + e >= a.head) break;
        float y[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) y[k] = steps && sum != 0.f ? r[e + k] * inv : 0.f;
        if (a.out_vec) {
          Pack<uint16_t, 8> p;
#pragma unroll
          for (uint32_t k = 0; k < 8; ++k) {
            if (a.type == GPUOS_F16) p.v[k] = __half_as_ushort(from_f<__half>(y[k]));
            else p.v[k] = __bfloat16_as_ushort(from_f<__nv_bfloat16>(y[k]));
          }
          store_pack(static_cast<uint16_t*>(a.out) + at + e, p);
        } else {
#pragma unroll
          for (uint32_t k = 0; k < 8; ++k) store_real(a.out, a.type, at + e + k, y[k]);
        }
      }
    }
    if (a.lse && row < row_all) a.lse[token * a.lt + q_head * a.lh] = sum == 0.f ? -INFINITY : (ref + log2f(sum)) * 0.69314718056f;
    before_sync();
  }
  __syncthreads();
  if (warp == 15) {
    after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int F, int DT, bool SPLIT>
void start_wide(const Args& a, cudaStream_t stream) {
  void (*const kernel)(const Args) = gpuos_attend_wide_kernel<F, DT, SPLIT>;
  static SharedMemory room;
  room.grant(reinterpret_cast<const void*>(kernel), Wide<DT>::total);
  run(kernel, dim3(a.wide_grid), kWideThreads, Wide<DT>::total, stream, a);
}

}  // namespace

template <int F>
void launch_wide(const Args& a, cudaStream_t stream) {
  if (a.head <= 64) a.split_p ? start_wide<F, 64, true>(a, stream) : start_wide<F, 64, false>(a, stream);
  else a.split_p ? start_wide<F, 128, true>(a, stream) : start_wide<F, 128, false>(a, stream);
}

}  // namespace attend
}  // namespace rowops
}  // namespace gpuos
