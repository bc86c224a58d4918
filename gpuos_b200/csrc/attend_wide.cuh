// gpuos_attend for prompts: blocks of 256 query rows on the tensor cores.
//
// A CTA takes 256 rows (queries x query heads of one key head) as two tiles of 128
// and walks over their positions 128 at a time:
//   S = Q K^T (accumulators in TMEM)  ->  P = 2^(S kappa - M) nu  ->  O += P V (TMEM)
// Four warps dequantise: codes become 16-bit floats exactly, once for both tiles,
// and go into shared memory as the tensor cores read them.  Four warps for each tile
// take S from TMEM, a row a thread, put P in its place as 16-bit floats (in two parts for
// 16-bit floats of 11 bits), and one of their threads issues the tile's products.  While one tile's weights
// are computed the tensor cores work on the other's.  The reference M of a row follows its maximum and the
// largest scale of V seen (as a power of two), and both O and the sum of weights are in its units; it is
// raised, and O rescaled, only when a weight could pass 2^14.
// The bound are the products: 4 * 128 operations a (row, position) of a head of 128;
// beside it, an SM has 16 exponentials a cycle, 1024 cycles a tile and step, as many as the
// two products take, and shared memory feeds Q, K and V to the tensor cores in three quarters of that time.
#pragma once
#include "attend.h"

namespace gpuos {
namespace rowops {
namespace attend {
namespace {

constexpr uint32_t kWideTile = 128, kWideThreads = 384;  // 8 warps of weights, 4 of codes
constexpr uint32_t kRings = 4;  // of scales: the weights' warps read them after the products that K fed

template <int DT>
struct Wide {
  static constexpr uint32_t blocks = DT / 64;               // of 64 elements: 128 bytes, the swizzle's width
  static constexpr uint32_t block = kWideTile * 128;        // bytes
  static constexpr uint32_t tile = blocks * block;
  static constexpr uint32_t q = 0, k = 2 * tile, v = k + 2 * tile, total = v + 2 * tile + 1024;
};

struct WideShared {
  uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], done[2], where_full;
  uint32_t tmem;
  int dead;
  uint32_t valid[kRings][4];
  alignas(16) float kappa[kRings][kWideTile];
  alignas(16) float nu[kRings][kWideTile];
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
    asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
                 : "=r"(ok) : "r"(shared_at(b)), "r"(parity) : "memory");
    if (ok) return true;
    if ((i & 63) == 63) {
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
__device__ __forceinline__ void product(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
               "l"(b), "r"(what), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void product_from_tmem(uint32_t d, uint32_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a),
               "l"(b), "r"(what), "r"((uint32_t)add) : "memory");
}
__device__ __forceinline__ void commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(shared_at(b)) : "memory");
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

// Row r of q times a power of two (the result undoes it), as 16-bit floats in a tile.
template <int DT>
__device__ __forceinline__ float stage_query(const Args& a, uint8_t* tile, uint32_t r, bool has, int64_t base) {
  float most = 0.f, v[8];
  if (has)
#pragma unroll 4
    for (uint32_t e = 0; e < a.head; e += 8) {
      load_query(a, base + e, v);
#pragma unroll
      for (uint32_t i = 0; i < 8; ++i) most = fmaxf(most, fabsf(v[i]));
    }
  int shift = 14 - (int)((__float_as_uint(most) >> 23) - 127);
  if (!(most > 0.f)) shift = 0;
  const int first = min(max(shift, -126), 126);
  const float up = __uint_as_float((uint32_t)(first + 127) << 23), more = __uint_as_float((uint32_t)(shift - first + 127) << 23);
  const float by = a.scale2 < 0.f ? -more : more;
#pragma unroll 4
  for (uint32_t x = 0; x < DT / 8; ++x) {
    uint32_t w[4] = {0, 0, 0, 0};
    if (has && x * 8 < a.head) {
      load_query(a, base + x * 8, v);
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) w[i] = pack16(make_float2(v[2 * i] * up * by, v[2 * i + 1] * up * by));
    }
    *reinterpret_cast<uint4*>(tile + (x >> 3) * Wide<DT>::block + r * 128 + (((x & 7) ^ (r & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  // (a scale of 0 as one that makes no difference: a masked score of -inf stays one)
  return fmaxf(fabsf(a.scale2) / up / more, 1e-38f);
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
    if (tid == 0) sh.units[0] = 0, sh.seq = a.sequences, sh.dead = 0;
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
  const Range range = seen(a, s, a.each_div.div((uint32_t)row_base), a.each_div.div((uint32_t)(min(row_base + kWideRows, row_all) - 1)));
  const uint32_t steps = (uint32_t)((range.hi - range.lo + kWideTile - 1) / kWideTile);

  if (tid == 0) {
    for (int i = 0; i < 2; ++i) {
      barrier_init(&sh.k_full[i], 128);
      barrier_init(&sh.v_full[i], 128);
      barrier_init(&sh.k_empty[i], 2);
      barrier_init(&sh.v_empty[i], 2);
      barrier_init(&sh.s_full[i], 1);
      barrier_init(&sh.p_full[i], 128);
      barrier_init(&sh.done[i], 1);
    }
    barrier_init(&sh.where_full, 128);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(shared_at(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // the weights' warps bring the block's rows of q
  float scale = 0.f;
  int64_t lo = 1, hi = 0, token = 0;
  uint32_t q_head = 0;
  const uint32_t t = warp >> 2;  // the tile of a weights' warp
  const int64_t row = row_base + tid;
  if (warp < 8) {
    const bool has = row < row_all;
    if (has) {
      const uint32_t query = a.each_div.div((uint32_t)row);
      token = s.first + query;
      q_head = head * a.each + (uint32_t)row - query * a.each;
      const int64_t last = last_seen(a, s, query);
      lo = first_seen(a, last);
      hi = last + 1;
    }
    scale = stage_query<DT>(a, smem + W::q + t * W::tile, tid & 127, has, token * a.qt + q_head * a.qh);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  before_sync();
  __syncthreads();
  after_sync();
  const uint32_t tmem = sh.tmem, t_s = tmem + t * 128, t_o = tmem + 256 + t * DT;

  if (warp >= 8) {
    // ---- codes: a thread finds a position; then 8 (heads up to 64: 4) threads load one, 16 bytes each
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    const uint32_t j = tid - 256;
    constexpr uint32_t X = DT / 16;                           // 16-byte pieces of a position
    constexpr uint32_t PASS = 128 / X, N = kWideTile / PASS;  // positions at once, and how often
    const uint32_t piece = j % X, own = j / X;
    const bool in = piece * 16 < a.head;
    const int64_t table = sh.seq * a.ps;
    const uint8_t* const k_codes = a.k.codes + head * a.k.ch + piece * 16;
    const uint8_t* const v_codes = a.v.codes + head * a.v.ch + piece * 16;
    auto page_at = [&](uint32_t step) -> int32_t {  // of this thread's position; -1: not seen
      const int64_t p = range.lo + (int64_t)step * kWideTile + j;
      if (p >= range.hi) return -1;
      const int64_t g = load_index(a.pages, a.page_wide, table + a.page.div((uint32_t)p) * a.pp);
      return g >= 0 && g < a.pool ? (int32_t)g : -1;
    };
    float kappa = 0.f, nu = 0.f;
    uint32_t valid = 0;
    auto find = [&](uint32_t step, int32_t page) {
      const uint32_t p = (uint32_t)(range.lo + (int64_t)step * kWideTile + j), at = p - a.page.div(p) * a.page.d;
      const bool has = page >= 0;
      sh.where[step & 1][0][j] = has ? page * a.k.cp + at * a.k.cr : -1;
      sh.where[step & 1][1][j] = has ? page * a.v.cp + at * a.v.cr : -1;
      kappa = has ? __ldg(a.k.scales + page * a.k.sp + at * a.k.sr + head * a.k.sh) : 0.f;
      nu = has ? __ldg(a.v.scales + page * a.v.sp + at * a.v.sr + head * a.v.sh) : 0.f;
      valid = __ballot_sync(~0u, has);
      arrive(&sh.where_full);
    };
    auto load = [&](const uint8_t* codes, uint32_t step, uint32_t which, uint4 (&r)[N]) {
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        const int64_t at = sh.where[step & 1][which][i * PASS + own];
        r[i] = at >= 0 && in ? __ldg(reinterpret_cast<const uint4*>(codes + at)) : make_uint4(0, 0, 0, 0);
      }
    };
    // (the two halves of 8 threads in turn: no two of them in a bank)
    const uint32_t flip = piece >> 2;
    uint32_t put0 = (piece >> 2) * W::block + own * 128 + (((2 * (piece & 3) + flip) ^ (own & 7)) << 4);
    uint32_t put1 = (piece >> 2) * W::block + own * 128 + (((2 * (piece & 3) + 1 - flip) ^ (own & 7)) << 4);
    auto put = [&](uint8_t* tile, const uint4 (&r)[N]) {
#pragma unroll
      for (uint32_t i = 0; i < N; ++i) {
        // (PASS is a multiple of 8: the swizzle is the same for all of a thread's positions)
        const uint32_t w0 = raw<F>(flip ? r[i].z : r[i].x), w1 = raw<F>(flip ? r[i].w : r[i].y);
        const uint32_t w2 = raw<F>(flip ? r[i].x : r[i].z), w3 = raw<F>(flip ? r[i].y : r[i].w);
        *reinterpret_cast<uint4*>(tile + put0 + i * PASS * 128) = make_uint4(pair_low<F>(w0), pair_high<F>(w0), pair_low<F>(w1), pair_high<F>(w1));
        *reinterpret_cast<uint4*>(tile + put1 + i * PASS * 128) = make_uint4(pair_low<F>(w2), pair_high<F>(w2), pair_low<F>(w3), pair_high<F>(w3));
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    };
    uint4 rk[N], rv[N];
    bool ok = true;
    int32_t page = -1;
    if (steps) {
      find(0, page_at(0));
      page = steps > 1 ? page_at(1) : -1;
      ok = await(&sh.where_full, 0, &sh.dead);
      if (ok) load(k_codes, 0, 0, rk);
    }
    for (uint32_t i = 0; ok && i < steps; ++i) {
      const uint32_t st = i & 1, ring = i % kRings;
      load(v_codes, i, 1, rv);
      if (i >= 2 && !await(&sh.k_empty[st], (i / 2 - 1) & 1, &sh.dead)) break;
      put(smem + W::k + st * W::tile, rk);
      sh.kappa[ring][j] = kappa;
      sh.nu[ring][j] = nu;
      if (lane == 0) sh.valid[ring][warp - 8] = valid;
      arrive(&sh.k_full[st]);
      if (i + 1 < steps) {
        __syncwarp();
        find(i + 1, page);
        page = i + 2 < steps ? page_at(i + 2) : -1;
        if (!await(&sh.where_full, (i + 1) & 1, &sh.dead)) break;
        load(k_codes, i + 1, 0, rk);
      }
      if (i >= 2 && !await(&sh.v_empty[st], (i / 2 - 1) & 1, &sh.dead)) break;
      put(smem + W::v + st * W::tile, rv);
      arrive(&sh.v_full[st]);
    }
  } else {
    // ---- weights: a row a thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const uint32_t lanes = (warp & 3) << 21;  // (32 lanes a warp, in the upper half of an address)
    const bool issuer = (tid & 127) == 0;
    constexpr uint32_t to_s = instruction(kWideTile, false), to_o = instruction(DT, true);
    auto scores = [&](uint32_t st) {
      const uint32_t q = shared_at(smem + W::q + t * W::tile), k = shared_at(smem + W::k + st * W::tile);
#pragma unroll
      for (uint32_t e = 0; e < DT / 16; ++e) {
        const uint32_t by = (e >> 2) * W::block + (e & 3) * 32;
        product(t_s, descriptor(q + by, 16, 1024), descriptor(k + by, 16, 1024), to_s, e > 0);
      }
      commit(&sh.s_full[t]);
      commit(&sh.k_empty[st]);
    };
    auto values = [&](uint32_t st, bool add) {
      const uint32_t v = shared_at(smem + W::v + st * W::tile);
#pragma unroll
      for (uint32_t e = 0; e < kWideTile / 16; ++e)
        product_from_tmem(t_o, t_s + e * 8, descriptor(v + e * 2048, W::block, 1024), to_o, add || e > 0);
      if constexpr (SPLIT) {
#pragma unroll
        for (uint32_t e = 0; e < kWideTile / 16; ++e)
          product_from_tmem(t_o, t_s + 64 + e * 8, descriptor(v + e * 2048, W::block, 1024), to_o, true);
      }
      commit(&sh.v_empty[st]);
    };
    float m = -INFINITY, ref = 0.f, unit = 0.f, sum = 0.f;  // the row's maximum; what weights are relative to
    bool ok = true;
    if (issuer && steps) {
      ok = await(&sh.k_full[0], 0, &sh.dead);
      if (ok) {
        after_sync();
        scores(0);
      }
    }
    __syncwarp();
    // a step's weights; those of positions that the row does not see are 0
    auto step = [&](auto plain, uint32_t i, int from, int to) {
      constexpr bool PLAIN = decltype(plain)::value;
      const uint32_t ring = i % kRings;
      const float* const kappa = sh.kappa[ring];
      const float* const nu = sh.nu[ring];
      float r[128];
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) tmem_load(t_s + lanes + c * 32, r, c * 32);
      float most = fmaxf(fmaxf(nu[lane], nu[lane + 32]), fmaxf(nu[lane + 64], nu[lane + 96]));
      most = warp_max(most);
      await_loads();
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) {
        uint32_t bits = ~0u;
        if constexpr (!PLAIN) {
          const int l = min(max(from - (int)c * 32, 0), 32), h = min(max(to - (int)c * 32, 0), 32);
          bits = (h >= 32 ? ~0u : (1u << h) - 1) & ~(l >= 32 ? ~0u : (1u << l) - 1) & sh.valid[ring][c];
        }
#pragma unroll
        for (uint32_t e = 0; e < 32; e += 4) {
          const float4 k4 = *reinterpret_cast<const float4*>(kappa + c * 32 + e);
          float2 u = mul2(make_float2(r[c * 32 + e], r[c * 32 + e + 1]), make_float2(k4.x, k4.y));
          float2 v = mul2(make_float2(r[c * 32 + e + 2], r[c * 32 + e + 3]), make_float2(k4.z, k4.w));
          if constexpr (!PLAIN) {
            u.x = bits >> e & 1 ? u.x : -INFINITY;
            u.y = bits >> e & 2 ? u.y : -INFINITY;
            v.x = bits >> e & 4 ? v.x : -INFINITY;
            v.y = bits >> e & 8 ? v.y : -INFINITY;
          }
          r[c * 32 + e] = u.x;
          r[c * 32 + e + 1] = u.y;
          r[c * 32 + e + 2] = v.x;
          r[c * 32 + e + 3] = v.y;
          top[c] = fmaxf(fmaxf(top[c], u.x), u.y);
          top[c] = fmaxf(fmaxf(top[c], v.x), v.y);
        }
      }
      float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if (high > -INFINITY) high *= scale;
      // weights are at most 2^14: 2^8 at the reference, 2^4 from scores above the maximum, 2^2 from scales above their unit
      const bool larger = most > 4.f * unit;
      if (__any_sync(~0u, high > m + 4.f || larger)) {
        if (larger) unit = fmaxf(__uint_as_float(min((__float_as_uint(most) & 0x7f800000u) + 0x00800000u, 0x7e800000u)), 0x1p-90f);
        const float before = ref;
        const bool none = m == -INFINITY;
        m = fmaxf(m, high);
        // (log2 of a power of two)
        ref = (m > -INFINITY ? m : 0.f) + (unit > 0.f ? (float)((int)(__float_as_uint(unit) >> 23) - 127) : 0.f) - 8.f;
        const float f = none ? 0.f : ex2(before - ref);
        if (i) {
          sum *= f;
#pragma unroll 1
          for (uint32_t c = 0; c < DT / 16; ++c) {
            float o[16];
            tmem_load16(t_o + lanes + c * 16, o);
            await_loads();
#pragma unroll
            for (uint32_t e = 0; e < 16; ++e) o[e] *= f;
            tmem_store16(t_o + lanes + c * 16, *reinterpret_cast<const uint32_t (*)[16]>(&o));
          }
        }
      }
      float2 add[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
      for (uint32_t c = 0; c < 4; ++c) {
        uint32_t w[16];
        [[maybe_unused]] uint32_t low[SPLIT ? 16 : 1];
#pragma unroll
        for (uint32_t e = 0; e < 32; e += 4) {
          const float4 n4 = *reinterpret_cast<const float4*>(nu + c * 32 + e);
          float2 u = fma2(make_float2(r[c * 32 + e], r[c * 32 + e + 1]), both(scale), both(-ref));
          float2 v = fma2(make_float2(r[c * 32 + e + 2], r[c * 32 + e + 3]), both(scale), both(-ref));
          u = make_float2(ex2(u.x), ex2(u.y));
          v = make_float2(ex2(v.x), ex2(v.y));
          add[0] = add2(add[0], u);
          add[1] = add2(add[1], v);
          float2 y = mul2(u, make_float2(n4.x, n4.y)), z = mul2(v, make_float2(n4.z, n4.w));
          if constexpr (!PLAIN) {  // (no weight, whatever the scale is)
            y.x = u.x == 0.f ? 0.f : y.x;
            y.y = u.y == 0.f ? 0.f : y.y;
            z.x = v.x == 0.f ? 0.f : z.x;
            z.y = v.y == 0.f ? 0.f : z.y;
          }
          w[e / 2] = pack16(y);
          w[e / 2 + 1] = pack16(z);
          if constexpr (SPLIT) {
            const float2 y1 = __half22float2(*reinterpret_cast<const __half2*>(&w[e / 2])), z1 = __half22float2(*reinterpret_cast<const __half2*>(&w[e / 2 + 1]));
            low[e / 2] = pack16(make_float2(y.x - y1.x, y.y - y1.y));
            low[e / 2 + 1] = pack16(make_float2(z.x - z1.x, z.y - z1.y));
          }
        }
        tmem_store16(t_s + lanes + c * 16, w);
        if constexpr (SPLIT) tmem_store16(t_s + 64 + lanes + c * 16, low);
      }
      add[0] = add2(add[0], add[1]);
      sum += add[0].x + add[0].y;
    };
    for (uint32_t i = 0; i < steps; ++i) {
      ok = ok && await(&sh.k_full[i & 1], (i / 2) & 1, &sh.dead) && await(&sh.s_full[t], i & 1, &sh.dead);
      if (!__all_sync(~0u, ok)) break;
      after_sync();
      const int64_t p0 = range.lo + (int64_t)i * kWideTile;
      const int from = (int)max(min(lo - p0, (int64_t)kWideTile), (int64_t)0), to = (int)max(min(hi - p0, (int64_t)kWideTile), (int64_t)0);
      const uint32_t* const v = sh.valid[i % kRings];
      if (__all_sync(~0u, (v[0] & v[1] & v[2] & v[3]) == ~0u && from == 0 && to == (int)kWideTile)) step(std::true_type{}, i, 0, 0);
      else step(std::false_type{}, i, from, to);
      await_stores();
      before_sync();
      arrive(&sh.p_full[t]);
      if (issuer) {
        ok = await(&sh.p_full[t], i & 1, &sh.dead) && await(&sh.v_full[i & 1], (i / 2) & 1, &sh.dead);
        if (ok) {
          after_sync();
          values(i & 1, i > 0);
          if (i + 1 < steps) {
            ok = await(&sh.k_full[(i + 1) & 1], ((i + 1) / 2) & 1, &sh.dead);
            if (ok) {
              after_sync();
              scores((i + 1) & 1);
            }
          }
        }
      }
      __syncwarp();
    }
    if (issuer && steps) commit(&sh.done[t]);
    __syncwarp();
    // (what was issued has to end before TMEM is given back, on a way out too)
    int alone = 0;
    if (steps) ok = await(&sh.done[t], 0, &alone) && ok;
    // ---- the block's rows of the result
    if (!__all_sync(~0u, ok)) sum = NAN;  // given up: shows in the results
    after_sync();
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
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
  if (warp == 8) {
    after_sync();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem));
  }
}

template <int F, int DT, bool SPLIT>
void start_wide(const Args& a, cudaStream_t stream) {
  void (*const kernel)(const Args) = gpuos_attend_wide_kernel<F, DT, SPLIT>;
  cuda_ok(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Wide<DT>::total), "shared memory");
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
