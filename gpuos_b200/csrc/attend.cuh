// gpuos_attend for few rows: query rows over a paged cache of 8-bit codes.
// With s_j = scale * q . (K_j kappa_j), K and V codes, kappa and nu their scales,
//
//   m = max s_j     l = sum e^(s_j - m)     out = sum e^(s_j - m) nu_j V_j / l
//
// over the positions j that a query sees.  Each code is read once for all query heads
// of its key head and, of drafted tokens, for all queries: a block of 8, 16 or 32
// rows.  At so few rows memory is the bound, and an SM's share of it is 24 codes a
// cycle, so what a code costs in instructions counts:
//   - codes are whole numbers, or e4m3 numbers, that 16-bit floats hold exactly: a
//     code becomes one in about 1.4 instructions (e4m3 1.7), unscaled.  kappa_j multiplies the
//     finished product; nu_j goes into the 16-bit weight e^(s_j - m) nu_j;
//   - the codes are the matrix product's first operand (16 positions, or 16 elements of
//     the head, a step) and the 8 rows its second one, so that no row of it is idle;
//   - a row's maximum is raised only when a score passes it by 2^4;
//   - q is held as 16-bit floats times a power of two a row, nu_j relative to a
//     power of two that follows the largest that the row sees: 16-bit floats then lose nothing of a 16-bit q,
//     and half a step, 2^-11, of a weight down to 2^-22 of the largest: an eighth of what a bf16 result is
//     rounded by.  32-bit queries take q and weights in two parts (2^-22), 16-bit floats of 11 bits the weights.
// A warp takes 32 positions at a time through a ring of its own (no barrier in the
// loop).  Items (sequence, key head, block of rows) are laid end to end and the CTAs
// take equal shares of all units; what is split is joined by a second launch in a fixed order.
// 200001 and 150001 positions of 8 heads of 128, int8 (739 MB): 178 us a call (4.15 TB/s), some 10 of them the join;
// 64 sequences to 8000, e4m3 (816 MB): 210 to 215 us (3.85 TB/s).  A warp's 32 positions (8 KB) are about 1000
// instructions, at half of the issue slots: those, and that a warp's loads wait for its pages, are what is left.
// Prompts on this kernel (32-bit queries, heads above 128, scales of part of the head), 16 rows a block: 2048 queries of 32
// heads over 8 of 128, fp32: 1.0 ms, over 2: 1.35 ms, bf16 with scales of 32: 1.3 ms; the tensor cores' rate would allow 20 us.
#pragma once
#include "attend.h"

namespace gpuos {
namespace rowops {
namespace attend {
namespace {

constexpr uint32_t kTile = 32;
constexpr float kSmallestUnit = 0x1p-100f;

// How a kernel lays out its shared memory.
template <int DT, int NT, bool GEN>
struct Layout {
  static constexpr uint32_t rows = 8 * NT;
  static constexpr uint32_t per_sm = ctas(DT, NT);
  static constexpr uint32_t stages = GEN || per_sm == 3 ? 2 : 3;
  static constexpr uint32_t scales = GEN ? DT / 32 : 1;                 // of a row, room for
  static constexpr uint32_t codes = kTile * DT;                         // bytes, of K or V
  static constexpr uint32_t stage = 2 * codes + 2 * kTile * scales * 4 + 16;
  static constexpr uint32_t ring = stages * stage > rows * DT * 4 ? stages * stage : rows * DT * 4;  // of a warp
  static constexpr uint32_t q_row = DT * 2 + 64;                        // bytes: 4 of 8 16-byte banks further each row
  static constexpr uint32_t q = rows * q_row * (GEN ? 2 : 1);
  static constexpr uint32_t total = kWarps * ring + q;
};

// Where the 16 bytes x of a row of codes lie: rows of 8 (K) and every second row (V) are read
// together without two of them in a bank.
template <int DT>
__device__ __forceinline__ uint32_t place(uint32_t row, uint32_t x) {
  if constexpr (DT == 64) {
    const uint32_t line = row >> 1;
    return line * 128 + ((((row & 1) * 4 + x) ^ ((line & 3) << 1)) << 4);
  } else {
    return row * DT + ((x ^ ((((row >> 1) & 3) << 1) ^ ((row & 1) << 2))) << 4);
  }
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool has) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(has ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool has) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(has ? 4 : 0) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }

// Items are laid out in units: blocks of a head, heads of a sequence, sequences.  A CTA's share begins at an edge: a unit
// of an item (or its end), and the units before it.  Edges are looked for once, by a thread for each, or by all threads
// where a sequence has many blocks; from there a CTA steps from item to item.
struct Edge {
  uint32_t seq, head, block, from;
  int64_t at;
};
constexpr uint32_t kFewBlocks = 64;  // that a thread walks over by itself: 100 cycles each, where a step of all takes some 500

template <uint32_t RB>
__device__ __forceinline__ uint32_t blocks(const Args& a, const Sequence& s) {
  const int64_t rows = s.n * a.each;
  return rows > a.few ? 0 : (uint32_t)((rows + RB - 1) / RB);
}
template <uint32_t RB>
__device__ __forceinline__ Range block_range(const Args& a, const Sequence& s, uint32_t b) {
  const int64_t first = (int64_t)b * RB, last = min(first + RB, s.n * a.each) - 1;
  return seen(a, s, a.each_div.div((uint32_t)first), a.each_div.div((uint32_t)last));
}
__device__ __forceinline__ uint32_t units_of(const Range& r) { return max((uint32_t)((r.hi - r.lo + kUnit - 1) / kUnit), 1u); }

// Units of a head of a sequence.
template <uint32_t RB>
__device__ __forceinline__ int64_t head_units(const Args& a, const Sequence& s) {
  const uint32_t n = blocks<RB>(a, s);
  int64_t u = 0;
  for (uint32_t b = 0; b < n; ++b) u += units_of(block_range<RB>(a, s, b));
  return u;
}
// The same by all threads together.
template <uint32_t RB>
__device__ __noinline__ int64_t head_units_together(const Args& a, const Sequence& s, int64_t (&sums)[kWarps]) {
  const uint32_t n = blocks<RB>(a, s);
  int64_t u = 0;
  for (uint32_t b = threadIdx.x; b < n; b += kThreads) u += units_of(block_range<RB>(a, s, b));
  for (int d = 16; d; d >>= 1) u += __shfl_xor_sync(~0u, u, d);
  __syncthreads();
  if (threadIdx.x % 32 == 0) sums[threadIdx.x / 32] = u;
  __syncthreads();
  u = 0;
  for (uint32_t w = 0; w < kWarps; ++w) u += sums[w];
  return u;
}

// The edge at unit u, block `b` of which it is unit `from` of `units`.  Short items stay whole: it is moved to their end.
__device__ __forceinline__ Edge edge_in(uint32_t seq, uint32_t head, uint32_t b, uint32_t from, uint32_t units, int64_t u) {
  const uint32_t to = from && units <= kWhole ? units : from;
  return Edge{seq, head, b, to, u + to - from};
}
// The edge at unit u, in sequence s whose first unit is `at`.
template <uint32_t RB>
__device__ __forceinline__ Edge find(const Args& a, uint32_t seq, const Sequence& s, int64_t per_head, int64_t u, int64_t at) {
  const uint32_t head = (uint32_t)((u - at) / per_head);
  int64_t rest = u - at - head * per_head;
  for (uint32_t b = 0;; ++b) {
    const uint32_t units = units_of(block_range<RB>(a, s, b));
    if (rest < units) return edge_in(seq, head, b, (uint32_t)rest, units, u);
    rest -= units;
  }
}
// The same by all threads together: one of them finds it.
template <uint32_t RB>
__device__ __noinline__ void find_together(const Args& a, uint32_t seq, const Sequence& s, int64_t per_head, int64_t u, int64_t at,
                                           int64_t (&sums)[kWarps], Edge& to) {
  const uint32_t n = blocks<RB>(a, s), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t head = (uint32_t)((u - at) / per_head);
  int64_t rest = u - at - head * per_head;
  for (uint32_t b0 = 0; b0 < n; b0 += kThreads) {
    const uint32_t b = b0 + threadIdx.x, units = b < n ? units_of(block_range<RB>(a, s, b)) : 0;
    int64_t until = units;
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(~0u, until, d);
      if (lane >= d) until += o;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = until;
    __syncthreads();
    int64_t total = 0;
    for (uint32_t w = 0; w < kWarps; ++w) {
      if (w == warp) until += total;
      total += sums[w];
    }
    if (rest < total) {
      if (until - units <= rest && rest < until) to = edge_in(seq, head, b, (uint32_t)(rest - (until - units)), units, u);
      return;
    }
    rest -= total;
  }
}

template <int F, int DT, int NT, bool GEN>
__global__ void __launch_bounds__(kThreads, ctas(DT, NT))
gpuos_attend_kernel(const __grid_constant__ Args a) {
  using L = Layout<DT, NT, GEN>;
  constexpr uint32_t RB = L::rows, kStages = L::stages;
  constexpr uint32_t MT = DT / 16;             // steps over the head's elements
  constexpr uint32_t HB = DT / 32;             // blocks of 32 elements
  // Weights are at most 2^14: 2^kSlack from scores that pass the row's maximum, 2^kSlackV from scales that pass
  // their unit, and the rest as a factor, so that small weights stay among the normal 16-bit numbers.
  constexpr int kSlack = GEN ? 0 : 4, kSlackV = GEN ? 0 : 2, kUp = 14 - kSlack - kSlackV;
  constexpr float kMostPer = (float)(1 << kUp) / kSmallestUnit;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t thread_units[kThreads + 1];
  __shared__ Edge edge[2];
  __shared__ int64_t sums[kWarps];
  __shared__ uint32_t turn;
  __shared__ float row_scale[RB];              // of a row's q, times scale * log2(e)
  __shared__ int64_t row_lo[RB], row_hi[RB];   // positions a row sees
  __shared__ float part_m[kWarps][RB], part_l[kWarps][RB], part_e[kWarps][RB];

  const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  uint8_t* const ring = smem + warp * L::ring;
  uint8_t* const sq = smem + kWarps * L::ring;
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);

  asm volatile("griddepcontrol.launch_dependents;");
  // tokens of no sequence get zeros
  if (a.offsets) {
    const int64_t end = min(max(load_index(a.offsets, a.offset_wide, (int64_t)a.sequences * a.os), (int64_t)0), (int64_t)a.tokens);
    const int64_t before = min(max(load_index(a.offsets, a.offset_wide, 0), (int64_t)0), end);
    const uint32_t heads = a.k_heads * a.each;
    for (int64_t i = blockIdx.x * kWarps + warp; i < (before + a.tokens - end) * heads; i += (int64_t)a.grid * kWarps) {
      int64_t t = i / heads;
      const int64_t h = i - t * heads;
      if (t >= before) t += end - before;
      for (uint32_t e = lane; e < a.head; e += 32) store_real(a.out, a.type, t * a.ot + h * a.oh + e, 0.f);
      if (a.lse && lane == 0) a.lse[t * a.lt + h * a.lh] = -INFINITY;
    }
  }

  // ---- this CTA's share: where unit blockIdx.x * per begins, and the next CTA's
  const uint32_t per_thread = (a.sequences + kThreads - 1) / kThreads;
  const uint32_t s0 = min(tid * per_thread, a.sequences), s1 = min(s0 + per_thread, a.sequences);
  bool large = false;  // whether a sequence has many blocks
  {
    int64_t u = 0;
    for (uint32_t s = s0; s < s1; ++s) {
      const Sequence q = sequence(a, s);
      if (blocks<RB>(a, q) > kFewBlocks) large = true;
      else u += a.k_heads * head_units<RB>(a, q);
    }
    large = __syncthreads_or(large);
    if (large) {
      uint32_t s = s0;  // the next of this thread's that has
      for (;;) {
        while (s < s1 && blocks<RB>(a, sequence(a, s)) <= kFewBlocks) ++s;
        if (tid == 0) turn = ~0u;
        __syncthreads();
        if (s < s1) atomicMin(&turn, s);
        __syncthreads();
        const uint32_t now = turn;
        if (now == ~0u) break;
        const int64_t n = head_units_together<RB>(a, sequence(a, now), sums);
        if (s < s1 && s == now) u += a.k_heads * n, ++s;  // (another's first is where this thread's end)
      }
    }
    int64_t sum = u;
    for (uint32_t d = 1; d < 32; d <<= 1) {
      const int64_t o = __shfl_up_sync(~0u, sum, d);
      if (lane >= d) sum += o;
    }
    thread_units[tid + 1] = sum;  // within the warp
    __syncthreads();
    int64_t ahead = 0;
    for (uint32_t w = 0; w < warp; ++w) ahead += thread_units[(w + 1) * 32];
    __syncthreads();
    thread_units[tid + 1] = sum + ahead;
    if (tid == 0) thread_units[0] = 0;
    __syncthreads();
  }
  const int64_t all = thread_units[kThreads];
  const int64_t per = max((all + a.grid - 1) / a.grid, (int64_t)1);
  if (blockIdx.x * per >= all) {
    if (tid == 0 && a.split) a.split[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  for (int i = 0; i < 2; ++i) {
    const int64_t u = (blockIdx.x + i) * per;
    if (u >= all) {
      if (tid == 0) edge[i].at = all;
      continue;
    }
    const bool here = thread_units[tid] <= u && u < thread_units[tid + 1];
    if (!large) {
      if (here) {
        int64_t at = thread_units[tid];
        for (uint32_t s = s0; s < s1; ++s) {
          const Sequence q = sequence(a, s);
          const int64_t n = head_units<RB>(a, q);
          if (u < at + a.k_heads * n) {
            edge[i] = find<RB>(a, s, q, n, u, at);
            break;
          }
          at += a.k_heads * n;
        }
      }
    } else {
      __syncthreads();  // (`turn` has been read)
      if (here) turn = tid;
      __syncthreads();
      int64_t at = thread_units[turn];
      for (uint32_t s = turn * per_thread; s < a.sequences; ++s) {
        const Sequence q = sequence(a, s);
        const int64_t n = head_units_together<RB>(a, q, sums);
        if (u < at + a.k_heads * n) {
          find_together<RB>(a, s, q, n, u, at, sums, edge[i]);
          break;
        }
        at += a.k_heads * n;
      }
    }
  }
  __syncthreads();
  int64_t todo = edge[1].at - edge[0].at;
  Edge it = edge[0];  // (`at` is not kept up)
  Sequence s{};
  uint32_t count = 0;  // blocks of the sequence
  if (todo > 0) {
    s = sequence(a, it.seq);
    count = blocks<RB>(a, s);
  }
  int4 goes_on = make_int4(0, 0, 0, 0);

  while (todo > 0) {
    // ---- the item, and how much of it is this CTA's
    const Range range = block_range<RB>(a, s, it.block);
    const uint32_t units = units_of(range);
    if (it.from == units) {  // on to the next one, which there is
      it.from = 0;
      if (++it.block == count) {
        it.block = 0;
        if (++it.head == a.k_heads) {
          it.head = 0;
          for (count = 0; count == 0 && ++it.seq < a.sequences;) {
            s = sequence(a, it.seq);
            count = blocks<RB>(a, s);
          }
          if (count == 0) break;  // (only if lengths or offsets have changed meanwhile)
        }
      }
      continue;
    }
    const uint32_t take = (uint32_t)min((int64_t)(units - it.from), todo);
    const uint32_t begin = (uint32_t)(range.lo + it.from * kUnit) + warp * kTile, stop = (uint32_t)range.hi;  // (below 2^31 + 2^8)
    const uint32_t row0 = it.block * RB, row_count = (uint32_t)min((int64_t)RB, s.n * a.each - row0);
    // positions that every row sees
    const int64_t all_hi = last_seen(a, s, a.each_div.div(row0)) + 1;
    const int64_t all_lo = first_seen(a, last_seen(a, s, a.each_div.div(row0 + row_count - 1)));

    // ---- loads: 32 positions of this warp into a stage
    const int64_t table = it.seq * a.ps;
    const uint8_t* const k_codes = a.k.codes + it.head * a.k.ch;
    const uint8_t* const v_codes = a.v.codes + it.head * a.v.ch;
    const float* const k_scales = a.k.scales + it.head * a.k.sh;
    const float* const v_scales = a.v.scales + it.head * a.v.sh;
    auto page_at = [&](uint32_t j) -> int32_t {  // of position j; -1 where there is none
      if (j >= stop) return -1;
      const int64_t p = load_index(a.pages, a.page_wide, table + a.page.div(j) * a.pp);
      return p >= 0 && p < a.pool ? (int32_t)p : -1;
    };
    int32_t next_page = page_at(begin + lane);
    uint32_t fill = 0;                          // the stage that is filled next
    auto issue = [&](uint32_t i) {  // unit i of the share
      if (i < take) {
        const uint32_t to = ring_at + fill;
        const uint32_t j = begin + i * kUnit + lane;
        const int32_t page = next_page;
        if (i + 1 < take) next_page = page_at(j + kUnit);
        const uint32_t row = j - a.page.div(j) * a.page.d;
        const bool has = page >= 0;
        const int64_t k_at = has ? page * a.k.cp + row * a.k.cr : 0;
        const int64_t v_at = a.alike ? k_at : has ? page * a.v.cp + row * a.v.cr : 0;
        const uint32_t valid = __ballot_sync(~0u, has);
        constexpr uint32_t X = DT / 16;
        if (a.vec == 16) {
          const uint32_t x = lane % X;
          const bool inside = x * 16 < a.head;
#pragma unroll
          for (uint32_t r0 = 0; r0 < X; ++r0) {
            const uint32_t r = r0 * (32 / X) + lane / X;
            const int64_t ko = __shfl_sync(~0u, k_at, r), vo = a.alike ? ko : __shfl_sync(~0u, v_at, r);
            const bool in = (valid >> r & 1) && inside;
            const uint32_t at = place<DT>(r, x);
            copy16(to + at, k_codes + ko + (inside ? x * 16 : 0), in);
            copy16(to + L::codes + at, v_codes + vo + (inside ? x * 16 : 0), in);
          }
        } else {
          uint8_t* const stage = ring + fill;
          for (uint32_t r = 0; r < kTile; ++r) {
            const int64_t ko = __shfl_sync(~0u, k_at, r), vo = __shfl_sync(~0u, v_at, r);
            const bool in = valid >> r & 1;
            for (uint32_t e = lane * 4; e < DT; e += 128) {
              const uint32_t at = place<DT>(r, e >> 4) + (e & 15);
              if (a.vec == 4) {
                copy4(to + at, k_codes + ko + (in && e < a.head ? e : 0), in && e < a.head);
                copy4(to + L::codes + at, v_codes + vo + (in && e < a.head ? e : 0), in && e < a.head);
              } else {
#pragma unroll
                for (uint32_t b = 0; b < 4; ++b) {
                  stage[at + b] = in && e < a.head ? k_codes[ko + e + b] : 0;
                  stage[L::codes + at + b] = in && e < a.head ? v_codes[vo + e + b] : 0;
                }
              }
            }
          }
        }
        const uint32_t sc = to + 2 * L::codes;
        const int64_t ks = has ? page * a.k.sp + row * a.k.sr : 0;
        const int64_t vs = a.alike ? ks : has ? page * a.v.sp + row * a.v.sr : 0;
        for (uint32_t gr = 0; gr < (GEN ? a.groups : 1); ++gr) {
          copy4(sc + (gr * kTile + lane) * 4, k_scales + ks + gr * a.k.sg, has);
          copy4(sc + ((L::scales + gr) * kTile + lane) * 4, v_scales + vs + gr * a.v.sg, has);
        }
        if (lane == 0) *reinterpret_cast<uint32_t*>(ring + fill + 2 * L::codes + 2 * kTile * L::scales * 4) = valid;
        fill = fill + L::stage == kStages * L::stage ? 0 : fill + L::stage;
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (uint32_t i = 0; i + 1 < kStages; ++i) issue(i);

    // ---- the block's rows of q: a warp takes every fourth row, all of them loaded before the first is looked at
    {
      constexpr uint32_t E = DT / 32, MINE = RB / kWarps;
      float v[MINE][E];
      uint32_t query[MINE];
#pragma unroll
      for (uint32_t k = 0; k < MINE; ++k) {
        const uint32_t r = warp + k * kWarps;
        query[k] = r < row_count ? a.each_div.div(row0 + r) : 0;
        const int64_t base = (s.first + query[k]) * a.qt + (int64_t)(it.head * a.each + row0 + r - query[k] * a.each) * a.qh;
#pragma unroll
        for (uint32_t i = 0; i < E; ++i) {
          const uint32_t e = i * 32 + lane;
          v[k][i] = r < row_count && e < a.head ? load_real(a.q, a.type, base + e) : 0.f;
        }
      }
#pragma unroll
      for (uint32_t k = 0; k < MINE; ++k) {
        const uint32_t r = warp + k * kWarps;
        float most = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < E; ++i) most = fmaxf(most, fabsf(v[k][i]));
        most = warp_max(most);
        // times a power of two that puts the largest into [2^14, 2^15): 16-bit floats reach 2^-29 of it
        int shift = 14 - (int)((__float_as_uint(most) >> 23) - 127);
        if (!(most > 0.f)) shift = 0;
        const float up = __uint_as_float((uint32_t)(min(max(shift, -126), 126) + 127) << 23);  // (in two steps for the smallest)
        const float more = __uint_as_float((uint32_t)(shift - min(max(shift, -126), 126) + 127) << 23);
#pragma unroll
        for (uint32_t i = 0; i < E; ++i) {
          const uint32_t e = i * 32 + lane;
          const float y = v[k][i] * up * more;
          const __half hi = __float2half_rn(y);
          *reinterpret_cast<__half*>(sq + r * L::q_row + e * 2) = hi;
          if (GEN) *reinterpret_cast<__half*>(sq + (RB + r) * L::q_row + e * 2) = __float2half_rn(a.split_q ? y - __half2float(hi) : 0.f);
        }
        if (lane == 0) {
          row_scale[r] = a.scale2 / up / more;
          const int64_t last = last_seen(a, s, query[k]);
          row_lo[r] = r < row_count ? first_seen(a, last) : 1;
          row_hi[r] = r < row_count ? last + 1 : 0;
        }
      }
    }
    __syncthreads();
    float scale[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      scale[t][0] = row_scale[8 * t + 2 * c];
      scale[t][1] = row_scale[8 * t + 2 * c + 1];
    }
    uint4 qf[NT == 1 && !GEN ? HB : 1];
    if constexpr (NT == 1 && !GEN) {
#pragma unroll
      for (uint32_t b = 0; b < HB; ++b) qf[b] = *reinterpret_cast<const uint4*>(sq + g * L::q_row + b * 64 + c * 16);
    }

    float o[MT][NT][4];
#pragma unroll
    for (uint32_t i = 0; i < MT; ++i)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][t][k] = 0.f;
    // per_v: 2^kUp / the power of two that nu is relative to, a row's own (a scale that a row does not see changes nothing of it)
    float m[NT][2], l[NT][2], per_v[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) m[t][0] = m[t][1] = -INFINITY, l[t][0] = l[t][1] = 0.f, per_v[t][0] = per_v[t][1] = kMostPer;

    uint32_t drain = 0;  // the stage that is read next
    for (uint32_t i = 0; i < take; ++i) {
      __syncwarp();  // the stage that is filled next has been read by all
      issue(i + kStages - 1);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      __syncwarp();
      const uint8_t* const stage = ring + drain;
      drain = drain + L::stage == kStages * L::stage ? 0 : drain + L::stage;
      const float* const kappa = reinterpret_cast<const float*>(stage + 2 * L::codes);
      const float* const nu = kappa + L::scales * kTile;
      const uint32_t valid = *reinterpret_cast<const uint32_t*>(nu + L::scales * kTile);

      // the largest scale of V (one that is not finite is left out: a row gets NaN from it where it sees it)
      float most = 0.f;
      for (uint32_t gr = 0; gr < (GEN ? a.groups : 1); ++gr) {
        const float x = fabsf(nu[gr * kTile + lane]);
        most = fmaxf(most, x < INFINITY ? x : 0.f);
      }
      most = warp_max(most);

      // scores of 32 positions (rows g and g + 8 of two products) x NT * 8 rows
      float sc[2][NT][4];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) sc[h][t][k] = 0.f;
      float acc[GEN ? 2 : 1][GEN ? NT : 1][4];
      if constexpr (GEN) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[h][t][k] = 0.f;
      }
#pragma unroll
      for (uint32_t b = 0; b < HB; ++b) {
        uint4 qb[NT], ql[GEN ? NT : 1];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (NT == 1 && !GEN) qb[t] = qf[b];
          else qb[t] = *reinterpret_cast<const uint4*>(sq + (8 * t + g) * L::q_row + b * 64 + c * 16);
          if constexpr (GEN) ql[t] = *reinterpret_cast<const uint4*>(sq + (RB + 8 * t + g) * L::q_row + b * 64 + c * 16);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint2 w0 = *reinterpret_cast<const uint2*>(stage + place<DT>(16 * h + g, 2 * b + (c >> 1)) + (c & 1) * 8);
          const uint2 w1 = *reinterpret_cast<const uint2*>(stage + place<DT>(16 * h + g + 8, 2 * b + (c >> 1)) + (c & 1) * 8);
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint32_t x0 = raw<F>(k ? w0.y : w0.x), x1 = raw<F>(k ? w1.y : w1.x);
            const uint32_t a0 = pair_low<F>(x0), a1 = pair_low<F>(x1), a2 = pair_high<F>(x0), a3 = pair_high<F>(x1);
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if constexpr (GEN) {
                mma(acc[h][t], a0, a1, a2, a3, k ? qb[t].z : qb[t].x, k ? qb[t].w : qb[t].y);
                if (a.split_q) mma(acc[h][t], a0, a1, a2, a3, k ? ql[t].z : ql[t].x, k ? ql[t].w : ql[t].y);
              } else {
                mma(sc[h][t], a0, a1, a2, a3, k ? qb[t].z : qb[t].x, k ? qb[t].w : qb[t].y);
              }
            }
          }
        }
        if constexpr (GEN) {
          if ((b + 1) * 32 % a.group == 0 || b + 1 == HB) {
            const uint32_t gr = min(b * 32 / a.group, a.groups - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float k0 = kappa[gr * kTile + 16 * h + g], k1 = kappa[gr * kTile + 16 * h + g + 8];
#pragma unroll
              for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  sc[h][t][k] = fmaf(acc[h][t][k], k < 2 ? k0 : k1, sc[h][t][k]);
                  acc[h][t][k] = 0.f;
                }
            }
          }
        }
      }
      const int64_t j0 = begin + i * kUnit;
      const bool plain = valid == ~0u && j0 >= all_lo && j0 + kTile <= all_hi;
      // the scales of V are relative to a power of two, which is raised when those that the row sees pass it by 2^kSlackV
      constexpr float kPass = (float)(1 << (kUp + kSlackV));
      bool higher = false, over = false;
#pragma unroll
      for (int t = 0; t < NT; ++t) over |= most * fmaxf(per_v[t][0], per_v[t][1]) > kPass;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float k0 = GEN ? 1.f : kappa[16 * h + g], k1 = GEN ? 1.f : kappa[16 * h + g + 8];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 4; ++k) sc[h][t][k] *= scale[t][k & 1] * (k < 2 ? k0 : k1);
      }
      if (!plain) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const int64_t lo = row_lo[8 * t + 2 * c + k] - j0, hi = row_hi[8 * t + 2 * c + k] - j0;
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              const int at = g + 8 * p;
              if (!(at >= lo && at < hi && (valid >> at & 1))) sc[p >> 1][t][(p & 1) * 2 + k] = -INFINITY;
            }
          }
      }
      float top[NT][2];
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          top[t][k] = fmaxf(fmaxf(sc[0][t][k], sc[0][t][k + 2]), fmaxf(sc[1][t][k], sc[1][t][k + 2]));
          higher |= top[t][k] > m[t][k] + (float)kSlack;  // (from nothing: -inf)
        }
      const bool raise = __any_sync(~0u, higher || over);
      if (raise) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float x = fmaxf(top[t][k], m[t][k]);
            for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(~0u, x, d));
            const float f = x == m[t][k] ? 1.f : ex2(m[t][k] - x);
            l[t][k] *= f;
            m[t][k] = x;
#pragma unroll
            for (uint32_t d = 0; d < MT; ++d) o[d][t][k] *= f, o[d][t][k + 2] *= f;
          }
      }
      if (raise && __any_sync(~0u, over)) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            float own = most;
            if (!plain) {
              own = 0.f;
              for (uint32_t gr = 0; gr < (GEN ? a.groups : 1); ++gr)
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                  const float x = fabsf(nu[gr * kTile + 8 * p + g]);
                  if (sc[p >> 1][t][(p & 1) * 2 + k] != -INFINITY && x < INFINITY) own = fmaxf(own, x);
                }
              for (int d = 4; d < 32; d <<= 1) own = fmaxf(own, __shfl_xor_sync(~0u, own, d));
            }
            if (own * per_v[t][k] > kPass) {
              const float up = fmaxf(__uint_as_float(min((__float_as_uint(own) & 0x7f800000u) + 0x00800000u, 0x7e800000u)), kSmallestUnit);
              const float per = __uint_as_float(0x7f000000u + (kUp << 23) - __float_as_uint(up)), f = per / per_v[t][k];
#pragma unroll
              for (uint32_t d = 0; d < MT; ++d) o[d][t][k] *= f, o[d][t][k + 2] *= f;
              per_v[t][k] = per;
            }
          }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const float from = m[t][k] == -INFINITY ? 0.f : m[t][k];
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            float& x = sc[p >> 1][t][(p & 1) * 2 + k];
            x = ex2(x - from);
            l[t][k] += x;
            x *= per_v[t][k];
          }
        }
      uint32_t bf[2][NT][2], bl[GEN ? 2 : 1][GEN ? NT : 1][2];
      auto weights = [&](uint32_t gr) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            const float w = nu[gr * kTile + 16 * h + 8 * q + g];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              // (a weight of 0 stays 0 whatever the scale is)
              const float x0 = sc[h][t][2 * q], x1 = sc[h][t][2 * q + 1];
              const float y0 = x0 == 0.f ? 0.f : x0 * w, y1 = x1 == 0.f ? 0.f : x1 * w;
              const uint32_t hi = pack(y0, y1);
              bf[h][t][q] = transposed(hi);
              if constexpr (GEN) {
                const float2 r = unpack(hi);
                bl[h][t][q] = transposed(pack(y0 - r.x, y1 - r.y));
              }
            }
          }
      };
      if constexpr (!GEN) weights(0);
      const uint8_t* const vs = stage + L::codes;
      if constexpr (!GEN) {
        // a lane's elements: 16 neighbours (8 of heads of 64) of each 128, those of a step two of them
        constexpr uint32_t HALVES = DT == 256 ? 2 : 1, W = DT == 64 ? 2 : 4;
#pragma unroll
        for (uint32_t half = 0; half < HALVES; ++half)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[4][W];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              const uint32_t r = 16 * h + 2 * c + (p & 1) + (p >> 1) * 8;
              if constexpr (DT == 64) {
                const uint2 x = *reinterpret_cast<const uint2*>(vs + place<DT>(r, g >> 1) + (g & 1) * 8);
                w[p][0] = raw<F>(x.x), w[p][1] = raw<F>(x.y);
              } else {
                const uint4 x = *reinterpret_cast<const uint4*>(vs + place<DT>(r, half * 8 + g));
                w[p][0] = raw<F>(x.x), w[p][1] = raw<F>(x.y), w[p][2] = raw<F>(x.z), w[p][3] = raw<F>(x.w);
              }
            }
#pragma unroll
            for (uint32_t k = 0; k < W; ++k)
#pragma unroll
              for (uint32_t e = 0; e < 2; ++e) {
                const uint32_t x = __byte_perm(w[0][k], w[1][k], e ? 0x7362 : 0x5140);
                const uint32_t y = __byte_perm(w[2][k], w[3][k], e ? 0x7362 : 0x5140);
                const uint32_t a0 = pair_low<F>(x), a1 = pair_high<F>(x), a2 = pair_low<F>(y), a3 = pair_high<F>(y);
#pragma unroll
                for (int t = 0; t < NT; ++t) mma(o[half * 8 + 2 * k + e][t], a0, a1, a2, a3, bf[h][t][0], bf[h][t][1]);
              }
          }
      } else {
        // four neighbours of each 32
#pragma unroll
        for (uint32_t b = 0; b < HB; ++b) {
          if (b * 32 % a.group == 0) weights(min(b * 32 / a.group, a.groups - 1));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            uint32_t w[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
              const uint32_t r = 16 * h + 2 * c + (p & 1) + (p >> 1) * 8;
              w[p] = raw<F>(*reinterpret_cast<const uint32_t*>(vs + place<DT>(r, 2 * b + (g >> 2)) + (g & 3) * 4));
            }
#pragma unroll
            for (uint32_t e = 0; e < 2; ++e) {
              const uint32_t x = __byte_perm(w[0], w[1], e ? 0x7362 : 0x5140);
              const uint32_t y = __byte_perm(w[2], w[3], e ? 0x7362 : 0x5140);
              const uint32_t a0 = pair_low<F>(x), a1 = pair_high<F>(x), a2 = pair_low<F>(y), a3 = pair_high<F>(y);
#pragma unroll
              for (int t = 0; t < NT; ++t) {
                mma(o[2 * b + e][t], a0, a1, a2, a3, bf[h][t][0], bf[h][t][1]);
                if (a.split_p) mma(o[2 * b + e][t], a0, a1, a2, a3, bl[h][t][0], bl[h][t][1]);
              }
            }
          }
        }
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncwarp();

    // ---- the warps' results joined
    float* const part = reinterpret_cast<float*>(ring);  // (row, element) of this warp
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x = l[t][k];
        for (int d = 4; d < 32; d <<= 1) x += __shfl_xor_sync(~0u, x, d);
        const uint32_t r = 8 * t + 2 * c + k;
        if (g == 0) part_m[warp][r] = m[t][k], part_l[warp][r] = x, part_e[warp][r] = 1.f / per_v[t][k];
#pragma unroll
        for (uint32_t d = 0; d < MT; ++d) {
          const uint32_t e = GEN ? (d >> 1) * 32 + g * 4 + (d & 1) * 2
                                 : DT == 64 ? g * 8 + d * 2 : (d >> 3) * 128 + g * 16 + (d & 7) * 2;
          part[r * DT + e] = o[d][t][k];
          part[r * DT + e + 1] = o[d][t][k + 2];
        }
      }
    __syncthreads();
    const bool whole = it.from == 0 && take == units;
    float* const slot = a.partial + ((size_t)blockIdx.x * 2 + (it.from == 0)) * RB * (a.head + 2);
    for (uint32_t r = warp; r < row_count; r += kWarps) {
      float top = part_m[0][r];
#pragma unroll
      for (uint32_t w = 1; w < kWarps; ++w) top = fmaxf(top, part_m[w][r]);
      float f[kWarps], sum = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < kWarps; ++w) {
        f[w] = part_m[w][r] == -INFINITY ? 0.f : ex2(part_m[w][r] - top);
        sum += f[w] * part_l[w][r];
        f[w] *= part_e[w][r];
      }
      const uint32_t query = a.each_div.div(row0 + r), h = it.head * a.each + row0 + r - query * a.each;
      const int64_t t = s.first + query;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      for (uint32_t e = lane; e < a.head; e += 32) {
        float x = 0.f;
#pragma unroll
        for (uint32_t w = 0; w < kWarps; ++w)
          if (f[w] != 0.f) x += f[w] * reinterpret_cast<const float*>(smem + w * L::ring)[r * DT + e];
        if (whole) store_real(a.out, a.type, t * a.ot + h * a.oh + e, x * inv);
        else slot[r * (a.head + 2) + e] = x;
      }
      if (lane == 0) {
        if (!whole) {
          slot[r * (a.head + 2) + a.head] = top;
          slot[r * (a.head + 2) + a.head + 1] = sum;
        } else if (a.lse) {
          a.lse[t * a.lt + h * a.lh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718056f;
        }
      }
    }
    if (it.from == 0 && !whole) {
      // the CTAs behind this one go on with it, a share each
      const int64_t rest = units - take;
      goes_on = make_int4((int)it.seq, (int)it.head, (int)it.block, (int)((rest + per - 1) / per));
    }
    __syncthreads();
    todo -= take;
    it.from += take;
  }
  if (tid == 0 && a.split) a.split[blockIdx.x] = goes_on;
}

// Joins the parts of split items: a CTA takes a row of every 8, its warps parts of it, and all sums are in a fixed order.
// (Launched while the other kernel runs, so that its start is not waited for: it waits here.)
template <uint32_t RB>
__global__ void __launch_bounds__(256) gpuos_attend_join_kernel(const __grid_constant__ Args a) {
  __shared__ float sums[8][kMaxHead + 2];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int4 it = a.split[blockIdx.x];
  if (it.w == 0) return;
  const Sequence s = sequence(a, (uint32_t)it.x);
  const uint32_t row0 = (uint32_t)it.z * RB, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rows = (uint32_t)min((int64_t)RB, s.n * a.each - row0);
  const uint32_t stride = a.head + 2;
  for (uint32_t r = blockIdx.y; r < rows; r += gridDim.y) {
    auto part = [&](int i) { return a.partial + (((size_t)blockIdx.x + i) * 2 + (i == 0)) * RB * stride + r * stride; };
    float top = -INFINITY;
    for (int i = lane; i <= it.w; i += 32) top = fmaxf(top, part(i)[a.head]);
    top = warp_max(top);
    float sum = 0.f, x[kMaxHead / 32];
#pragma unroll
    for (uint32_t k = 0; k < kMaxHead / 32; ++k) x[k] = 0.f;
    for (int i = warp; i <= it.w; i += 8) {
      const float* const p = part(i);
      const float m = p[a.head], f = m == -INFINITY ? 0.f : ex2(m - top);
      float y[kMaxHead / 32];
#pragma unroll
      for (uint32_t k = 0; k < kMaxHead / 32; ++k) y[k] = k * 32 + lane < a.head ? p[k * 32 + lane] : 0.f;
      sum += f * p[a.head + 1];
#pragma unroll
      for (uint32_t k = 0; k < kMaxHead / 32; ++k) x[k] += f == 0.f ? 0.f : f * y[k];  // (no weight, whatever it holds)
    }
#pragma unroll
    for (uint32_t k = 0; k < kMaxHead / 32; ++k) sums[warp][k * 32 + lane] = x[k];
    if (lane == 0) sums[warp][kMaxHead] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < 8; ++w) sum += sums[w][kMaxHead];
    const uint32_t query = a.each_div.div(row0 + r), h = it.y * a.each + row0 + r - query * a.each, e = threadIdx.x;
    const int64_t t = s.first + query;
    if (e < a.head) {
      float y = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < 8; ++w) y += sums[w][e];
      store_real(a.out, a.type, t * a.ot + h * a.oh + e, sum == 0.f ? 0.f : y / sum);
    }
    if (a.lse && e == 0) a.lse[t * a.lt + h * a.lh] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.69314718056f;
    __syncthreads();
  }
}

template <int F, int DT, int NT, bool GEN>
void start(const Args& a, cudaStream_t stream) {
  using L = Layout<DT, NT, GEN>;
  void (*const kernel)(const Args) = gpuos_attend_kernel<F, DT, NT, GEN>;
  static SharedMemory room;
  room.grant(reinterpret_cast<const void*>(kernel), L::total);
  run(kernel, dim3(a.grid), kThreads, L::total, stream, a);
  if (!a.split) return;
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(a.grid, 8);
  c.blockDim = dim3(256);
  c.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  c.attrs = at;
  c.numAttrs = 1;
  cuda_ok(cudaLaunchKernelEx(&c, gpuos_attend_join_kernel<L::rows>, a), "launch");
}

template <int F, int DT>
void start(const Plan& p, const Args& a, cudaStream_t stream) {
  if (p.general) start<F, DT, 2, true>(a, stream);
  else if (p.tiles == 1) start<F, DT, 1, false>(a, stream);
  else start<F, DT, DT == 256 ? 2 : 4, false>(a, stream);
}

}  // namespace

template <int F>
void launch(const Plan& p, const Args& a, cudaStream_t stream) {
  if (p.padded == 64) start<F, 64>(p, a, stream);
  else if (p.padded == 128) start<F, 128>(p, a, stream);
  else start<F, 256>(p, a, stream);
}

}  // namespace attend
}  // namespace rowops
}  // namespace gpuos
