// gpuos_attend: checks, and the choice of a kernel.  The kernels are in attend.cuh
// (attend_int8.cu and attend_e4m3.cu compile them).
#include "attend.h"

using namespace gpuos::rowops;
using namespace gpuos::rowops::attend;

namespace {

constexpr int64_t kMostPositions = 1ll << 31;

// What a call's launch and its workspace follow from.
struct Shape {
  Plan plan;
  uint32_t grid;
  bool join;  // whether an item may be split
  int64_t bytes;
};

Shape shape(int64_t sequences, int64_t longest, int64_t q_heads, int64_t k_heads, int64_t head, int64_t groups, int32_t type,
            int64_t capacity) {
  Shape s;
  const int64_t each = q_heads / k_heads;
  s.plan = plan((uint32_t)head, (uint32_t)groups, type != GPUOS_BF16, longest * each);
  const int64_t rows = 8 * s.plan.tiles;
  const int64_t blocks = (longest * each + rows - 1) / rows, units = std::max<int64_t>((capacity + kUnit - 1) / kUnit, 1);
  // (as 64-bit products: at most 2^31 of each)
  const double most = (double)sequences * (double)k_heads * (double)std::max<int64_t>(blocks, 1) * (double)units;
  s.grid = (uint32_t)std::max(std::min(most, (double)sm_count() * s.plan.per_sm), 1.0);  // (tokens of no sequence are written too)
  s.join = units > kWhole;
  s.bytes = s.join ? (int64_t)s.grid * (16 + 2 * rows * (head + 2) * 4) : 0;
  return s;
}

void check_held(const gpuos_tensor& c, const gpuos_tensor& s, const char* name) {
  check_tensor(&c, 4, name);
  check_tensor(&s, 4, "scales");
  need(c.dtype == GPUOS_I8 || c.dtype == GPUOS_E4M3, "codes must be int8 or float8_e4m3fn (a 4-bit cache is read with cache_read)");
  need(s.dtype == GPUOS_F32, "scales must be float32");
  for (int d = 0; d < 3; ++d) need(c.sizes[d] == s.sizes[d], "codes and scales must have the same pages, rows and heads");
  need(c.sizes[3] <= 1 || c.strides[3] == 1, "codes: the last dim must be contiguous");
}

}  // namespace

extern "C" int32_t gpuos_attend_workspace(const gpuos_tensor* q, const gpuos_tensor* codes, const gpuos_tensor* scales,
                                          const gpuos_tensor* pages, int64_t longest, int64_t* bytes) {
  return entry("gpuos_attend_workspace", [&] {
    need(q && codes && scales && pages && bytes, "an argument is NULL");
    need(q->ndim == 3 && codes->ndim == 4 && scales->ndim == 4 && pages->ndim == 2, "q must have 3 dims, codes and scales 4, pages 2");
    const int64_t hk = codes->sizes[2], page = codes->sizes[1];
    need(hk >= 1 && q->sizes[1] >= hk && q->sizes[1] % hk == 0, "the query heads must be a multiple of the cache's");
    need(page >= 0 && page < kMostPositions && pages->sizes[1] >= 0 && pages->sizes[1] < kMostPositions && page * pages->sizes[1] < kMostPositions,
         "a sequence has fewer than 2^31 positions");
    need(longest >= 1 && longest < kMostPositions, "longest must be at least 1");
    const int64_t most = std::min(longest, std::max<int64_t>(q->sizes[0], 1));
    *bytes = shape(pages->sizes[0], most, q->sizes[1], hk, q->sizes[2], scales->sizes[3], q->dtype, page * pages->sizes[1]).bytes;
  });
}

extern "C" int32_t gpuos_attend(const gpuos_tensor* q, const gpuos_tensor* codes, const gpuos_tensor* scales,
                                const gpuos_tensor* pages, const gpuos_tensor* lengths, const gpuos_tensor* offsets,
                                const gpuos_tensor* out, const gpuos_tensor* lse, void* workspace, int64_t workspace_bytes,
                                int64_t longest, int64_t window, float scale, int32_t flags, void* stream) {
  return entry("gpuos_attend", [&] {
    check_tensor(q, 3, "q");
    need(is_real(q->dtype), "q must be float32, float16 or bfloat16");
    need(codes && scales, "codes and scales are needed");
    check_held(codes[0], scales[0], "codes");
    check_held(codes[1], scales[1], "codes");
    need(codes[0].dtype == codes[1].dtype, "keys and values must have one format");
    same_sizes(codes[0], codes[1], "keys and values must have the same sizes");
    same_sizes(scales[0], scales[1], "keys and values must have the same scales");
    const int64_t pool = codes->sizes[0], page = codes->sizes[1], hk = codes->sizes[2], head = codes->sizes[3];
    const int64_t groups = scales->sizes[3], hq = q->sizes[1];
    need(head >= 16 && head <= kMaxHead && head % 16 == 0, "the head size must be a multiple of 16, at most 256");
    need(q->sizes[2] == head, "q and the cache must have one head size");
    need(groups >= 1 && head % groups == 0 && (groups == 1 || head / groups % 32 == 0),
         "a scale must cover the head, or a multiple of 32 elements");
    need(hk >= 1 && hq >= hk && hq % hk == 0, "the query heads must be a multiple of the cache's");
    need(q->strides[2] == 1, "q: the last dim must be contiguous");
    check_tensor(pages, 2, "pages");
    check_tensor(lengths, 1, "lengths");
    need(is_index(pages->dtype) && is_index(lengths->dtype), "pages and lengths must be int32 or int64");
    const int64_t n = pages->sizes[0], tokens = q->sizes[0];
    need(lengths->sizes[0] == n, "lengths must have one element for each row of pages");
    need(page >= 1, "pages must have rows");
    need(page < kMostPositions && pages->sizes[1] < kMostPositions && page * pages->sizes[1] < kMostPositions,
         "a sequence has fewer than 2^31 positions");
    need(pool < kMostPositions && n < (1ll << 30) && tokens < kMostPositions / hq, "the call is too large");
    if (offsets) {
      check_tensor(offsets, 1, "offsets");
      need(is_index(offsets->dtype), "offsets must be int32 or int64");
      need(offsets->sizes[0] == n + 1, "offsets must have one element more than there are sequences");
    } else {
      need(tokens == n, "without offsets each sequence has one query");
    }
    need(longest >= 1 && longest < kMostPositions, "longest must be at least 1");
    need(window >= 0, "window must not be negative");
    need((flags & ~GPUOS_ATTEND_CAUSAL) == 0, "unknown flag");
    const bool causal = flags & GPUOS_ATTEND_CAUSAL;
    need(causal || window == 0, "a window needs causal order");
    need(scale <= 2e38f && scale >= -2e38f, "scale must be in [-2e38, 2e38]");  // (times log2(e) it stays a 32-bit number)
    check_tensor(out, 3, "out");
    need(out->dtype == q->dtype, "q and out must have one dtype");
    same_sizes(*out, *q, "out must have the sizes of q");
    need(out->strides[2] == 1, "out: the last dim must be contiguous");
    check_output(*out, "out");
    if (lse) {
      check_tensor(lse, 2, "lse");
      need(lse->dtype == GPUOS_F32, "lse must be float32");
      need(lse->sizes[0] == tokens && lse->sizes[1] == hq, "lse must be (token, query head)");
      check_output(*lse, "lse");
    }
    const gpuos_tensor* in[8] = {q, codes, codes + 1, scales, scales + 1, pages, lengths, offsets};
    for (const gpuos_tensor* o : {out, lse})
      for (const gpuos_tensor* i : in)
        if (o && i) no_overlap(*o, *i, "an output must not overlap an input");
    if (lse) no_overlap(*out, *lse, "outputs overlap");
    if (tokens == 0) return;

    const int64_t capacity = page * pages->sizes[1];
    const Shape s = shape(n, std::min(longest, tokens), hq, hk, head, groups, q->dtype, capacity);
    need(s.bytes == 0 || (workspace && workspace_bytes >= s.bytes), "the workspace is too small: gpuos_attend_workspace says how large");
    need(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be aligned to 16 bytes");
    Args a{};
    a.q = q->data;
    a.qt = q->strides[0];
    a.qh = q->strides[1];
    a.out = out->data;
    a.ot = out->strides[0];
    a.oh = out->strides[1];
    if (lse) {
      a.lse = static_cast<float*>(lse->data);
      a.lt = lse->strides[0];
      a.lh = lse->strides[1];
    }
    a.vec = 16;
    for (int i = 0; i < 2; ++i) {
      Held& h = i ? a.v : a.k;
      h.codes = static_cast<const uint8_t*>(codes[i].data);
      h.cp = codes[i].strides[0];
      h.cr = codes[i].strides[1];
      h.ch = codes[i].strides[2];
      h.scales = static_cast<const float*>(scales[i].data);
      h.sp = scales[i].strides[0];
      h.sr = scales[i].strides[1];
      h.sh = scales[i].strides[2];
      h.sg = scales[i].strides[3];
      while (a.vec > 1 && !rows_aligned(codes[i], a.vec)) a.vec = a.vec == 16 ? 4 : 1;
    }
    a.alike = 1;
    for (int d = 0; d < 3; ++d) a.alike &= codes[0].strides[d] == codes[1].strides[d] && scales[0].strides[d] == scales[1].strides[d];
    a.pages = pages->data;
    a.ps = pages->strides[0];
    a.pp = pages->strides[1];
    a.lengths = lengths->data;
    a.ls = lengths->strides[0];
    if (offsets) {
      a.offsets = offsets->data;
      a.os = offsets->strides[0];
    }
    a.pool = pool;
    a.capacity = capacity;
    a.tokens = (uint32_t)tokens;
    a.sequences = (uint32_t)n;
    a.k_heads = (uint32_t)hk;
    a.each = (uint32_t)(hq / hk);
    a.head = (uint32_t)head;
    a.groups = (uint32_t)groups;
    a.group = (uint32_t)(head / groups);
    a.grid = s.grid;
    a.window = window;
    a.scale2 = (float)((double)scale * 1.44269504088896340736);
    a.page = FastDiv((uint32_t)page);
    a.each_div = FastDiv(a.each);
    a.causal = causal;
    a.type = q->dtype;
    a.page_wide = pages->dtype == GPUOS_I64;
    a.length_wide = lengths->dtype == GPUOS_I64;
    a.offset_wide = offsets && offsets->dtype == GPUOS_I64;
    a.split_q = q->dtype == GPUOS_F32;
    a.split_p = q->dtype != GPUOS_BF16;
    if (s.join) {
      a.split = static_cast<int4*>(workspace);
      a.partial = reinterpret_cast<float*>(a.split + s.grid);
    }
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool int8 = codes->dtype == GPUOS_I8;
    a.few = kAll;
    if (n && groups == 1 && q->dtype != GPUOS_F32 && s.plan.padded <= 128 && a.vec == 16 && std::min(longest, tokens) * a.each > kWideFrom) {
      a.few = kWideFrom;
      // blocks of all sequences with more rows than kWideFrom
      const int64_t most = std::min(tokens * a.each / kWideRows + n, tokens * a.each / kWideFrom) * hk;
      need(most < (1ll << 31), "the call is too large");
      a.wide_grid = (uint32_t)most;
      a.q_vec = rows_aligned(*q, 8);
      a.out_vec = rows_aligned(*out, 8);
      int8 ? launch_wide<kInt8>(a, st) : launch_wide<kE4M3>(a, st);
    }
    int8 ? launch<kInt8>(s.plan, a, st) : launch<kE4M3>(s.plan, a, st);
  });
}
