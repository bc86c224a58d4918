// What the row operators' entry points share: argument checks, errors and
// launch set-up.  The operators (rotary.cu, cache.cu, route.cu, logprobs.cu)
// run at once on the caller's stream, as gpuos_reduce_rows_noalloc does: they
// allocate nothing, keep nothing between calls and need no executor.
#pragma once
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <exception>
#include <mutex>
#include <string>

#include "../../include/gpuos_b200.h"

namespace gpuos {
void set_last_error(const char* msg);  // runtime.cpp: message for gpuos_last_error()

namespace rowops {

struct Fail {
  int32_t code;
  std::string msg;
};

[[noreturn]] inline void invalid(const std::string& msg) { throw Fail{GPUOS_EINVAL, msg}; }

inline void need(bool ok, const char* msg) {
  if (!ok) invalid(msg);
}

inline void cuda_ok(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return;
  cudaGetLastError();  // reported here, not by a later check
  throw Fail{GPUOS_ECUDA, std::string(what) + ": " + cudaGetErrorString(e)};
}

// Runs an entry point's body; nothing is thrown past the C boundary.
template <typename F>
int32_t entry(const char* name, F&& body) noexcept {
  try {
    try {
      body();
      return GPUOS_OK;
    } catch (const Fail& f) {
      set_last_error((std::string(name) + ": " + f.msg).c_str());
      return f.code;
    } catch (const std::exception& e) {
      set_last_error((std::string(name) + ": " + e.what()).c_str());
      return GPUOS_EINVAL;
    }
  } catch (...) {  // no memory for the message
    return GPUOS_EINVAL;
  }
}

inline int esize(int32_t dt) {
  switch (dt) {
    case GPUOS_F64: case GPUOS_I64: return 8;
    case GPUOS_F32: case GPUOS_I32: return 4;
    case GPUOS_F16: case GPUOS_BF16: return 2;
    default: return 1;
  }
}

inline bool is_real(int32_t dt) { return dt == GPUOS_F32 || dt == GPUOS_F16 || dt == GPUOS_BF16; }
inline bool is_index(int32_t dt) { return dt == GPUOS_I32 || dt == GPUOS_I64; }

inline int64_t numel(const gpuos_tensor& t) {
  int64_t n = 1;
  for (int d = 0; d < t.ndim; ++d) n *= t.sizes[d];
  return n;
}

// Shape checks every tensor argument gets: dims, sizes whose product and byte
// extent stay within 62 bits, a data pointer where there are elements,
// aligned to its elements.
inline void check_tensor(const gpuos_tensor* t, int ndim, const char* name) {
  if (!t) invalid(std::string(name) + " is NULL");
  if (t->ndim != ndim)
    invalid(std::string(name) + " must have " + std::to_string(ndim) + " dims, not " + std::to_string(t->ndim));
  __int128 n = 1, ext = 0;
  for (int d = 0; d < ndim; ++d) {
    if (t->sizes[d] < 0) invalid(std::string(name) + " has a negative size");
    n *= t->sizes[d];
    if (n > ((__int128)1 << 62)) invalid(std::string(name) + " is too large");
  }
  if (n == 0) return;
  for (int d = 0; d < ndim; ++d) {
    if (t->strides[d] < 0) invalid(std::string(name) + " has a negative stride");
    ext += (__int128)(t->sizes[d] - 1) * t->strides[d];
  }
  if (ext * esize(t->dtype) > ((__int128)1 << 62)) invalid(std::string(name) + " is too large");
  if (!t->data) invalid(std::string(name) + " has no data pointer");
  if (reinterpret_cast<uintptr_t>(t->data) % esize(t->dtype))
    invalid(std::string(name) + " is not aligned to its elements");
}

// The bytes [lo, hi) a tensor covers (strides are not negative).
struct Span {
  uint64_t lo = 0, hi = 0;
};

inline Span span(const gpuos_tensor& t) {
  if (numel(t) == 0) return Span{};
  int64_t n = 0;
  for (int d = 0; d < t.ndim; ++d) n += (t.sizes[d] - 1) * t.strides[d];
  const uint64_t lo = reinterpret_cast<uint64_t>(t.data);
  return Span{lo, lo + (uint64_t)(n + 1) * esize(t.dtype)};
}

// Whether two tensors may share memory.  Tensors whose spans are apart do not;
// nor do slices of one buffer (queries and keys side by side in each token's
// row) whose elements stay apart modulo a stride that they share: with every
// stride of both either a multiple of S or part of an extent below S, the
// first covers [0, ea) and the second [at, at + eb) of every period of S bytes.
inline bool overlap(const gpuos_tensor& a, const gpuos_tensor& b) {
  const Span x = span(a), y = span(b);
  if (x.lo >= y.hi || y.lo >= x.hi) return false;
  const gpuos_tensor* both[2] = {&a, &b};
  for (const gpuos_tensor* t : both) {
    for (int c = 0; c < t->ndim; ++c) {
      if (t->sizes[c] <= 1 || t->strides[c] == 0) continue;
      const int64_t S = t->strides[c] * esize(t->dtype);
      int64_t ext[2];
      for (int i = 0; i < 2; ++i) {
        ext[i] = esize(both[i]->dtype);
        for (int d = 0; d < both[i]->ndim; ++d) {
          const int64_t st = both[i]->strides[d] * esize(both[i]->dtype);
          if (both[i]->sizes[d] > 1 && st % S) ext[i] += (both[i]->sizes[d] - 1) * st;
        }
      }
      const int64_t at = (int64_t)((y.lo >= x.lo ? (y.lo - x.lo) % (uint64_t)S
                                                 : (S - (int64_t)((x.lo - y.lo) % (uint64_t)S)) % S));
      if (at >= ext[0] && at + ext[1] <= S) return false;
    }
  }
  return true;
}

inline bool same_view(const gpuos_tensor& a, const gpuos_tensor& b) {
  if (a.data != b.data || a.dtype != b.dtype || a.ndim != b.ndim) return false;
  for (int d = 0; d < a.ndim; ++d)
    if (a.sizes[d] != b.sizes[d] || (a.sizes[d] > 1 && a.strides[d] != b.strides[d])) return false;
  return true;
}

inline void same_sizes(const gpuos_tensor& a, const gpuos_tensor& b, const char* what) {
  bool same = a.ndim == b.ndim;
  for (int d = 0; same && d < a.ndim; ++d) same = a.sizes[d] == b.sizes[d];
  if (!same) invalid(what);
}

// An output whose elements share memory with one another would be written
// twice: going from the smallest stride up, each must step past what the dims
// before it cover.
inline void check_output(const gpuos_tensor& t, const char* name) {
  int order[8], n = 0;
  for (int d = 0; d < t.ndim; ++d) {
    if (t.sizes[d] == 0) return;
    if (t.sizes[d] > 1) order[n++] = d;
  }
  std::sort(order, order + n, [&](int a, int b) { return t.strides[a] < t.strides[b]; });
  int64_t covered = 0;
  for (int i = 0; i < n; ++i) {
    if (t.strides[order[i]] <= covered)
      invalid(std::string(name) + " must not overlap itself (an expanded output?)");
    covered += (t.sizes[order[i]] - 1) * t.strides[order[i]];
  }
}

inline void no_overlap(const gpuos_tensor& a, const gpuos_tensor& b, const char* what) {
  if (overlap(a, b)) invalid(what);
}

// Whether every element of the dims before the last starts on a multiple of
// `n` elements (and the pointer on that many bytes).
inline bool rows_aligned(const gpuos_tensor& t, int n) {
  if (reinterpret_cast<uintptr_t>(t.data) % ((size_t)n * esize(t.dtype))) return false;
  for (int d = 0; d + 1 < t.ndim; ++d)
    if (t.sizes[d] > 1 && t.strides[d] % n) return false;
  return true;
}

// Multiprocessors of the current device.
inline int sm_count() {
  static std::mutex mu;
  static int known[64];
  int dev = -1;
  cuda_ok(cudaGetDevice(&dev), "cudaGetDevice");
  if (dev < 0 || dev >= 64) invalid("device index out of range");
  std::lock_guard<std::mutex> lk(mu);
  if (!known[dev])
    cuda_ok(cudaDeviceGetAttribute(&known[dev], cudaDevAttrMultiProcessorCount, dev),
            "cudaDeviceGetAttribute");
  return known[dev];
}

// How tokens of `heads` rows of `units` groups are spread over CTAs: a thread
// belongs to one token and one group and walks over about 8 heads in steps of
// groups * split; with few tokens the heads are spread over more threads, then
// over more CTAs, so that their loads start at once on many SMs.  (Rotary positions of 8 tokens x 40 heads:
// 2.4 us, 16.4 with one thread for all heads; of 9001 tokens 35 and 49; a cache's read of 64 tokens 1.8
// and 2.5.)
struct Spread {
  uint32_t lanes;   // threads side by side over a head's groups
  uint32_t groups;  // heads a CTA takes at once
  uint32_t tile;    // tokens a CTA takes
  uint32_t tiles;   // CTAs over the tokens
  uint32_t split;   // CTAs over the heads
};

inline Spread spread(uint32_t tokens, uint32_t units, uint32_t heads, uint32_t threads, uint32_t most_tile) {
  const uint32_t sms = (uint32_t)sm_count();
  Spread s;
  s.lanes = std::min(std::max(units, 1u), threads);
  s.groups = 1;
  while (s.lanes * s.groups * 2 <= threads && s.groups * 2 <= heads &&
         (s.groups * 16 <= heads || (uint64_t)tokens * s.lanes * s.groups < (uint64_t)threads * 4 * sms))
    s.groups *= 2;
  s.tile = std::min(threads / (s.lanes * s.groups), most_tile);
  s.tiles = (tokens + s.tile - 1) / s.tile;
  s.split = 1;
  while (s.tiles * s.split < sms && s.groups * s.split < heads) s.split *= 2;
  return s;
}

}  // namespace rowops
}  // namespace gpuos
