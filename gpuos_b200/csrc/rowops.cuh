// Device helpers of the row operators: vector loads and stores of 32- and
// 16-bit elements, division by a launch constant, packed 32-bit arithmetic.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>
#include <type_traits>

#include "rowops.h"

namespace gpuos {
namespace rowops {

// One launch of a kernel that takes one parameter block.
template <typename A>
inline void run(void (*kernel)(A), dim3 grid, unsigned threads, size_t smem, cudaStream_t stream,
                const std::remove_const_t<A>& args) {
  void* p[1] = {const_cast<std::remove_const_t<A>*>(&args)};
  cuda_ok(cudaLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3(threads), p, smem, stream), "launch");
}

// n / d for n < 2^31 by one multiplication: with s = ceil(log2 d) and
// m = ceil(2^(32+s-1) / d) the error of n * m / 2^(32+s-1) stays below 1 / d.
struct FastDiv {
  uint32_t d = 1, m = 0, s = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    if (d <= 1) return;
    while ((1ull << s) < d) ++s;
    m = (uint32_t)(((1ull << (32 + s - 1)) + d - 1) / d);
  }
  __device__ __forceinline__ uint32_t div(uint32_t n) const {
    return d <= 1 ? n : __umulhi(n, m) >> (s - 1);
  }
};

template <typename T> __device__ __forceinline__ float to_f(T x);
template <> __device__ __forceinline__ float to_f<float>(float x) { return x; }
template <> __device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// N elements of T moved by one access (N * sizeof(T) is 1, 2, 4, 8 or 16).
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// STREAM marks data that is not read again.
template <typename T, int N, bool STREAM = true>
__device__ __forceinline__ Pack<T, N> load_pack(const T* p) {
  Pack<T, N> r;
  constexpr int B = sizeof(T) * N;
  if constexpr (!STREAM) r = *reinterpret_cast<const Pack<T, N>*>(p);
  else if constexpr (B == 16) *reinterpret_cast<uint4*>(&r) = __ldcs(reinterpret_cast<const uint4*>(p));
  else if constexpr (B == 8) *reinterpret_cast<uint2*>(&r) = __ldcs(reinterpret_cast<const uint2*>(p));
  else if constexpr (B == 4) *reinterpret_cast<uint32_t*>(&r) = __ldcs(reinterpret_cast<const uint32_t*>(p));
  else if constexpr (B == 2) *reinterpret_cast<uint16_t*>(&r) = __ldcs(reinterpret_cast<const unsigned short*>(p));
  else r = *reinterpret_cast<const Pack<T, N>*>(p);
  return r;
}

template <typename T, int N>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, N>& r) {
  *reinterpret_cast<Pack<T, N>*>(p) = r;
}

// Two 32-bit products or sums in one instruction, each rounded on its own.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r)
      : "l"(*reinterpret_cast<unsigned long long*>(&a)), "l"(*reinterpret_cast<unsigned long long*>(&b)),
        "l"(*reinterpret_cast<unsigned long long*>(&c)));
  return *reinterpret_cast<float2*>(&r);
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// `n` of the index tensor, 32 or 64 bit.
__device__ __forceinline__ int64_t load_index(const void* p, bool wide, int64_t n) {
  return wide ? __ldg(static_cast<const long long*>(p) + n) : (int64_t)__ldg(static_cast<const int*>(p) + n);
}

}  // namespace rowops
}  // namespace gpuos
