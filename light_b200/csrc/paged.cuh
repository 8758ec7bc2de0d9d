// What the kernels over a paged key-value cache share: element access at three types, division by a page size, bits of the status word.
#pragma once
#include "common.cuh"
#include "mma_sync.cuh"
#include "umma.cuh"

namespace lb {

enum { PAGED_LENGTH = 1, PAGED_PAGE = 2, PAGED_SLOT = 4, PAGED_REFUSED = 8 };  // light_b200_paged_status

namespace {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// two f32 in a 64-bit register
__device__ __forceinline__ uint64_t two(float a, float b) { return (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a); }
__device__ __forceinline__ float lo(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float hi(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// n / d for 0 <= n < 2^31: n m >> (31 + s) with 2^s >= d and m = ceil(2^(31 + s) / d).  m d exceeds 2^(31 + s) by less than d <= 2^s, so the
// product's excess stays under 2^(31 + s).  (2 n has 32 bits: the upper half of 2 n m is n m >> 31.)
struct FastDiv {
  uint32_t m = 0;
  int s = 0, d = 1;
  FastDiv() = default;
  explicit FastDiv(int d_) : d(d_) {
    while ((1ll << s) < d) s++;
    m = (uint32_t)(((1ull << (31 + s)) + (unsigned)d - 1) / (unsigned)d);
  }
  __device__ __forceinline__ int div(int n) const { return (int)(__umulhi((unsigned)n << 1, m) >> s); }
};

// The word as it was, and 0 in its place, in one: what a launch adds meanwhile is in this answer or the next.
__device__ unsigned int g_taken;
__global__ void take_status_kernel(unsigned int *word) { g_taken = atomicExch(word, 0u); }
inline int taken_status(const unsigned int &symbol, unsigned int *bits) {
  static std::mutex one;  // (g_taken is one word)
  std::lock_guard<std::mutex> lk(one);
  void *word = nullptr;
  cudaError_t e = cudaGetSymbolAddress(&word, symbol);
  if (e == cudaSuccess) {
    take_status_kernel<<<1, 1>>>(static_cast<unsigned int *>(word));
    e = cudaGetLastError();
  }
  return (int)(e != cudaSuccess ? e : cudaMemcpyFromSymbol(bits, g_taken, sizeof(*bits)));
}

}  // namespace
}  // namespace lb
