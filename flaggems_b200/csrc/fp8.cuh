// 8-bit floating point cache types: conversions shared by the cache and attention kernels.
#pragma once
#include "common.cuh"

namespace fg {

// What the K/V rows of a cache are held in.
enum CacheKind : int { kCache16 = 0, kCacheE4M3 = 1, kCacheE5M2 = 2 };
inline bool is_fp8(int cache_dtype) { return cache_dtype == FG_E4M3 || cache_dtype == FG_E5M2; }

// Two 8-bit values (low byte first) as a pair of fp16.  Both types are subsets of fp16, so this is
// exact; NaN and (E5M2) infinities stay what they are.
template <int KIND>
__device__ __forceinline__ uint32_t fp8x2_to_f16x2(uint16_t v) {
  uint32_t r;
  if constexpr (KIND == kCacheE4M3)
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  else
    asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
// Four of them, packed in a word, as two pairs.
template <int KIND>
__device__ __forceinline__ void fp8x4_to_f16x4(uint32_t v, uint32_t& lo, uint32_t& hi) {
  lo = fp8x2_to_f16x2<KIND>((uint16_t)(v & 0xffffu));
  hi = fp8x2_to_f16x2<KIND>((uint16_t)(v >> 16));
}
// Two fp32 values rounded to nearest even; beyond the largest finite value (infinities too) they
// become that value, NaN stays NaN.
template <int KIND>
__device__ __forceinline__ uint16_t f32x2_to_fp8x2(float lo, float hi) {
  uint16_t r;
  if constexpr (KIND == kCacheE4M3)
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

// n / d for 32-bit n and a divisor fixed at launch: one high multiply and a shift.  With l = ceil(log2 d)
// and m = floor(2^32 (2^l - d) / d) + 1, n / d = (mulhi(n, m) + n) >> l in 33 bits (Granlund and
// Montgomery, 1994).
struct FastDiv {
  uint32_t d, m, l;
  FastDiv() : d(1), m(1), l(0) {}
  explicit FastDiv(uint32_t div) : d(div), l(0) {
    while (l < 32 && (1ull << l) < div) ++l;
    m = (uint32_t)((((1ull << l) - div) << 32) / div + 1);
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
#ifdef __CUDA_ARCH__
    const uint32_t t = __umulhi(n, m);
#else
    const uint32_t t = (uint32_t)(((uint64_t)n * m) >> 32);
#endif
    return (uint32_t)(((uint64_t)t + n) >> l);
  }
};

}  // namespace fg
