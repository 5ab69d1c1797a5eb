// Shared by the paged-serving kernels: division by the page size, and fp32
// arithmetic on pairs.
#pragma once
#include "mt_common.cuh"

namespace mt {

// n / d for 0 <= n < 2^31 by one multiplication: with s = 31 + ceil(log2 d) and
// m = ceil(2^s / d) < 2^32, m d exceeds 2^s by less than 2^(s - 31), so
// floor(n m / 2^s) = floor(n / d) for every such n.
struct FastDiv {
  uint32_t mul;
  int shift, d;
  static FastDiv of(int d) {
    int c = 0;
    while ((1ll << c) < d) ++c;
    return {static_cast<uint32_t>(((1ull << (31 + c)) + d - 1) / d), 31 + c, d};
  }
  __device__ __forceinline__ int div(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
  }
};

// two fp32 operations in one instruction
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace mt
