// Device helpers shared by the paged cache's kernels.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace mlxvs_b200 {

// Division of 0 <= x < 2^31 by a launch constant: one high multiplication.
// mul = ceil(2^(32 + shift) / d) with 2^shift < d <= 2^(shift + 1) fits 33
// bits; its low 32 are kept and x is added back (the method of Granlund and
// Montgomery, 1994).
struct FastDiv {
  uint32_t d = 1, mul = 0, shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    while ((1ull << (shift + 1)) < d) ++shift;
    if (d > 1) mul = (uint32_t)(((1ull << 32) * ((1ull << (shift + 1)) - d)) / d + 1);
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t x) const {
    if (d == 1) return x;
    const uint32_t hi = (uint32_t)(((uint64_t)x * mul) >> 32);
    return (hi + ((x - hi) >> 1)) >> shift;
  }
};

// Element types of queries and caches.
template <class T>
__device__ __forceinline__ float to_float(T x) {
  return static_cast<float>(x);
}

// x rounded to T, to nearest even.
template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ __nv_bfloat16 from_float(float x) {
  return __float2bfloat16_rn(x);
}
template <>
__device__ __forceinline__ __half from_float(float x) {
  return __float2half_rn(x);
}

// The exponent e of an 8-bit code x * 2^e for values of at most `top` in
// magnitude: top * 2^e lies in [64, 128).  Kept within +-100 so that 2^e and
// 2^-e are ordinary floats; zero, subnormal and infinite tops end there.
__device__ __forceinline__ int code_exponent(float top) {
  const int floor_log2 = (int)((__float_as_uint(top) >> 23) & 255u) - 127;
  return max(-100, min(100, 6 - floor_log2));
}

// The same for queries that go to the tensor cores as float16: kept within +-126,
// the widest that leaves 2^e and 2^-e ordinary floats, so that neither the
// largest bfloat16 queries overflow nor the smallest vanish.
__device__ __forceinline__ int query_exponent(float top) {
  const int floor_log2 = (int)((__float_as_uint(top) >> 23) & 255u) - 127;
  return max(-126, min(126, 6 - floor_log2));
}

__device__ __forceinline__ float exp2_int(int e) {
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

}  // namespace mlxvs_b200
