// e4m3 with power-of-two scales: what the kernels that quantise share.
#pragma once
#include "sm100.cuh"
#include <cuda_fp8.h>

namespace mbf8 {

constexpr uint32_t INF16 = 0x7f80u, INF32 = 0x7f800000u;

__device__ __forceinline__ float pow2(int k) { return __uint_as_float(static_cast<uint32_t>(k + 127) << 23); }
// smallest k in [k_min, 120] with amax <= 448 * 2^k = 1.75 * 2^(k + 8)
__device__ __forceinline__ int block_exponent(uint32_t amax_bits, int k_min = -117) {
  const int e = static_cast<int>(amax_bits >> 23) - 127;                       // amax in [2^e, 2^(e+1)), or below 2^-126
  const int k = (amax_bits & 0x7fffffu) <= 0x600000u ? e - 8 : e - 7;
  return min(max(k, k_min), 120);
}
// e4m3 codes of two values (x in the low byte); NaN gives the NaN code
__device__ __forceinline__ uint32_t encode2(float2 v) {
  return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(v, __NV_SATFINITE, __NV_E4M3));
}
// where the exponent byte of row r (of a 128-row tile) and block b (of a group of 4) lies among 512
__device__ __forceinline__ int scale_at(int r, int b) { return (r & 31) * 16 + (r >> 5) * 4 + b; }

}  // namespace mbf8
