// 8-bit values (e4m3: 4 bits of exponent, 3 of mantissa, largest value 448) with a scale per group of 128: the rules that the
// kernels which make them share.
//
// A group's scale is the smallest power of two that brings its largest magnitude to 448 = 1.75 * 2^8 or less, 2^-126 at least,
// and 1 for a group of zeros.  x / scale is then exact (or far below the smallest 8-bit value), so that the only rounding is the
// one to 3 bits of mantissa, to nearest, the even one of two: half a step, 2^-4 of the value.  A group that holds an infinity or
// a NaN has the scale NaN and the values 0: whatever is computed from it is NaN.
#pragma once
#include <cuda_fp8.h>

#include "common.cuh"

namespace tllm {

constexpr int FP8_GROUP = 128;
constexpr int FP8_MOST = 0x7FFFFFFF - 4095;    // rows or values of a row: the kernels round them up to whole tiles, runs and groups in 32 bits

// The scale's biased exponent (what e8m0 holds; 255 is NaN) from the bits of the largest magnitude (maximum as integers, which
// puts NaN above infinity above the finite values).
__device__ __forceinline__ uint32_t fp8_scale_byte(uint32_t largest) {
  if (largest >= 0x7F800000u) return 255u;
  const int byte = (int)((largest + 0x1FFFFFu) >> 23) - 8;   // a mantissa above 1.75 carries into the exponent
  return largest == 0u ? 127u : (uint32_t)max(byte, 1);
}
// 1 / scale (whatever for NaN: fp8_pack4 leaves zeros there)
__device__ __forceinline__ float fp8_inverse_scale(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// The scale an e8m0 byte stands for: 2^(byte - 127), 255 NaN.
__device__ __forceinline__ float fp8_scale(uint32_t byte) {
  return byte == 255u ? __uint_as_float(0x7FC00000u) : byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}
__device__ __forceinline__ uint32_t fp8_abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// four values over the scale 2^(byte - 127) as four e4m3 bytes, the first in the lowest; zeros where the scale is NaN
__device__ __forceinline__ uint32_t fp8_pack4(float a, float b, float c, float d, float inverse, uint32_t byte) {
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a * inverse, b * inverse), __NV_SATFINITE, __NV_E4M3);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c * inverse, d * inverse), __NV_SATFINITE, __NV_E4M3);
  return byte == 255u ? 0u : __byte_perm(lo, hi, 0x5410);
}

}  // namespace tllm
