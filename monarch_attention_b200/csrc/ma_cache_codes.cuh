// Codes (e4m3) and scales of the paged cache.
#pragma once

#include <cuda_fp8.h>

#include "ma_cache.cuh"

namespace ma {

// The smallest n in [-40, 60] with amax <= 448 * 2^n, as 2^n: 448 = 1.75 * 2^8, so a mantissa above 1.75 takes one more.
__device__ __forceinline__ float scale_for(float amax) {
  const int n = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;
  return __uint_as_float((uint32_t)(min(max(n, -40), 60) + 127) << 23);
}

__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3) |
         (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3) << 16;
}
// Codes of a block whose scale has risen by 1 / ratio.
__device__ __forceinline__ uint32_t moved(uint32_t codes, float ratio) {
  const float2 lo = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)codes, __NV_E4M3)));
  const float2 hi = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(codes >> 16), __NV_E4M3)));
  return four_codes(lo.x * ratio, lo.y * ratio, hi.x * ratio, hi.y * ratio);
}

}  // namespace ma
