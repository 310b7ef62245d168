// Conversions of the 8-bit key/value cache's codes (see kv8.cu for its layout).
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

namespace msgl {

// two values to two e4m3 codes, nearest, ties to even (the first one in the low byte)
MSGL_DEVICE uint16_t kv8_e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// the two values of a pair of codes (the low 16 bits)
template <bool FP8>
MSGL_DEVICE float2 kv8_decode2(uint32_t pair) {
  if constexpr (FP8) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(pair & 0xffffu), __NV_E4M3);
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
  } else {
    return make_float2((float)(int8_t)(pair & 255u), (float)(int8_t)((pair >> 8) & 255u));
  }
}

}  // namespace msgl
