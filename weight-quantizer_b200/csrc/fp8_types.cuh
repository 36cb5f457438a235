// Element types of the 8-bit floating-point operators: 16- and 32-bit inputs
// and outputs, e4m3 codes, and the scale of a block of codes.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace wq {

template <typename T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Element i of an array of one of the three types (0 for a null array).
__device__ __forceinline__ float load_any(const void* p, int type, int64_t i) {
    if (p == nullptr) return 0.0f;
    if (type == kF16) return to_f32<__half>(static_cast<const __half*>(p)[i]);
    if (type == kBf16) return to_f32<__nv_bfloat16>(static_cast<const __nv_bfloat16*>(p)[i]);
    return static_cast<const float*>(p)[i];
}

// Two e4m3 codes (a in the low byte): nearest, ties to even. Codes have no
// infinity: an input that is not finite becomes the NaN code, so that an
// overflow upstream stays visible instead of reading as 448.
__device__ __forceinline__ uint32_t e4m3x2_finite(float a, float b) {
    return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
    a = fabsf(a) <= 3.402823466e38f ? a : __int_as_float(0x7fc00000);
    b = fabsf(b) <= 3.402823466e38f ? b : __int_as_float(0x7fc00000);
    return e4m3x2_finite(a, b);
}

// The values of two codes; every e4m3 value is exact in fp16.
__device__ __forceinline__ float2 e4m3x2_values(uint32_t w) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3);
    return __half22float2(__half2(h));
}

// Exponent k of a block's scale 2^k: the least k >= -117 with amax <= 448 * 2^k.
// 448 = 1.75 * 2^8, so k = e - 8 for amax = m * 2^e (1 <= m < 2) with m <= 1.75
// and e - 7 above; integer comparisons on the bits, nothing rounds. The floor
// keeps the least code times the scale (2^-9 * 2^-117) a normal bf16, so that
// code * scale is exact there; subnormal amax falls under it by itself. A
// block of zeros has the scale 1.
__device__ __forceinline__ int fp8_scale_exponent(float amax) {
    const uint32_t u = __float_as_uint(amax);
    if (u == 0u) return 0;
    const int e = (int)(u >> 23) - 127;
    const int k = e - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return k < -117 ? -117 : k;
}

}  // namespace wq
