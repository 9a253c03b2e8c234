// fp8.cuh -- element conversions shared by the 8-bit quantiser and the norms.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace st {

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }

__device__ __forceinline__ void from_float(float v, float &out) { out = v; }
__device__ __forceinline__ void from_float(float v, __half &out) { out = __float2half_rn(v); }
__device__ __forceinline__ void from_float(float v, __nv_bfloat16 &out) { out = __float2bfloat16_rn(v); }

__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Four values as 8-bit codes in one word, the first in the low byte (round to
// nearest even, saturating; NaN stays NaN).
__device__ __forceinline__ uint32_t to_fp8x4(float a, float b, float c, float d, bool e5m2) {
    const __nv_fp8_interpretation_t kind = e5m2 ? __NV_E5M2 : __NV_E4M3;
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, kind);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, kind);
    return lo | (hi << 16);
}

// The scale of a block whose largest |value| has the bit pattern `bits`, and
// its reciprocal: see quantize.cu.
constexpr float kFp8LeastScale = 1.1754943508222875e-38f;  // 2^-126
__device__ __forceinline__ float fp8_scale(uint32_t bits, float limit) {
    const uint32_t s = __float_as_uint(__fdiv_rn(__uint_as_float(bits), limit));
    return __uint_as_float(max(s, __float_as_uint(kFp8LeastScale)));
}

}  // namespace st
