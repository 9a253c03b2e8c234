// fp8.cuh -- element conversions and packed fp32 arithmetic shared by the
// 8-bit quantiser, the 8-bit matmul and the norms.
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

// ---- pairs of fp32 in one register pair: the packed instructions halve the
// issue slots of the row kernels, which were bound by them
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    return static_cast<uint64_t>(__float_as_uint(a)) | (static_cast<uint64_t>(__float_as_uint(b)) << 32);
}
__device__ __forceinline__ float lo2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float hi2(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}

// max(|m|, |a|, |b|); a NaN wins
__device__ __forceinline__ float max_abs(float m, float a, float b) {
    float r;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(m), "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float max_abs(float a, float b) { return max_abs(a, b, b); }

// Eight elements in 16-byte words to four pairs and back.
__device__ __forceinline__ void unpack8(const uint4 (&w)[1], uint64_t (&f)[4], __nv_bfloat16) {
    const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = static_cast<uint64_t>(u[j] << 16) | (static_cast<uint64_t>(u[j] & 0xffff0000u) << 32);
}
__device__ __forceinline__ void unpack8(const uint4 (&w)[1], uint64_t (&f)[4], __half) {
    const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2 *>(&u[j]));
        f[j] = pack2(v.x, v.y);
    }
}
__device__ __forceinline__ void unpack8(const uint4 (&w)[2], uint64_t (&f)[4], float) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        f[2 * j] = static_cast<uint64_t>(w[j].x) | (static_cast<uint64_t>(w[j].y) << 32);
        f[2 * j + 1] = static_cast<uint64_t>(w[j].z) | (static_cast<uint64_t>(w[j].w) << 32);
    }
}
__device__ __forceinline__ void pack8(const uint64_t (&f)[4], uint4 (&w)[1], __nv_bfloat16) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo2(f[j]), hi2(f[j]));
        u[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
    w[0] = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void pack8(const uint64_t (&f)[4], uint4 (&w)[1], __half) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const __half2 h = __floats2half2_rn(lo2(f[j]), hi2(f[j]));
        u[j] = *reinterpret_cast<const uint32_t *>(&h);
    }
    w[0] = make_uint4(u[0], u[1], u[2], u[3]);
}
__device__ __forceinline__ void pack8(const uint64_t (&f)[4], uint4 (&w)[2], float) {
#pragma unroll
    for (int j = 0; j < 2; ++j)
        w[j] = make_uint4(static_cast<uint32_t>(f[2 * j]), static_cast<uint32_t>(f[2 * j] >> 32),
                          static_cast<uint32_t>(f[2 * j + 1]), static_cast<uint32_t>(f[2 * j + 1] >> 32));
}

// Four values as 8-bit codes in one word, the first in the low byte (round to
// nearest even, saturating; NaN stays NaN).
template <bool E5M2>
__device__ __forceinline__ uint32_t to_fp8x4(float a, float b, float c, float d) {
    constexpr __nv_fp8_interpretation_t kind = E5M2 ? __NV_E5M2 : __NV_E4M3;
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, kind);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, kind);
    return lo | (hi << 16);
}
__device__ __forceinline__ uint32_t to_fp8x4(float a, float b, float c, float d, bool e5m2) {
    return e5m2 ? to_fp8x4<true>(a, b, c, d) : to_fp8x4<false>(a, b, c, d);
}
// The codes of four pairs times `scale`.
template <bool E5M2>
__device__ __forceinline__ uint2 to_fp8x8(const uint64_t (&f)[4], float scale) {
    const uint64_t s = pack2(scale, scale);
    const uint64_t y[4] = {mul2(f[0], s), mul2(f[1], s), mul2(f[2], s), mul2(f[3], s)};
    return make_uint2(to_fp8x4<E5M2>(lo2(y[0]), hi2(y[0]), lo2(y[1]), hi2(y[1])),
                      to_fp8x4<E5M2>(lo2(y[2]), hi2(y[2]), lo2(y[3]), hi2(y[3])));
}

// Maxima of four blocks that 16 lanes hold each: every exchange halves the
// blocks that a lane still carries, so a lane ends with the maximum of block
// (lane >> 2) & 3 of its half warp, after 5 shuffles for the 16 of four
// separate reductions.
__device__ __forceinline__ float max_of_four(const float (&m)[4], int lane) {
    const bool up = lane & 8, odd = lane & 4;
    float k0 = up ? m[2] : m[0], k1 = up ? m[3] : m[1];
    k0 = max_abs(k0, __shfl_xor_sync(0xffffffffu, up ? m[0] : m[2], 8));
    k1 = max_abs(k1, __shfl_xor_sync(0xffffffffu, up ? m[1] : m[3], 8));
    float k = max_abs(odd ? k1 : k0, __shfl_xor_sync(0xffffffffu, odd ? k0 : k1, 4));
    k = max_abs(k, __shfl_xor_sync(0xffffffffu, k, 2));
    return max_abs(k, __shfl_xor_sync(0xffffffffu, k, 1));
}

// The scale of a block from its largest |value|, a NaN kept: see quantize.cu.
constexpr float kFp8LeastScale = 1.1754943508222875e-38f;  // 2^-126
__device__ __forceinline__ float fp8_scale(float top, float limit) {
    return max_abs(__fdiv_rn(top, limit), kFp8LeastScale);
}

}  // namespace st
