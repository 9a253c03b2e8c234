// quantize_fp4.cu -- 4-bit blocks (e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their
// negatives) as matmul_fp4 reads them, and back.
//
//   blocks of 16   t = least power of two >= 2^-126 with 2688 t >= max|a| of the tensor (or of a known maximum)
//                  s = e4m3(max|a| of the block / (6 t)),   q = e2m1(a / (s t)),   a ~ q s t
//   blocks of 32   s = least power of two >= 2^-127 with 6 s >= max|a| of the block (e8m0),   q = e2m1(a / s),   a ~ q s
//
// 2688 = 6 * 448: with t the largest block scale stays within e4m3.  t and
// the e8m0 scales are powers of two, so that a border between two codes,
// times the scale, is a number of a few bits: whether an element lies above
// it is decided exactly, and the codes are the same on any machine that
// rounds the quotients correctly.  A block with a NaN or an infinity gets the
// scale NaN, and what is computed from it is NaN; t is taken over the finite
// elements.
//
// Scales leave in the order in which the tensor core takes them:
// [row / 128][block / 4][row % 32][row / 32 % 4][block % 4], one byte each,
// zeros where a row or a block of that grid does not exist.
#include <cuda_fp4.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <utility>

#include "common.h"
#include "fp8.cuh"

namespace st {
namespace {

constexpr int kThreads = 256;
constexpr int kAmaxPerSm = 4;  // CTAs of the tensor's maximum; each leaves one number
constexpr int kMostMaxima = 1024;

__device__ __forceinline__ int64_t cdiv_dev(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The tensor scale of an empty tensor.
__global__ void unit_scale_kernel(float *t) {
    pdl_wait();
    *t = 1.0f;
    pdl_trigger();
}
constexpr int kWarps = kThreads / 32;

// The exponent e of the least power of two with limit * 2^e >= top, limit
// given as fraction in [1, 2) times 2^shift; top > 0 and finite.
__device__ __forceinline__ int least_power(float top, float fraction, int shift) {
    const uint32_t bits = __float_as_uint(top);
    const int exponent = static_cast<int>(bits >> 23);  // 0: subnormal, far below any limit's reach
    if (exponent == 0) return -1000;
    const float m = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
    return exponent - 127 - shift + (m > fraction ? 1 : 0);
}

__device__ __forceinline__ float power_of_two(int e) {  // -149 <= e <= 127
    return e >= -126 ? __uint_as_float(static_cast<uint32_t>(e + 127) << 23) : __uint_as_float(1u << (e + 149));
}

__device__ __forceinline__ float finite_abs(float m, float v) {
    v = fabsf(v);
    return v < INFINITY && v > m ? v : m;  // false for a NaN
}

__device__ __forceinline__ float block_max(float m, float *shared) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = m;
    __syncthreads();
    m = shared[0];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) m = fmaxf(m, shared[w]);
    __syncthreads();
    return m;
}

// ---------------------------------------------------------------- the tensor's largest |a|
// One maximum per CTA; the quantiser's CTAs reduce them.
template <typename T, bool WORDS>
__global__ void __launch_bounds__(kThreads) amax_kernel(const T *a, int64_t s0, int64_t s1, int64_t rows, int64_t cols,
                                                        float *maxima) {
    pdl_wait();
    __shared__ float shared[kWarps];
    float m = 0.0f;
    constexpr int kVec = 16 / static_cast<int>(sizeof(T));
    const int64_t per_row = WORDS ? cols / kVec : cols;
    const int64_t total = rows * per_row, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    if constexpr (WORDS) {
        // the row and column of a stride's step, so that the loop divides nothing
        const int64_t dr = stride / per_row, dc = stride - dr * per_row;
        int64_t r = first / per_row, c = first - r * per_row;
        for (int64_t i = first; i < total; i += 4 * stride) {
            uint4 w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = make_uint4(0, 0, 0, 0);
                if (i + j * stride < total) w[j] = *reinterpret_cast<const uint4 *>(a + r * s0 + c * kVec);
                r += dr;
                c += dc;
                if (c >= per_row) {
                    c -= per_row;
                    ++r;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const T *e = reinterpret_cast<const T *>(&w[j]);
#pragma unroll
                for (int k = 0; k < kVec; ++k) m = finite_abs(m, to_float(e[k]));
            }
        }
        const int64_t tail = per_row * kVec, left = cols - tail;  // the columns behind the last whole word
        for (int64_t i = first; i < rows * left; i += stride) m = finite_abs(m, to_float(a[i / left * s0 + tail + i % left]));
    } else {
        for (int64_t i = first; i < total; i += stride) {
            const int64_t r = i / cols;
            m = finite_abs(m, to_float(a[r * s0 + (i - r * cols) * s1]));
        }
    }
    m = block_max(m, shared);
    if (threadIdx.x == 0) maxima[blockIdx.x] = m;
    pdl_trigger();
}

// ---------------------------------------------------------------- the tensor scale of a call, in every CTA
struct Unit {
    float t, inverse;   // a power of two and its inverse, both times (over) lift
    float lift;         // elements are multiplied by it first: 1, or 2^100 for tensors so small that t / 448 is subnormal
};

__device__ __forceinline__ Unit tensor_unit(const Quantize4Args &p, float *shared) {
    float m = 0.0f;
    for (int i = threadIdx.x; i < p.n_maxima; i += kThreads) m = finite_abs(m, p.maxima[i]);
    m = block_max(m, shared);
    int e = 0;
    if (m > 0.0f) {
        e = least_power(m, 1.3125f, 11);
        if (e < -126) e = -126;
    }
    if (p.tensor_scale != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *p.tensor_scale = power_of_two(e);
    const int lift = e < -100 ? 100 : 0;
    return Unit{power_of_two(e + lift), power_of_two(-e - lift), power_of_two(lift)};
}

// ---------------------------------------------------------------- one block
// What one block needs: its scale's byte, s t and its inverse (0 for a block
// of zeros, whose codes are then zeros).
struct BlockScale {
    uint32_t byte;
    float unit, inverse;
};

template <bool WIDE>  // blocks of 32
__device__ __forceinline__ BlockScale block_scale(float top, const Unit &u) {
    if (!(top < INFINITY)) return BlockScale{WIDE ? 0xffu : 0x7fu, 0.0f, 0.0f};
    if constexpr (WIDE) {
        int e = top > 0.0f ? least_power(top, 1.5f, 2) : -127;
        if (e < -127) e = -127;
        return BlockScale{static_cast<uint32_t>(e + 127), power_of_two(e), power_of_two(-e)};
    } else {
        const uint32_t byte = __nv_cvt_float_to_fp8(__fdiv_rn(top * u.inverse, 6.0f), __NV_SATFINITE, __NV_E4M3);
        const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
        if (s == 0.0f) return BlockScale{0u, 0.0f, 0.0f};
        return BlockScale{byte, s * u.t, __frcp_rn(s) * u.inverse};
    }
}

// Eight codes of four pairs, the first in the low half of the low byte.
__device__ __forceinline__ uint32_t to_fp4x8(const uint64_t (&f)[4]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(lo2(f[0])), "f"(hi2(f[0])), "f"(lo2(f[1])), "f"(hi2(f[1])), "f"(lo2(f[2])), "f"(hi2(f[2])), "f"(lo2(f[3])),
          "f"(hi2(f[3])));
    return r;
}

// The codes of eight elements.  Blocks of 16: the quotient by s t is the
// product with the rounded inverse, corrected once by its residual (Markstein
// 1990), so that an element on a border between two codes is found there.  It
// is taken with the opposite sign, which is turned at the end: so a zero keeps
// the sign that x - x would lose.
template <bool WIDE>
__device__ __forceinline__ uint32_t codes8(const uint64_t (&x)[4], const BlockScale &b) {
    const float inverse = WIDE ? b.inverse : -b.inverse;
    const uint64_t inv = pack2(inverse, inverse);
    uint64_t q[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[j] = mul2(x[j], inv);
        if constexpr (!WIDE) {
            const uint64_t rest = fma2(q[j], pack2(b.unit, b.unit), x[j]);
            q[j] = fma2(rest, inv, q[j]);
        }
    }
    return to_fp4x8(q) ^ (WIDE ? 0u : 0x88888888u);
}

__device__ __forceinline__ float max_abs8(float m, const uint64_t (&x)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) m = max_abs(m, lo2(x[j]), hi2(x[j]));
    return m;
}

// Where the scale of block b (of `quads` groups of four a row) of a row lies.
__device__ __forceinline__ int64_t scale_at(int64_t row, int64_t b, int64_t quads) {
    return ((row >> 7) * quads + (b >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (b & 3);
}

// Sixteen elements of one row from column c on (of the view's columns) as
// fp32 pairs; zeros behind the edge.
template <typename T>
__device__ __forceinline__ void load16_words(const T *src, int64_t left, uint64_t (&x)[2][4]) {
    constexpr int kWords = static_cast<int>(sizeof(T) / 2);
    uint4 w[2][kWords];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) w[h][k] = make_uint4(0, 0, 0, 0);
        if (left >= 8 * h + 8) {
#pragma unroll
            for (int k = 0; k < kWords; ++k) w[h][k] = __ldcs(reinterpret_cast<const uint4 *>(src + 8 * h) + k);
        } else {
            T *e = reinterpret_cast<T *>(w[h]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (8 * h + j < left) e[j] = src[8 * h + j];
        }
    }
    unpack8(w[0], x[0], T{});
    unpack8(w[1], x[1], T{});
}

// The 8 bytes of 16 codes, or those of the first n elements.
__device__ __forceinline__ void store_codes(uint8_t *to, uint32_t lo, uint32_t hi, int64_t left, bool words) {
    if (left >= 16 && words) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(lo, hi);
    } else {
        const int bytes = left >= 16 ? 8 : static_cast<int>((left + 1) / 2);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < bytes) to[j] = static_cast<uint8_t>((j < 4 ? lo : hi) >> (8 * (j & 3)));
    }
}

// A lane holds 16 elements of a row, consecutive lanes consecutive ones: their
// codes, and four lanes' (blocks of 32: eight lanes') scales as one word.
// row / unit name the 16 elements; every lane of the warp comes here.
template <bool WIDE>
__device__ __forceinline__ void quantize_unit(const Quantize4Args &p, const Unit &u, uint64_t (&x)[2][4], int64_t row,
                                              int64_t unit, int64_t quads, bool here, bool words) {
    if (!WIDE && u.lift != 1.0f) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[h][j] = mul2(x[h][j], pack2(u.lift, u.lift));
    }
    float top = max_abs8(max_abs8(0.0f, x[0]), x[1]);
    if constexpr (WIDE) top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, 1));
    const BlockScale b = block_scale<WIDE>(top, u);
    const uint32_t lo = codes8<WIDE>(x[0], b), hi = codes8<WIDE>(x[1], b);
    // one byte from each of four blocks, to the first of their lanes
    const int step = WIDE ? 2 : 1;
    uint32_t word = b.byte | (__shfl_down_sync(0xffffffffu, b.byte, step) << 8);
    word |= __shfl_down_sync(0xffffffffu, word, 2 * step) << 16;
    if (!here) return;
    const int64_t left = p.cols - unit * 16;
    if (row < p.rows && left > 0) store_codes(p.q + row * p.sq0 + unit * 8, lo, hi, left, words);
    const int64_t block = WIDE ? unit >> 1 : unit;
    if ((WIDE ? unit & 7 : unit & 3) == 0) *reinterpret_cast<uint32_t *>(p.scale + scale_at(row, block, quads)) = word;
}

// ---------------------------------------------------------------- rows on 16-byte boundaries
// A lane takes 16 elements of a row, a CTA walks the tensor from its end: the
// maximum has just passed over it from the start, and the end is still in L2.
// Rows are padded to 128 and a row's blocks to four, as the scales are.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) quantize4_rows_kernel(const Quantize4Args p, int64_t units, int64_t quads,
                                                                  bool words) {
    pdl_wait();
    __shared__ float shared[kWarps];
    const Unit u = WIDE ? Unit{1.0f, 1.0f, 1.0f} : tensor_unit(p, shared);
    const int64_t padded = (p.rows + 127) / 128 * 128, total = padded * units, chunks = cdiv_dev(total, 32);
    const int lane = threadIdx.x & 31;
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < chunks;
         w += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int64_t i = (chunks - 1 - w) * 32 + lane;
        const bool here = i < total;
        // units of a row are a multiple of the lanes of one scale word, so a word's lanes lie in one row
        const int64_t row = here ? i / units : 0, unit = here ? i - row * units : 0;
        uint64_t x[2][4] = {};
        if (here && row < p.rows) load16_words(static_cast<const T *>(p.a) + row * p.sa0 + unit * 16, p.cols - unit * 16, x);
        quantize_unit<WIDE>(p, u, x, row, unit, quads, here, words);
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- any strides
// A warp takes 512 elements of a row, 32 of them a read, and turns them in
// shared memory into 16 a lane (17 words apart, without bank conflicts).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) quantize4_any_kernel(const Quantize4Args p, int64_t units, int64_t quads,
                                                                 bool words) {
    pdl_wait();
    __shared__ float shared[kWarps];
    __shared__ float turned[kWarps][32 * 17];
    const Unit u = WIDE ? Unit{1.0f, 1.0f, 1.0f} : tensor_unit(p, shared);
    const int64_t padded = (p.rows + 127) / 128 * 128, per_row = cdiv_dev(units, 32), chunks = padded * per_row;
    const int lane = threadIdx.x & 31;
    float *mine = turned[threadIdx.x >> 5];
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < chunks;
         w += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int64_t at = chunks - 1 - w, row = at / per_row, first = (at - row * per_row) * 512;
        const T *src = static_cast<const T *>(p.a) + row * p.sa0;
        T v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int64_t c = first + 32 * j + lane;
            from_float(0.0f, v[j]);
            if (row < p.rows && c < p.cols) v[j] = src[c * p.sa1];
        }
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int e = 32 * j + lane;
            mine[e + e / 16] = to_float(v[j]);
        }
        __syncwarp();
        uint64_t x[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) x[h][j] = pack2(mine[17 * lane + 8 * h + 2 * j], mine[17 * lane + 8 * h + 2 * j + 1]);
        const int64_t unit = first / 16 + lane;
        quantize_unit<WIDE>(p, u, x, row, unit, quads, unit < units, words);
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- stored by columns (rows contiguous)
// A lane takes ROWS neighbouring rows and the four blocks of one scale word,
// so that a read of the warp is 32 * ROWS neighbouring elements and a row's
// codes leave as whole 32-byte (64-byte) sectors.
template <typename T, bool WIDE, int ROWS>
__global__ void __launch_bounds__(kThreads) quantize4_columns_kernel(const Quantize4Args p, int64_t quads, bool words) {
    pdl_wait();
    __shared__ float shared[kWarps];
    const Unit u = WIDE ? Unit{1.0f, 1.0f, 1.0f} : tensor_unit(p, shared);
    constexpr int kSpan = WIDE ? 128 : 64, kUnits = kSpan / 16;
    const int64_t padded = (p.rows + 127) / 128 * 128, groups = padded / (32 * ROWS), chunks = groups * quads;
    const int lane = threadIdx.x & 31;
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < chunks;
         w += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int64_t at = chunks - 1 - w, quad = at / groups, row0 = (at - quad * groups) * 32 * ROWS + lane * ROWS;
        uint32_t codes[ROWS][2 * kUnits], scales[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) scales[r] = 0;
        float tops[ROWS];
        uint64_t x[ROWS][WIDE ? 4 : 2][4];
        constexpr int kStep = WIDE ? 2 : 1;  // units of a block
#pragma unroll
        for (int b = 0; b < 4; ++b) {
#pragma unroll
            for (int s = 0; s < kStep; ++s) {
                T v[ROWS][16];
                const int64_t c0 = quad * kSpan + (b * kStep + s) * 16;
                const T *src = static_cast<const T *>(p.a) + row0 + c0 * p.sa1;
#pragma unroll
                for (int j = 0; j < 16; ++j) {
#pragma unroll
                    for (int r = 0; r < ROWS; ++r) from_float(0.0f, v[r][j]);
                    if (c0 + j < p.cols) {
                        if (ROWS == 2 && row0 + 1 < p.rows) {
                            const uint32_t both = __ldcs(reinterpret_cast<const uint32_t *>(src + j * p.sa1));
                            *reinterpret_cast<uint16_t *>(&v[0][j]) = static_cast<uint16_t>(both);
                            *reinterpret_cast<uint16_t *>(&v[ROWS - 1][j]) = static_cast<uint16_t>(both >> 16);
                        } else if (row0 < p.rows) {
                            v[0][j] = src[j * p.sa1];
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < ROWS; ++r)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            x[r][2 * s + h][j] = mul2(pack2(to_float(v[r][8 * h + 2 * j]), to_float(v[r][8 * h + 2 * j + 1])),
                                                      pack2(u.lift, u.lift));
            }
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                tops[r] = max_abs8(max_abs8(0.0f, x[r][0]), x[r][1]);
                if constexpr (WIDE) tops[r] = max_abs8(max_abs8(tops[r], x[r][2]), x[r][3]);
                const BlockScale s = block_scale<WIDE>(tops[r], u);
                scales[r] |= s.byte << (8 * b);
#pragma unroll
                for (int h = 0; h < 2 * kStep; ++h) codes[r][2 * kStep * b + h] = codes8<WIDE>(x[r][h], s);
            }
        }
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            const int64_t row = row0 + r;
            *reinterpret_cast<uint32_t *>(p.scale + scale_at(row, quad * 4, quads)) = scales[r];
            if (row >= p.rows) continue;
            uint8_t *to = p.q + row * p.sq0 + quad * (kSpan / 2);
#pragma unroll
            for (int k = 0; k < kUnits; ++k) {
                const int64_t left = p.cols - quad * kSpan - 16 * k;
                if (left > 0) store_codes(to + 8 * k, codes[r][2 * k], codes[r][2 * k + 1], left, words);
            }
        }
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- back to values
// A thread per 16 codes.
template <typename T>
__global__ void __launch_bounds__(kThreads) dequantize4_kernel(const Dequantize4Args p, int64_t units, int64_t quads, bool words,
                                                               bool out_words) {
    pdl_wait();
    const float t = p.tensor_scale != nullptr ? *p.tensor_scale : 1.0f;
    const int64_t total = p.rows * units, stride = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < total; i += stride) {
        const int64_t row = i / units, unit = i - row * units, left = p.cols - unit * 16;
        const uint8_t *q = p.q + row * p.sq0 + unit * 8 * p.sq1;
        uint32_t code[2] = {0, 0};
        if (left >= 16 && words) {
            const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(q));
            code[0] = v.x;
            code[1] = v.y;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (2 * j < left) code[j / 4] |= static_cast<uint32_t>(q[j * p.sq1]) << (8 * (j & 3));
        }
        const uint32_t byte = p.scale[scale_at(row, p.wide ? unit >> 1 : unit, quads)];
        float s;
        if (p.wide) s = byte == 255u ? NAN : power_of_two(static_cast<int>(byte) - 127);
        else s = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
        const float unit_scale = s * t;
        uint64_t f[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const __half2_raw v = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(code[h] >> (8 * j)), __NV_E2M1);
                const float2 w = __half22float2(__half2(v));
                f[h][j] = mul2(pack2(w.x, w.y), pack2(unit_scale, unit_scale));
            }
        T *out = static_cast<T *>(p.out) + row * p.so0 + unit * 16 * p.so1;
        if (left >= 16 && out_words) {
            constexpr int kWords = static_cast<int>(sizeof(T) / 2);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint4 w[kWords];
                pack8(f[h], w, T{});
#pragma unroll
                for (int k = 0; k < kWords; ++k) reinterpret_cast<uint4 *>(out + 8 * h)[k] = w[k];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < left) from_float(j & 1 ? hi2(f[j / 8][j % 8 / 2]) : lo2(f[j / 8][j % 8 / 2]), out[j * p.so1]);
        }
    }
    pdl_trigger();
}

int checked(const char *what) {
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), what);
}

// CTAs for `work` of them, at most `per_sm` on each SM.
unsigned grid_of(int64_t work, int sm_count, int per_sm) {
    const int64_t most = static_cast<int64_t>(sm_count) * per_sm;
    return static_cast<unsigned>(work < 1 ? 1 : work < most ? work : most);
}

bool on16(const void *p, int64_t stride, int64_t rows, int64_t size) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && (rows == 1 || stride * size % 16 == 0);
}

template <typename T>
int launch_amax(Quantize4Args &p, float *maxima, int sm_count, cudaStream_t stream) {
    // the maximum does not mind the order: along whichever dimension is contiguous
    int64_t rows = p.rows, cols = p.cols, s0 = p.sa0, s1 = p.sa1;
    if (s1 != 1 && s0 == 1) {
        std::swap(rows, cols);
        std::swap(s0, s1);
    }
    const T *a = static_cast<const T *>(p.a);
    constexpr int kVec = 16 / static_cast<int>(sizeof(T));
    const bool words = (s1 == 1 || cols == 1) && cols >= kVec && on16(a, s0, rows, sizeof(T));
    unsigned grid = grid_of(cdiv(rows * cols, kThreads * (words ? 4 * kVec : 4)), sm_count, kAmaxPerSm);
    if (grid > kMostMaxima) grid = kMostMaxima;
    if (words) ST_CUDA_TRY(launch_kernel(amax_kernel<T, true>, grid, kThreads, 0, stream, a, s0, s1, rows, cols, maxima));
    else ST_CUDA_TRY(launch_kernel(amax_kernel<T, false>, grid, kThreads, 0, stream, a, s0, s1, rows, cols, maxima));
    p.maxima = maxima;
    p.n_maxima = static_cast<int>(grid);
    return checked("amax_kernel");
}

template <typename T, bool WIDE>
int launch_quantize(const Quantize4Args &p, int sm_count, cudaStream_t stream) {
    const int64_t blocks = cdiv(p.cols, WIDE ? 32 : 16), quads = cdiv(blocks, 4), units = quads * (WIDE ? 8 : 4);
    const int64_t padded = cdiv(p.rows, 128) * 128;
    const bool words = reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.sq0 % 8 == 0);
    if (p.cols == 1 || p.sa1 == 1) {
        if (on16(p.a, p.sa0, p.rows, sizeof(T))) {
            const unsigned grid = grid_of(cdiv(padded * units, kThreads), sm_count, 8);
            ST_CUDA_TRY(launch_kernel(quantize4_rows_kernel<T, WIDE>, grid, kThreads, 0, stream, p, units, quads, words));
            return checked("quantize4_rows_kernel");
        }
    } else if (p.sa0 == 1 && p.rows > 1) {
        const bool two = sizeof(T) == 2 && reinterpret_cast<uintptr_t>(p.a) % 4 == 0 && p.sa1 % 2 == 0;
        const unsigned grid = grid_of(cdiv(padded / (two ? 64 : 32) * quads, kWarps), sm_count, 8);
        if constexpr (sizeof(T) == 2) {
            if (two) {
                ST_CUDA_TRY(launch_kernel(quantize4_columns_kernel<T, WIDE, 2>, grid, kThreads, 0, stream, p, quads, words));
                return checked("quantize4_columns_kernel");
            }
        }
        ST_CUDA_TRY(launch_kernel(quantize4_columns_kernel<T, WIDE, 1>, grid, kThreads, 0, stream, p, quads, words));
        return checked("quantize4_columns_kernel");
    }
    const unsigned grid = grid_of(cdiv(padded * cdiv(units, 32), kWarps), sm_count, 8);
    ST_CUDA_TRY(launch_kernel(quantize4_any_kernel<T, WIDE>, grid, kThreads, 0, stream, p, units, quads, words));
    return checked("quantize4_any_kernel");
}

template <typename T>
int launch_typed(Quantize4Args p, float *maxima, int sm_count, cudaStream_t stream) {
    if (p.wide) return launch_quantize<T, true>(p, sm_count, stream);
    if (p.maxima == nullptr) ST_TRY(launch_amax<T>(p, maxima, sm_count, stream));
    return launch_quantize<T, false>(p, sm_count, stream);
}

template <typename T>
int launch_dequantize(const Dequantize4Args &p, int sm_count, cudaStream_t stream) {
    const int64_t units = cdiv(p.cols, 16), quads = cdiv(cdiv(p.cols, p.wide ? 32 : 16), 4);
    const bool words = p.sq1 == 1 && reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.sq0 % 8 == 0);
    const bool out_words = p.so1 == 1 && on16(p.out, p.so0, p.rows, sizeof(T));
    const unsigned grid = grid_of(cdiv(p.rows * units, kThreads), sm_count, 8);
    ST_CUDA_TRY(launch_kernel(dequantize4_kernel<T>, grid, kThreads, 0, stream, p, units, quads, words, out_words));
    return checked("dequantize4_kernel");
}

}  // namespace

int64_t quantize_fp4_workspace_bytes() { return kMostMaxima * sizeof(float); }

int launch_quantize_fp4(const Quantize4Args &p, void *workspace, int sm_count, cudaStream_t stream) {
    if (p.rows == 0 || p.cols == 0) {
        if (p.tensor_scale != nullptr) {
            ST_CUDA_TRY(launch_kernel(unit_scale_kernel, 1, 1, 0, stream, p.tensor_scale));
            return checked("unit_scale_kernel");
        }
        return ST_OK;
    }
    float *maxima = static_cast<float *>(workspace);
    switch (p.a_dtype) {
    case ST_F32: return launch_typed<float>(p, maxima, sm_count, stream);
    case ST_F16: return launch_typed<__half>(p, maxima, sm_count, stream);
    default: return launch_typed<__nv_bfloat16>(p, maxima, sm_count, stream);
    }
}

int launch_dequantize_fp4(const Dequantize4Args &p, int sm_count, cudaStream_t stream) {
    if (p.rows == 0 || p.cols == 0) return ST_OK;
    switch (p.out_dtype) {
    case ST_F32: return launch_dequantize<float>(p, sm_count, stream);
    case ST_F16: return launch_dequantize<__half>(p, sm_count, stream);
    default: return launch_dequantize<__nv_bfloat16>(p, sm_count, stream);
    }
}

}  // namespace st
