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
// Bound by DRAM: 8192 x 8192 bf16 in 33 us in blocks of 16 with a known maximum
// and in 30 in blocks of 32 (26.2 at the copy rate); the maximum's own pass takes
// 25; back to values 32 (26.2).  (A replayed graph over three inputs; over one,
// part of which stays in L2, 29 and 26.)
//
// Scales leave in the order in which the tensor core takes them:
// [row / 128][block / 4][row % 32][row / 32 % 4][block % 4], one byte each,
// zeros where a row or a block of that grid does not exist.
#include <cuda_fp4.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>
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
// One maximum per CTA; the quantiser's CTAs reduce them.  A NaN loses every
// comparison; a CTA whose maximum comes out infinite takes it again, over the
// finite ones of the elements that it has read.
__device__ __forceinline__ float max_of_word(float m, const uint4 &w, float) {
    m = fmaxf(fmaxf(m, fabsf(__uint_as_float(w.x))), fabsf(__uint_as_float(w.y)));
    return fmaxf(fmaxf(m, fabsf(__uint_as_float(w.z))), fabsf(__uint_as_float(w.w)));
}
template <typename T2>
__device__ __forceinline__ T2 max_of_word2(T2 m, const uint4 &w) {
    const T2 *e = reinterpret_cast<const T2 *>(&w);
    return __hmax2(__hmax2(m, __hmax2(__habs2(e[0]), __habs2(e[1]))), __hmax2(__habs2(e[2]), __habs2(e[3])));
}
__device__ __forceinline__ __half2 max_of_word(__half2 m, const uint4 &w, __half) { return max_of_word2(m, w); }
__device__ __forceinline__ __nv_bfloat162 max_of_word(__nv_bfloat162 m, const uint4 &w, __nv_bfloat16) { return max_of_word2(m, w); }
__device__ __forceinline__ float start_of(float) { return 0.0f; }
__device__ __forceinline__ __half2 start_of(__half) { return __float2half2_rn(0.0f); }
__device__ __forceinline__ __nv_bfloat162 start_of(__nv_bfloat16) { return __float2bfloat162_rn(0.0f); }
__device__ __forceinline__ float end_of(float m) { return m; }
__device__ __forceinline__ float end_of(__half2 m) { return fmaxf(__low2float(m), __high2float(m)); }
__device__ __forceinline__ float end_of(__nv_bfloat162 m) { return fmaxf(__low2float(m), __high2float(m)); }

// A thread's maximum over the finite ones of the elements that amax_kernel has
// it read: of the same words, as no other CTA has seen them.  (Its loops
// unrolled it takes registers from the first pass: 8192 x 8192 f32 93 -> 95 us a call.)
template <typename T, bool WORDS>
__device__ __forceinline__ float finite_max(const T *a, int64_t s0, int64_t s1, int64_t rows, int64_t cols, int64_t first, int64_t stride) {
    float m = 0.0f;
    if constexpr (WORDS) {
        constexpr int kVec = 16 / static_cast<int>(sizeof(T));
        const int64_t per_row = cols / kVec, tail = per_row * kVec, left = cols - tail;
#pragma unroll 1
        for (int64_t i = first; i < rows * per_row; i += stride) {
            const T *word = a + i / per_row * s0 + i % per_row * kVec;
#pragma unroll 1
            for (int j = 0; j < kVec; ++j) m = finite_abs(m, to_float(word[j]));
        }
#pragma unroll 1
        for (int64_t i = first; i < rows * left; i += stride) m = finite_abs(m, to_float(a[i / left * s0 + tail + i % left]));
    } else {
#pragma unroll 1
        for (int64_t i = first; i < rows * cols; i += stride) {
            const int64_t r = i / cols;
            m = finite_abs(m, to_float(a[r * s0 + (i - r * cols) * s1]));
        }
    }
    return m;
}

template <typename T, bool WORDS>
__global__ void __launch_bounds__(kThreads) amax_kernel(const T *a, int64_t s0, int64_t s1, int64_t rows, int64_t cols,
                                                        float *maxima) {
    pdl_wait();
    __shared__ float shared[kWarps];
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x;
    float m = 0.0f;
    if constexpr (WORDS) {
        constexpr int kVec = 16 / static_cast<int>(sizeof(T)), kAtOnce = 8;
        const int64_t per_row = cols / kVec, total = rows * per_row;
        // the row and column of a stride's step, so that the loop divides nothing
        const int64_t dr = stride / per_row, dc = stride - dr * per_row;
        int64_t r = first / per_row, c = first - r * per_row;
        auto most = start_of(T{});
        for (int64_t i = first; i < total; i += kAtOnce * stride) {
            uint4 w[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
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
            for (int j = 0; j < kAtOnce; ++j) most = max_of_word(most, w[j], T{});
        }
        m = end_of(most);
        const int64_t tail = per_row * kVec, left = cols - tail;  // the columns behind the last whole word
        for (int64_t i = first; i < rows * left; i += stride) m = fmaxf(m, fabsf(to_float(a[i / left * s0 + tail + i % left])));
    } else {
        for (int64_t i = first; i < rows * cols; i += stride) {
            const int64_t r = i / cols;
            m = fmaxf(m, fabsf(to_float(a[r * s0 + (i - r * cols) * s1])));
        }
    }
    m = block_max(m, shared);
    if (m == INFINITY) m = block_max(finite_max<T, WORDS>(a, s0, s1, rows, cols, first, stride), shared);
    if (threadIdx.x == 0) maxima[blockIdx.x] = m;
    pdl_trigger();
}

// ---------------------------------------------------------------- the tensor scale of a call, in every CTA
struct Unit {
    float t, inverse;   // a power of two and its inverse, both times (over) lift
    float lift;         // elements are multiplied by it first: 1, or 2^100 for tensors so small that t / 448 is subnormal
    float usual;        // a block with a larger maximum (or a NaN) goes through limit_top and limit8
};

// What blocks beyond u.usual take first.  8192 t is more than three times what
// t provides for: from there on the block's scale is the largest one and the
// element's code too, whatever is above, so that elements are taken as 8192 t
// (infinite for the largest t) and nothing behind this overflows.  Then the lift.
__device__ __forceinline__ float most_of(const Unit &u) { return u.lift != 1.0f ? u.t * (8192.0f * 0x1p-100f) : u.t * 8192.0f; }
__device__ __forceinline__ float limit_top(float top, const Unit &u) {
    return top < INFINITY ? fminf(top, most_of(u)) * u.lift : top;  // infinity and NaN stay
}
__device__ __forceinline__ void limit8(uint64_t (&x)[4], const Unit &u) {
    const float most = most_of(u);
#pragma unroll
    for (int j = 0; j < 4; ++j)
        x[j] = mul2(pack2(fminf(fmaxf(lo2(x[j]), -most), most), fminf(fmaxf(hi2(x[j]), -most), most)), pack2(u.lift, u.lift));
}

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
    const float t = power_of_two(e + lift);
    return Unit{t, power_of_two(-e - lift), power_of_two(lift), lift ? -1.0f : t * 8192.0f};
}

// ---------------------------------------------------------------- one block
// What one block needs: its scale's byte, s t and its inverse (0 for a block
// of zeros, whose codes are then zeros).
struct BlockScale {
    uint32_t byte;
    float unit, inverse;
};

__device__ __forceinline__ float approximate_inverse(float v) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

template <bool WIDE>  // blocks of 32
__device__ __forceinline__ BlockScale block_scale(float top, const Unit &u) {
    const bool finite = top < INFINITY;
    if constexpr (WIDE) {
        int e = least_power(top, 1.5f, 2);
        if (e < -127) e = -127;
        return finite ? BlockScale{static_cast<uint32_t>(e + 127), power_of_two(e), power_of_two(-e)} : BlockScale{0xffu, 0.0f, 0.0f};
    } else {
        // a sixth, correctly rounded: the product with the rounded inverse, corrected by its residual (see codes8)
        const float y = top * u.inverse, r = 1.0f / 6.0f, q = y * r;
        const uint32_t byte = __nv_cvt_float_to_fp8(__fmaf_rn(__fmaf_rn(q, -6.0f, y), r, q), __NV_SATFINITE, __NV_E4M3);
        const float s = __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
        const bool live = finite && s > 0.0f;
        return BlockScale{finite ? byte : 0x7fu, live ? s * u.t : 0.0f, live ? approximate_inverse(s) * u.inverse : 0.0f};
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
// product with the inverse, corrected once by its residual (Markstein 1990), so
// that an element on a border between two codes is found there.  (s has four
// bits, so a quotient by it is a thirtieth of a step or more from the middle
// between two fp32 numbers, unless it is on it; the corrected product is off by
// about 2^-45 of itself, so it rounds like the quotient although the inverse is
// only good to a step.)  It
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
// A row's blocks are padded to four and the rows to 128, so that one row of
// 2^29 elements has 2^32 bytes of scales: only the count of 512 bytes, of
// which no GPU has 2^32, and the place inside of them are 32 bits.
__device__ __forceinline__ int64_t scale_at(int64_t row, int64_t b, int64_t quads) {
    const uint32_t r = static_cast<uint32_t>(row), k = static_cast<uint32_t>(b);
    return static_cast<int64_t>((r >> 7) * static_cast<uint32_t>(quads) + (k >> 2)) * 512 + ((r & 31u) * 16u + ((r >> 5) & 3u) * 4u + (k & 3u));
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
template <bool WIDE, bool WHOLE>
__device__ __forceinline__ void quantize_unit(const Quantize4Args &p, const Unit &u, uint64_t (&x)[2][4], int64_t row,
                                              int64_t unit, int64_t quads, bool here, bool words) {
    float top = max_abs8(max_abs8(0.0f, x[0]), x[1]);
    if constexpr (WIDE) {
        top = max_abs(top, __shfl_xor_sync(0xffffffffu, top, 1));
    } else {
        if (!(top <= u.usual)) {
            top = limit_top(top, u);
            limit8(x[0], u);
            limit8(x[1], u);
        }
    }
    const BlockScale b = block_scale<WIDE>(top, u);
    const uint32_t lo = codes8<WIDE>(x[0], b), hi = codes8<WIDE>(x[1], b);
    // one byte from each of four blocks, to the first of their lanes
    const int step = WIDE ? 2 : 1;
    uint32_t word = b.byte | (__shfl_down_sync(0xffffffffu, b.byte, step) << 8);
    word |= __shfl_down_sync(0xffffffffu, word, 2 * step) << 16;
    if (!here) return;
    const int64_t left = p.cols - unit * 16;
    if (row < p.rows && left > 0) {
        uint8_t *to = p.q + row * p.sq0 + unit * 8;
        if constexpr (WHOLE) *reinterpret_cast<uint2 *>(to) = make_uint2(lo, hi);
        else store_codes(to, lo, hi, left, words);
    }
    const int64_t block = WIDE ? unit >> 1 : unit;
    if ((WIDE ? unit & 7 : unit & 3) == 0) *reinterpret_cast<uint32_t *>(p.scale + scale_at(row, block, quads)) = word;
}

// ---------------------------------------------------------------- rows on 16-byte boundaries
// A lane takes 16 columns of two rows, whose reads are under way together.  The
// CTAs walk the tensor from its end: the maximum has just passed over it from
// the start, and the end is still in L2.  Rows are padded to 128 and a row's
// blocks to four, as the scales are.
// WHOLE: rows are a multiple of 16 columns, their codes on 8-byte boundaries.
template <typename T, bool WIDE, bool WHOLE>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 2 ? 4 : 3)
    quantize4_rows_kernel(const Quantize4Args p, uint32_t units, uint32_t across, uint32_t chunks, int64_t quads, bool words) {
    pdl_wait();
    __shared__ float shared[kWarps];
    const Unit u = WIDE ? Unit{1.0f, 1.0f, 1.0f, INFINITY} : tensor_unit(p, shared);
    constexpr int kWords = static_cast<int>(sizeof(T) / 2);
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t w = blockIdx.x * kWarps + (threadIdx.x >> 5); w < chunks; w += gridDim.x * kWarps) {
        const uint32_t at = chunks - 1 - w, pair = at / across, unit = (at - pair * across) * 32 + lane;
        const int64_t row0 = static_cast<int64_t>(pair) * 2;
        const int left = static_cast<int>(p.cols) - static_cast<int>(unit) * 16;  // columns from this lane's first on
        const T *src = static_cast<const T *>(p.a) + row0 * p.sa0 + unit * 16;
        uint4 raw[2][2][kWords];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool here = row0 + i < p.rows && left > 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int k = 0; k < kWords; ++k) raw[i][h][k] = make_uint4(0, 0, 0, 0);
                if (here && (WHOLE || left >= 8 * h + 8)) {
#pragma unroll
                    for (int k = 0; k < kWords; ++k) raw[i][h][k] = __ldcs(reinterpret_cast<const uint4 *>(src + i * p.sa0 + 8 * h) + k);
                } else if (!WHOLE && here) {
                    T *e = reinterpret_cast<T *>(raw[i][h]);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (8 * h + j < left) e[j] = src[i * p.sa0 + 8 * h + j];
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint64_t x[2][4];
            unpack8(raw[i][0], x[0], T{});
            unpack8(raw[i][1], x[1], T{});
            quantize_unit<WIDE, WHOLE>(p, u, x, row0 + i, unit, quads, unit < units, words);
        }
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
    const Unit u = WIDE ? Unit{1.0f, 1.0f, 1.0f, INFINITY} : tensor_unit(p, shared);
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
        quantize_unit<WIDE, false>(p, u, x, row, unit, quads, unit < units, words);
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- stored by columns (rows contiguous)
// A CTA takes 128 bytes of neighbouring rows and 8 units of 16 (of 32) columns
// into shared memory, where a warp finds a unit's elements of all the rows;
// the codes go through shared memory too, and leave as whole rows of the tile.
// (Each lane reading its rows' elements from global memory and storing 8 bytes
// a row took 255 us for 8192 x 8192 bf16.)
template <typename T, bool WIDE>
struct ColumnTile {
    static constexpr int kSpan = WIDE ? 32 : 16;  // columns of a block and a warp
    static constexpr int kCols = 8 * kSpan;
    static constexpr int kPer = 4 / static_cast<int>(sizeof(T));  // rows of a lane
    static constexpr int kRows = 32 * kPer;
    static constexpr int kPitch = 128 + 16;             // bytes of a column's rows
    static constexpr int kCodePitch = kCols / 2 + 4;    // bytes of a row's codes; a lane's rows lie on other banks than its neighbours'
    uint8_t in[kCols * kPitch];
    uint8_t codes[kRows * kCodePitch];
    uint8_t scales[kRows * 8];
};

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, WIDE && sizeof(T) == 2 ? 2 : 4)
    quantize4_columns_kernel(const Quantize4Args p, int64_t quads, bool in_words, bool words) {
    using Tile = ColumnTile<T, WIDE>;
    pdl_wait();
    __shared__ float shared[kWarps];
    extern __shared__ __align__(16) uint8_t tile_bytes[];
    Tile &tile = *reinterpret_cast<Tile *>(tile_bytes);
    const Unit u = WIDE ? Unit{1.0f, 1.0f, 1.0f, INFINITY} : tensor_unit(p, shared);
    const int64_t groups = (p.rows + 127) / 128 * (128 / Tile::kRows), total = groups * cdiv_dev(quads, 2);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // tile w from the end: its first row and column, and how many of each are inside
    struct Place {
        int64_t across, row0, col0;
        int rows, cols;
    };
    auto place = [&](int64_t w) {
        const int64_t at = total - 1 - w;
        Place t;
        t.across = at / groups;
        t.row0 = (at - t.across * groups) * Tile::kRows;
        t.col0 = t.across * Tile::kCols;
        t.rows = p.rows - t.row0 < Tile::kRows ? static_cast<int>(p.rows - t.row0) : Tile::kRows;
        t.cols = p.cols - t.col0 < Tile::kCols ? static_cast<int>(p.cols - t.col0) : Tile::kCols;
        return t;
    };
    // 16 bytes of a column a thread, 8 threads a column
    constexpr int kVec = 16 / static_cast<int>(sizeof(T)), kSteps = Tile::kCols / 32;
    auto read = [&](const Place &t, uint4 (&v)[kSteps]) {
        const T *src = static_cast<const T *>(p.a) + t.row0 + t.col0 * p.sa1;
        const int r = (threadIdx.x & 7) * kVec;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            const int c = static_cast<int>(threadIdx.x >> 3) + 32 * j;
            v[j] = make_uint4(0, 0, 0, 0);
            if (c < t.cols && r + kVec <= t.rows) {
                v[j] = __ldcs(reinterpret_cast<const uint4 *>(src + r + c * p.sa1));
            } else if (c < t.cols) {
                T *e = reinterpret_cast<T *>(&v[j]);
#pragma unroll
                for (int i = 0; i < kVec; ++i)
                    if (r + i < t.rows) e[i] = src[r + i + c * p.sa1];
            }
        }
    };
    // blocks of 32 of 16 bits, which fill the registers of two CTAs anyway, read the next tile beside this one's work
    // (8192 x 8192 bf16 43 -> 36 us; blocks of 16, with four CTAs an SM, 41 -> 44, over one input)
    constexpr bool kAhead = WIDE && sizeof(T) == 2;
    uint4 v[kSteps];
    if (kAhead && in_words && blockIdx.x < total) read(place(blockIdx.x), v);
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const Place t = place(w);
        const int64_t across = t.across, row0 = t.row0, col0 = t.col0;
        const int rows = t.rows, cols = t.cols;
        if (in_words) {
            if (!kAhead) read(t, v);
#pragma unroll
            for (int j = 0; j < kSteps; ++j)
                *reinterpret_cast<uint4 *>(tile.in + ((threadIdx.x >> 3) + 32 * j) * Tile::kPitch + (threadIdx.x & 7) * 16) = v[j];
            if (kAhead && w + gridDim.x < total) read(place(w + gridDim.x), v);
        } else {  // a column a warp at a time, an element a lane
            const T *src = static_cast<const T *>(p.a) + row0 + col0 * p.sa1;
#pragma unroll
            for (int j0 = 0; j0 < Tile::kSpan; j0 += 8) {
                T e[8][Tile::kPer];
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < Tile::kPer; ++i) {
                        const int c = warp * Tile::kSpan + j0 + j, r = lane + 32 * i;
                        from_float(0.0f, e[j][i]);
                        if (c < cols && r < rows) e[j][i] = src[r + c * p.sa1];
                    }
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int i = 0; i < Tile::kPer; ++i)
                        *reinterpret_cast<T *>(tile.in + (warp * Tile::kSpan + j0 + j) * Tile::kPitch + (lane + 32 * i) * sizeof(T)) = e[j][i];
            }
        }
        __syncthreads();
        // rows kPer lane, ... of the block of this warp: column j's in word j
        uint32_t word[Tile::kSpan];
        const uint8_t *mine = tile.in + warp * Tile::kSpan * Tile::kPitch + lane * 4;
#pragma unroll
        for (int j = 0; j < Tile::kSpan; ++j) word[j] = *reinterpret_cast<const uint32_t *>(mine + j * Tile::kPitch);
#pragma unroll
        for (int i = 0; i < Tile::kPer; ++i) {
            auto value = [&](int j) { return to_float(reinterpret_cast<const T *>(&word[j])[i]); };
            uint64_t x[Tile::kSpan / 8][4];
            float top = 0.0f;
#pragma unroll
            for (int j = 0; j < Tile::kSpan; j += 8) {
#pragma unroll
                for (int h = 0; h < 4; ++h) x[j / 8][h] = pack2(value(j + 2 * h), value(j + 2 * h + 1));
                top = max_abs8(top, x[j / 8]);
            }
            if constexpr (!WIDE) {
                if (!(top <= u.usual)) {
                    top = limit_top(top, u);
                    limit8(x[0], u);
                    limit8(x[1], u);
                }
            }
            const BlockScale b = block_scale<WIDE>(top, u);
            const int r = lane * Tile::kPer + i;
            tile.scales[r * 8 + warp] = static_cast<uint8_t>(b.byte);
#pragma unroll
            for (int j = 0; j < Tile::kSpan; j += 8)
                *reinterpret_cast<uint32_t *>(tile.codes + r * Tile::kCodePitch + (warp * Tile::kSpan + j) / 2) = codes8<WIDE>(x[j / 8], b);
        }
        __syncthreads();
        constexpr int kPieces = Tile::kCols / 32;  // 16 bytes of codes each
        const int bytes = (cols + 1) / 2;
        for (int i = threadIdx.x; i < Tile::kRows * kPieces; i += kThreads) {
            const int r = i / kPieces, q = i - r * kPieces, n = bytes - 16 * q;
            if (r >= rows || n <= 0) continue;
            const uint8_t *from = tile.codes + r * Tile::kCodePitch + 16 * q;
            uint8_t *to = p.q + (row0 + r) * p.sq0 + col0 / 2 + 16 * q;
            if (n >= 16 && words) {
                const uint32_t *f = reinterpret_cast<const uint32_t *>(from);
                *reinterpret_cast<uint4 *>(to) = make_uint4(f[0], f[1], f[2], f[3]);
            } else {
                for (int j = 0; j < 16 && j < n; ++j) to[j] = from[j];
            }
        }
        for (int i = threadIdx.x; i < Tile::kRows * 2; i += kThreads) {
            const int64_t quad = across * 2 + i / Tile::kRows;
            const int r = i % Tile::kRows;
            if (quad < quads)
                *reinterpret_cast<uint32_t *>(p.scale + scale_at(row0 + r, 4 * quad, quads)) =
                    *reinterpret_cast<const uint32_t *>(tile.scales + r * 8 + 4 * (i / Tile::kRows));
        }
        __syncthreads();  // the tile's next contents
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- back to values
// What a block's codes are multiplied by: an e4m3 scale in f16, where its
// product with a code is exact (6 bits, 2^-10 to 2688), then the tensor's scale
// in fp32, the one rounding; an e8m0 scale in fp32.
template <bool WIDE>
struct Back {
    __half2 scale;
    float factor;
    __device__ __forceinline__ Back(uint32_t byte, float t) {
        if constexpr (WIDE) {
            factor = byte == 255u ? NAN : power_of_two(static_cast<int>(byte) - 127);
        } else {
            scale = __half2half2(__half(__nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3)));
            factor = t;
        }
    }
    __device__ __forceinline__ uint64_t two(uint32_t byte) const {
        __half2 code = __half2(__nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(byte), __NV_E2M1));
        if constexpr (!WIDE) code = __hmul2(code, scale);
        const float2 v = __half22float2(code);
        return mul2(pack2(v.x, v.y), pack2(factor, factor));
    }
};

// The values of 16 codes.
template <bool WIDE>
__device__ __forceinline__ void values16(uint64_t (&f)[2][4], uint2 code, const Back<WIDE> &b) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < 4; ++j) f[h][j] = b.two((h ? code.y : code.x) >> (8 * j) & 0xffu);
}

// A lane takes 8 columns of eight rows, whose reads are under way together; its
// values of a row are 16 bytes of 16 bits, so that a warp's store is whole
// sectors (16 columns a lane: 42 us for 8192 x 8192 bf16, so 33).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads, 4) dequantize4_words_kernel(const Dequantize4Args p, uint32_t across, uint32_t chunks,
                                                                        int64_t quads) {
    pdl_wait();
    const float t = p.tensor_scale != nullptr ? *p.tensor_scale : 1.0f;
    const uint32_t lane = threadIdx.x & 31;
    constexpr int kRows = 8;
    for (uint32_t w = blockIdx.x * kWarps + (threadIdx.x >> 5); w < chunks; w += gridDim.x * kWarps) {
        const uint32_t group = w / across, part = (w - group * across) * 32 + lane;
        const int64_t row0 = static_cast<int64_t>(group) * kRows;
        const int left = static_cast<int>(p.cols) - static_cast<int>(part) * 8;
        if (left <= 0) continue;
        const uint8_t *q = p.q + row0 * p.sq0 + part * 4;
        const uint8_t *scale = p.scale + scale_at(row0, WIDE ? part >> 2 : part >> 1, quads);  // the next row's 16 bytes on
        uint32_t code[kRows], byte[kRows];
#pragma unroll
        for (int i = 0; i < kRows; ++i) {
            code[i] = byte[i] = 0;
            if (row0 + i >= p.rows) continue;
            if (left >= 8) {
                code[i] = __ldcs(reinterpret_cast<const uint32_t *>(q + i * p.sq0));
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (2 * j < left) code[i] |= static_cast<uint32_t>(q[i * p.sq0 + j]) << (8 * j);
            }
            byte[i] = scale[16 * i];
        }
        T *out = static_cast<T *>(p.out) + row0 * p.so0 + part * 8;
#pragma unroll
        for (int i = 0; i < kRows; ++i, out += p.so0) {
            if (row0 + i >= p.rows) break;
            const Back<WIDE> b(byte[i], t);
            uint64_t f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = b.two(code[i] >> (8 * j) & 0xffu);
            if (left >= 8) {
                constexpr int kWords = static_cast<int>(sizeof(T) / 2);
                uint4 o[kWords];
                pack8(f, o, T{});
#pragma unroll
                for (int k = 0; k < kWords; ++k) reinterpret_cast<uint4 *>(out)[k] = o[k];
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (j < left) from_float(j & 1 ? hi2(f[j / 2]) : lo2(f[j / 2]), out[j]);
            }
        }
    }
    pdl_trigger();
}

// Any strides, unit ones among them: a lane's 16 values are turned in shared
// memory, so that neighbouring lanes store neighbouring elements.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads) dequantize4_any_kernel(const Dequantize4Args p, uint32_t across, int64_t chunks,
                                                                   int64_t quads, bool words) {
    pdl_wait();
    __shared__ float turned[kWarps][32 * 17];
    const float t = p.tensor_scale != nullptr ? *p.tensor_scale : 1.0f;
    const uint32_t lane = threadIdx.x & 31;
    float *mine = turned[threadIdx.x >> 5];
    for (int64_t w = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5); w < chunks;
         w += static_cast<int64_t>(gridDim.x) * kWarps) {
        const int64_t row = w / across;
        const uint32_t chunk = static_cast<uint32_t>(w - row * across), unit = chunk * 32 + lane;
        const int left = static_cast<int>(p.cols) - static_cast<int>(unit) * 16;
        uint2 code = make_uint2(0, 0);
        uint32_t byte = 0;
        if (left > 0) {
            const uint8_t *q = p.q + row * p.sq0 + unit * 8 * p.sq1;
            if (left >= 16 && words) {
                code = __ldcs(reinterpret_cast<const uint2 *>(q));
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (2 * j < left) (j < 4 ? code.x : code.y) |= static_cast<uint32_t>(q[j * p.sq1]) << (8 * (j & 3));
            }
            byte = p.scale[scale_at(row, WIDE ? unit >> 1 : unit, quads)];
        }
        uint64_t f[2][4];
        values16(f, code, Back<WIDE>(byte, t));
        __syncwarp();
#pragma unroll
        for (int j = 0; j < 16; ++j) mine[17 * lane + j] = j & 1 ? hi2(f[j / 8][j % 8 / 2]) : lo2(f[j / 8][j % 8 / 2]);
        __syncwarp();
        T *out = static_cast<T *>(p.out) + row * p.so0 + static_cast<int64_t>(chunk) * 512 * p.so1;
        const int here = static_cast<int>(p.cols) - static_cast<int>(chunk) * 512;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int c = 32 * j + static_cast<int>(lane);
            if (c < here) from_float(mine[c + c / 16], out[c * p.so1]);
        }
    }
    pdl_trigger();
}

int checked(const char *what) {
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), what);
}

// CTAs for `work` of them, as many as are resident at once at most.
template <typename Kernel, typename... Instance>
unsigned resident_grid(Kernel kern, int64_t work, int sm_count, size_t smem) {
    static int per_sm = 0;  // the same on every device of this architecture
    if (per_sm == 0) {
        int n = 0;
        per_sm = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, kThreads, smem) == cudaSuccess && n > 0 ? n : 2;
    }
    const int64_t most = static_cast<int64_t>(sm_count) * per_sm;
    return static_cast<unsigned>(work < 1 ? 1 : work < most ? work : most);
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
    unsigned grid = grid_of(cdiv(rows * cols, kThreads * (words ? 8 * kVec : 4)), sm_count, kAmaxPerSm);
    if (grid > kMostMaxima) grid = kMostMaxima;
    if (words) ST_CUDA_TRY(launch_kernel(amax_kernel<T, true>, grid, kThreads, 0, stream, a, s0, s1, rows, cols, maxima));
    else ST_CUDA_TRY(launch_kernel(amax_kernel<T, false>, grid, kThreads, 0, stream, a, s0, s1, rows, cols, maxima));
    p.maxima = maxima;
    p.n_maxima = static_cast<int>(grid);
    return checked("amax_kernel");
}

template <typename T, bool WIDE>
int launch_columns(const Quantize4Args &p, int64_t quads, int sm_count, cudaStream_t stream) {
    using Tile = ColumnTile<T, WIDE>;
    auto kern = quantize4_columns_kernel<T, WIDE>;
    static_assert(sizeof(Tile) <= 48 * 1024, "shared memory that a kernel has without asking");
    const bool in_words = reinterpret_cast<uintptr_t>(p.a) % 16 == 0 && (p.cols == 1 || p.sa1 * static_cast<int64_t>(sizeof(T)) % 16 == 0);
    const bool words = on16(p.q, p.sq0, p.rows, 1);
    const int64_t work = cdiv(p.rows, 128) * (128 / Tile::kRows) * cdiv(quads, 2);
    const unsigned grid = resident_grid<decltype(kern), T, std::bool_constant<WIDE>>(kern, work, sm_count, sizeof(Tile));
    ST_CUDA_TRY(launch_kernel(kern, grid, kThreads, sizeof(Tile), stream, p, quads, in_words, words));
    return checked("quantize4_columns_kernel");
}

template <typename T, bool WIDE>
int launch_quantize(const Quantize4Args &p, int sm_count, cudaStream_t stream) {
    const int64_t blocks = cdiv(p.cols, WIDE ? 32 : 16), quads = cdiv(blocks, 4), units = quads * (WIDE ? 8 : 4);
    const int64_t padded = cdiv(p.rows, 128) * 128;
    if (p.cols == 1 || p.sa1 == 1) {
        if (on16(p.a, p.sa0, p.rows, sizeof(T))) {
            const bool words = reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.sq0 % 8 == 0);
            const int64_t across = cdiv(units, 32), chunks = padded / 2 * across;
            if (chunks > INT32_MAX) return fail(ST_ERR_UNSUPPORTED, "quantize_fp4: too many blocks");
            auto go = [&](auto kern, auto whole) -> int {
                const unsigned grid = resident_grid<decltype(kern), T, std::bool_constant<WIDE>, decltype(whole)>(kern, cdiv(chunks, kWarps),
                                                                                                                  sm_count, 0);
                ST_CUDA_TRY(launch_kernel(kern, grid, kThreads, 0, stream, p, static_cast<uint32_t>(units), static_cast<uint32_t>(across),
                                          static_cast<uint32_t>(chunks), quads, words));
                return ST_OK;
            };
            if (words && p.cols % 16 == 0) ST_TRY(go(quantize4_rows_kernel<T, WIDE, true>, std::true_type{}));
            else ST_TRY(go(quantize4_rows_kernel<T, WIDE, false>, std::false_type{}));
            return checked("quantize4_rows_kernel");
        }
    } else if (p.sa0 == 1 && p.rows > 1) {
        return launch_columns<T, WIDE>(p, quads, sm_count, stream);
    }
    const bool words = reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.sq0 % 8 == 0);
    auto kern = quantize4_any_kernel<T, WIDE>;
    const unsigned grid =
        resident_grid<decltype(kern), T, std::bool_constant<WIDE>, int>(kern, cdiv(padded * cdiv(units, 32), kWarps), sm_count, 0);
    ST_CUDA_TRY(launch_kernel(kern, grid, kThreads, 0, stream, p, units, quads, words));
    return checked("quantize4_any_kernel");
}

template <typename T>
int launch_typed(Quantize4Args p, float *maxima, int sm_count, cudaStream_t stream) {
    if (p.wide) return launch_quantize<T, true>(p, sm_count, stream);
    if (p.maxima == nullptr) ST_TRY(launch_amax<T>(p, maxima, sm_count, stream));
    return launch_quantize<T, false>(p, sm_count, stream);
}

template <typename T, bool WIDE>
int launch_dequantize(const Dequantize4Args &p, int sm_count, cudaStream_t stream) {
    const int64_t quads = cdiv(cdiv(p.cols, WIDE ? 32 : 16), 4);
    const bool words = p.sq1 == 1 && reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.sq0 % 8 == 0);
    if (words && p.so1 == 1 && on16(p.out, p.so0, p.rows, sizeof(T)) && cdiv(p.rows, 8) * cdiv(p.cols, 256) <= INT32_MAX) {
        const int64_t across = cdiv(p.cols, 256), chunks = cdiv(p.rows, 8) * across;
        auto kern = dequantize4_words_kernel<T, WIDE>;
        const unsigned grid = resident_grid<decltype(kern), T, std::bool_constant<WIDE>>(kern, cdiv(chunks, kWarps), sm_count, 0);
        ST_CUDA_TRY(launch_kernel(kern, grid, kThreads, 0, stream, p, static_cast<uint32_t>(across), static_cast<uint32_t>(chunks), quads));
        return checked("dequantize4_words_kernel");
    }
    const int64_t across = cdiv(p.cols, 512);
    auto kern = dequantize4_any_kernel<T, WIDE>;
    const unsigned grid = resident_grid<decltype(kern), T, std::bool_constant<WIDE>, int>(kern, cdiv(p.rows * across, kWarps), sm_count, 0);
    ST_CUDA_TRY(launch_kernel(kern, grid, kThreads, 0, stream, p, static_cast<uint32_t>(across), p.rows * across, quads, words));
    return checked("dequantize4_any_kernel");
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
    case ST_F32: return p.wide ? launch_dequantize<float, true>(p, sm_count, stream) : launch_dequantize<float, false>(p, sm_count, stream);
    case ST_F16: return p.wide ? launch_dequantize<__half, true>(p, sm_count, stream) : launch_dequantize<__half, false>(p, sm_count, stream);
    default: return p.wide ? launch_dequantize<__nv_bfloat16, true>(p, sm_count, stream) : launch_dequantize<__nv_bfloat16, false>(p, sm_count, stream);
    }
}

}  // namespace st
