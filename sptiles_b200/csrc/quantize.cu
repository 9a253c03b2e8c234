// quantize.cu -- 8-bit blocks with one float32 scale each, as matmul_fp8 reads them.
//
//   scale = max(max|a| / limit, 2^-126)   over a block (limit 448 for e4m3, 57344 for e5m2)
//   q     = fp8(a * (1 / scale))          round to nearest even, saturating
//
// Every step is one IEEE fp32 operation, so the codes are the same on any
// machine that computes them this way.  A NaN or infinity in a block makes
// its scale NaN or infinite, and every product that reads the block NaN.
//
// One CTA takes a tile of 128 columns and up to 128 rows: 16 threads of 8
// columns across, 16 rows down, the tile in registers between the maximum
// and the conversion, so that the input is read once.
#include <cuda_runtime.h>

#include <cstdint>
#include <utility>

#include "common.h"
#include "fp8.cuh"

namespace st {
namespace {

constexpr int kThreads = 256;
constexpr int kTile = 128;

template <typename T>
struct Vec8 {
    uint4 w[sizeof(T) / 2];  // 8 elements: one 16-byte word, two for fp32
};

template <typename T>
__device__ __forceinline__ void unpack8(const Vec8<T> &v, float (&f)[8]) {
    const T *e = reinterpret_cast<const T *>(&v);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = to_float(e[j]);
}

enum : int { kRowBlocks = 0, kColumnBlocks = 1, kSquareBlocks = 2 };  // 1 x 128, 128 x 1, 128 x 128

// NROWS rows per thread: 16 * NROWS rows a tile.  VEC: unit column stride
// with rows on 16-byte boundaries of a and 8-byte boundaries of q; otherwise
// a thread's columns are 16 apart, which keeps a warp's loads together.
template <typename T, int MODE, int NROWS, bool VEC>
__global__ void __launch_bounds__(kThreads) quantize_kernel(const QuantizeArgs p) {
    pdl_wait();
    __shared__ uint32_t red[MODE == kColumnBlocks ? 16 * kTile : 16];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const int64_t col_tiles = (p.cols + kTile - 1) / kTile;
    const int64_t tile_r = blockIdx.x / col_tiles, tile_c = blockIdx.x % col_tiles;
    const int64_t r0 = tile_r * (16 * NROWS), c0 = tile_c * kTile;
    const T *a = static_cast<const T *>(p.a);
    auto column = [&](int j) { return c0 + (VEC ? tx * 8 + j : tx + 16 * j); };

    float x[NROWS][8];
    const bool whole = VEC && c0 + tx * 8 + 8 <= p.cols;
    if (whole) {
        Vec8<T> v[NROWS];
#pragma unroll
        for (int i = 0; i < NROWS; ++i) {
            const int64_t r = r0 + ty + 16 * i;
            v[i] = Vec8<T>{};
            if (r < p.rows) {
                const uint4 *src = reinterpret_cast<const uint4 *>(a + r * p.sa0 + c0 + tx * 8);
#pragma unroll
                for (int w = 0; w < static_cast<int>(sizeof(T) / 2); ++w) v[i].w[w] = __ldcs(src + w);
            }
        }
#pragma unroll
        for (int i = 0; i < NROWS; ++i) unpack8(v[i], x[i]);
    } else {
#pragma unroll
        for (int i = 0; i < NROWS; ++i) {
            const int64_t r = r0 + ty + 16 * i;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t c = column(j);
                x[i][j] = r < p.rows && c < p.cols ? to_float(a[r * p.sa0 + c * p.sa1]) : 0.0f;
            }
        }
    }

    // maxima as bit patterns of |x|: order preserving, and a NaN wins
    const float limit = p.e5m2 ? 57344.0f : 448.0f;
    float inv[MODE == kColumnBlocks ? 8 : NROWS];
    if constexpr (MODE == kRowBlocks) {
#pragma unroll
        for (int i = 0; i < NROWS; ++i) {
            uint32_t m = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, abs_bits(x[i][j]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float s = fp8_scale(m, limit);
            inv[i] = __fdiv_rn(1.0f, s);
            const int64_t r = r0 + ty + 16 * i;
            if (tx == 0 && r < p.rows) p.scale[r * p.ss0 + tile_c * p.ss1] = s;
        }
    } else if constexpr (MODE == kColumnBlocks) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < NROWS; ++i) m = max(m, abs_bits(x[i][j]));
            red[ty * kTile + static_cast<int>(column(j) - c0)] = m;
        }
        __syncthreads();
        if (threadIdx.x < kTile) {
            uint32_t m = 0;
#pragma unroll
            for (int t = 0; t < 16; ++t) m = max(m, red[t * kTile + threadIdx.x]);
            const float s = fp8_scale(m, limit);
            const int64_t c = c0 + threadIdx.x;
            if (c < p.cols) p.scale[tile_r * p.ss0 + c * p.ss1] = s;
            red[threadIdx.x] = __float_as_uint(__fdiv_rn(1.0f, s));
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) inv[j] = __uint_as_float(red[static_cast<int>(column(j) - c0)]);
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < NROWS; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) m = max(m, abs_bits(x[i][j]));
        m = __reduce_max_sync(0xffffffffu, m);
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        m = 0;
#pragma unroll
        for (int t = 0; t < kThreads / 32; ++t) m = max(m, red[t]);
        const float s = fp8_scale(m, limit);
        if (threadIdx.x == 0) p.scale[tile_r * p.ss0 + tile_c * p.ss1] = s;
        const float v = __fdiv_rn(1.0f, s);
#pragma unroll
        for (int i = 0; i < NROWS; ++i) inv[i] = v;
    }

    uint8_t *q = static_cast<uint8_t *>(p.q);
#pragma unroll
    for (int i = 0; i < NROWS; ++i) {
        const int64_t r = r0 + ty + 16 * i;
        if (r >= p.rows) continue;
        uint32_t w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (MODE == kColumnBlocks) y[j] = __fmul_rn(x[i][4 * h + j], inv[4 * h + j]);
                else y[j] = __fmul_rn(x[i][4 * h + j], inv[i]);
            }
            w[h] = to_fp8x4(y[0], y[1], y[2], y[3], p.e5m2);
        }
        if (whole) {
            *reinterpret_cast<uint2 *>(q + r * p.sq0 + c0 + tx * 8) = make_uint2(w[0], w[1]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int64_t c = column(j);
                if (c < p.cols) q[r * p.sq0 + c * p.sq1] = static_cast<uint8_t>(w[j / 4] >> (8 * (j % 4)));
            }
        }
    }
    pdl_trigger();
}

template <typename T, int MODE, int NROWS>
int launch_mode(const QuantizeArgs &p, bool vec, cudaStream_t stream) {
    const int64_t grid = cdiv(p.rows, 16 * NROWS) * cdiv(p.cols, kTile);
    if (grid > INT32_MAX) return fail(ST_ERR_UNSUPPORTED, "quantize_fp8: too many blocks");
    const unsigned g = static_cast<unsigned>(grid);
    if (vec) ST_CUDA_TRY(launch_kernel(quantize_kernel<T, MODE, NROWS, true>, g, kThreads, 0, stream, p));
    else ST_CUDA_TRY(launch_kernel(quantize_kernel<T, MODE, NROWS, false>, g, kThreads, 0, stream, p));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "quantize_kernel");
}

template <typename T>
int launch_typed(const QuantizeArgs &p, cudaStream_t stream) {
    const bool vec = p.sa1 == 1 && p.sq1 == 1 && reinterpret_cast<uintptr_t>(p.a) % 16 == 0 &&
                     (p.rows == 1 || p.sa0 * static_cast<int64_t>(sizeof(T)) % 16 == 0) &&
                     reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.sq0 % 8 == 0);
    if (p.block_rows == 1) {
        // row blocks need no common tile: few rows stay spread over many CTAs
        if (p.rows <= 1024) return launch_mode<T, kRowBlocks, 1>(p, vec, stream);
        return launch_mode<T, kRowBlocks, 4>(p, vec, stream);
    }
    if (p.block_cols == 1) return launch_mode<T, kColumnBlocks, 8>(p, vec, stream);
    return launch_mode<T, kSquareBlocks, 8>(p, vec, stream);
}

}  // namespace

int launch_quantize_fp8(const QuantizeArgs &args, cudaStream_t stream) {
    if (args.rows == 0 || args.cols == 0) return ST_OK;
    QuantizeArgs p = args;
    // an input stored column by column is the transposed problem
    if (p.cols > 1 && p.sa1 != 1 && p.sa0 == 1) {
        std::swap(p.rows, p.cols);
        std::swap(p.sa0, p.sa1);
        std::swap(p.sq0, p.sq1);
        std::swap(p.ss0, p.ss1);
        std::swap(p.block_rows, p.block_cols);
    }
    if (p.cols == 1) p.sa1 = p.sq1 = 1;  // one column: its stride is never used
    switch (p.a_dtype) {
    case ST_F32: return launch_typed<float>(p, stream);
    case ST_F16: return launch_typed<__half>(p, stream);
    default: return launch_typed<__nv_bfloat16>(p, stream);
    }
}

}  // namespace st
