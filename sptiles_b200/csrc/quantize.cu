// quantize.cu -- 8-bit blocks with one float32 scale each, as matmul_fp8 reads them.
//
//   scale = max(max|a| / limit, 2^-126)   over a block (limit 448 for e4m3, 57344 for e5m2)
//   q     = fp8(a * (1 / scale))          round to nearest even, saturating
//
// Every step is one IEEE fp32 operation, so the codes are the same on any
// machine that computes them this way.  A NaN or infinity in a block makes
// its scale NaN or infinite, and every product that reads the block NaN.
//
// The input is read once and stays in registers between a block's maximum and
// its conversion.
#include <cuda_runtime.h>

#include <cstdint>
#include <utility>

#include "common.h"
#include "fp8.cuh"

namespace st {
namespace {

constexpr int kTile = 128;

// ---------------------------------------------------------------- 1 x 128 blocks on 16-byte rows
// A warp takes four rows of 256 columns, 8 columns a lane: 2 KB of 16-bit
// input in flight per warp, 16 lanes a block.  The four rows' maxima are
// reduced together, so that each lane ends with one row's maximum and does one
// division pair for it.  Bound by DRAM: 8192 x 8192 bf16 in 35.7 us, 31.0 at
// the copy rate.
constexpr int kRowThreads = 128;

template <typename T, bool E5M2>
__global__ void __launch_bounds__(kRowThreads) quantize_rows_kernel(const QuantizeArgs p, uint32_t chunks) {
    pdl_wait();
    const uint32_t unit = blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
    const uint32_t rg = unit / chunks, chunk = unit - rg * chunks;
    const int64_t row0 = static_cast<int64_t>(rg) * 4;
    if (row0 >= p.rows) return;
    const int lane = threadIdx.x & 31;
    const int col = static_cast<int>(chunk) * 256 + lane * 8, cols = static_cast<int>(p.cols);
    const int here = p.rows - row0 < 4 ? static_cast<int>(p.rows - row0) : 4;
    const bool whole = cols - col >= 8;
    constexpr int kWords = static_cast<int>(sizeof(T) / 2);
    const T *src = static_cast<const T *>(p.a) + row0 * p.sa0 + col;
    uint4 raw[4][kWords];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int w = 0; w < kWords; ++w) raw[i][w] = make_uint4(0, 0, 0, 0);
        if (i < here && whole) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) raw[i][w] = __ldcs(reinterpret_cast<const uint4 *>(src + i * p.sa0) + w);
        } else if (i < here) {
            T *e = reinterpret_cast<T *>(raw[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (col + j < cols) e[j] = src[i * p.sa0 + j];
        }
    }
    float m[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint64_t f[4];
        unpack8(raw[i], f, T{});
        m[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) m[i] = max_abs(m[i], lo2(f[j]), hi2(f[j]));
    }
    const float scale = fp8_scale(max_of_four(m, lane), E5M2 ? 57344.0f : 448.0f);
    const float inverse = __frcp_rn(scale);
    const int mine = (lane >> 2) & 3, block = static_cast<int>(chunk) * 2 + (lane >> 4);
    if ((lane & 3) == 0 && mine < here && block * kTile < cols) p.scale[(row0 + mine) * p.ss0 + block * p.ss1] = scale;
    uint8_t *q = static_cast<uint8_t *>(p.q) + row0 * p.sq0 + col;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float inv = __shfl_sync(0xffffffffu, inverse, (lane & 16) | (i * 4));
        uint64_t f[4];
        unpack8(raw[i], f, T{});
        const uint2 c = to_fp8x8<E5M2>(f, inv);
        if (i >= here) continue;
        if (whole) {
            *reinterpret_cast<uint2 *>(q + i * p.sq0) = c;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (col + j < cols) q[i * p.sq0 + j] = static_cast<uint8_t>((j < 4 ? c.x : c.y) >> (8 * (j % 4)));
        }
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- tiles of 128 columns
// The other blocks, and any stride: a CTA takes 128 columns and 16 * NROWS
// rows, 16 threads of 8 columns across, 16 rows down.  The elements stay as
// they were read and are unpacked twice: at 4 registers for 8 of 16 bits,
// three such CTAs have 96 KB of an SM's reads under way (unpacked, two CTAs
// of 512 threads took 64 us for 8192 x 8192; so 39, and 41 in 128 x 1 blocks).
constexpr int kTileThreads = 256;
constexpr int kDown = kTileThreads / 16;

enum : int { kRowBlocks = 0, kColumnBlocks = 1, kSquareBlocks = 2 };  // 1 x 128, 128 x 1, 128 x 128
// How a thread reads its 8 columns: as 16-byte words (rows of a on 16-byte,
// of q on 8-byte boundaries); one by one, 16 apart, so that neighbouring
// threads read neighbouring elements; the same with any column stride.
enum : int { kWordsAccess = 0, kUnitAccess = 1, kAnyAccess = 2 };

template <typename T, int MODE, int NROWS, int ACCESS>
__global__ void __launch_bounds__(kTileThreads, NROWS == 2 ? 4 : ACCESS == kWordsAccess ? 3 : 2)
    quantize_tiles_kernel(const QuantizeArgs p, uint32_t col_tiles) {
    pdl_wait();
    __shared__ float red[MODE == kColumnBlocks ? kDown * kTile : kTileThreads / 32];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    const uint32_t tile_r = blockIdx.x / col_tiles, tile_c = blockIdx.x - tile_r * col_tiles;
    const int64_t r0 = static_cast<int64_t>(tile_r) * (kDown * NROWS) + ty;
    const int c0 = static_cast<int>(tile_c) * kTile, left = static_cast<int>(p.cols) - c0;  // columns from c0 on
    auto column = [&](int j) { return ACCESS == kWordsAccess ? tx * 8 + j : tx + 16 * j; };
    const T *a = static_cast<const T *>(p.a) + c0 * p.sa1;
    const bool whole = ACCESS == kWordsAccess && tx * 8 + 8 <= left;

    constexpr int kWords = static_cast<int>(sizeof(T) / 2);
    uint4 raw[NROWS][kWords];
#pragma unroll
    for (int i = 0; i < NROWS; ++i) {
        const int64_t r = r0 + kDown * i;
        const T *row = a + r * p.sa0;
#pragma unroll
        for (int k = 0; k < kWords; ++k) raw[i][k] = make_uint4(0, 0, 0, 0);
        if (r >= p.rows) continue;
        if (whole) {
#pragma unroll
            for (int k = 0; k < kWords; ++k) raw[i][k] = __ldcs(reinterpret_cast<const uint4 *>(row + tx * 8) + k);
        } else {
            T *e = reinterpret_cast<T *>(raw[i]);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (column(j) < left) e[j] = row[ACCESS == kAnyAccess ? column(j) * p.sa1 : column(j)];
        }
    }

    const float limit = p.e5m2 ? 57344.0f : 448.0f;
    float inv[MODE == kColumnBlocks ? 8 : NROWS];
    if constexpr (MODE == kRowBlocks) {
#pragma unroll
        for (int i = 0; i < NROWS; ++i) {
            uint64_t x[4];
            unpack8(raw[i], x, T{});
            float m = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) m = max_abs(m, lo2(x[j]), hi2(x[j]));
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
            const float s = fp8_scale(m, limit);
            inv[i] = __frcp_rn(s);
            const int64_t r = r0 + kDown * i;
            if (tx == 0 && r < p.rows) p.scale[r * p.ss0 + tile_c * p.ss1] = s;
        }
    } else if constexpr (MODE == kColumnBlocks) {
        float m[8] = {};
#pragma unroll
        for (int i = 0; i < NROWS; ++i) {
            uint64_t x[4];
            unpack8(raw[i], x, T{});
#pragma unroll
            for (int j = 0; j < 8; ++j) m[j] = max_abs(m[j], j & 1 ? hi2(x[j / 2]) : lo2(x[j / 2]));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) red[ty * kTile + column(j)] = m[j];
        __syncthreads();
        if (threadIdx.x < kTile) {
            float m = 0.0f;
#pragma unroll
            for (int t = 0; t < kDown; t += 2)
                m = max_abs(m, red[t * kTile + threadIdx.x], red[(t + 1) * kTile + threadIdx.x]);
            const float s = fp8_scale(m, limit);
            if (static_cast<int>(threadIdx.x) < left) p.scale[tile_r * p.ss0 + (c0 + static_cast<int>(threadIdx.x)) * p.ss1] = s;
            red[threadIdx.x] = __frcp_rn(s);  // read by the others only after the barrier
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) inv[j] = red[column(j)];
    } else {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < NROWS; ++i) {
            uint64_t x[4];
            unpack8(raw[i], x, T{});
#pragma unroll
            for (int j = 0; j < 4; ++j) m = max_abs(m, lo2(x[j]), hi2(x[j]));
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = max_abs(m, __shfl_xor_sync(0xffffffffu, m, o));
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
        __syncthreads();
        m = 0.0f;
#pragma unroll
        for (int t = 0; t < kTileThreads / 32; t += 2) m = max_abs(m, red[t], red[t + 1]);
        const float s = fp8_scale(m, limit);
        if (threadIdx.x == 0) p.scale[tile_r * p.ss0 + tile_c * p.ss1] = s;
        const float v = __frcp_rn(s);
#pragma unroll
        for (int i = 0; i < NROWS; ++i) inv[i] = v;
    }

    uint8_t *q = static_cast<uint8_t *>(p.q) + c0 * p.sq1;
#pragma unroll
    for (int i = 0; i < NROWS; ++i) {
        const int64_t r = r0 + kDown * i;
        if (r >= p.rows) continue;
        uint64_t x[4], y[4];
        unpack8(raw[i], x, T{});
#pragma unroll
        for (int j = 0; j < 4; ++j)
            y[j] = MODE == kColumnBlocks ? mul2(x[j], pack2(inv[2 * j], inv[2 * j + 1])) : mul2(x[j], pack2(inv[i], inv[i]));
        const uint2 c = p.e5m2 ? to_fp8x8<true>(y, 1.0f) : to_fp8x8<false>(y, 1.0f);
        uint8_t *to = q + r * p.sq0;
        if (whole) {
            *reinterpret_cast<uint2 *>(to + tx * 8) = c;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (column(j) < left)
                    to[ACCESS == kAnyAccess ? column(j) * p.sq1 : column(j)] =
                        static_cast<uint8_t>((j < 4 ? c.x : c.y) >> (8 * (j % 4)));
        }
    }
    pdl_trigger();
}

int checked(const char *what) {
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), what);
}

template <typename T, int MODE, int NROWS>
int launch_tiles(const QuantizeArgs &p, int access, cudaStream_t stream) {
    const int64_t col_tiles = cdiv(p.cols, kTile), grid = cdiv(p.rows, kDown * NROWS) * col_tiles;
    if (grid > INT32_MAX) return fail(ST_ERR_UNSUPPORTED, "quantize_fp8: too many blocks");
    const unsigned g = static_cast<unsigned>(grid);
    const uint32_t ct = static_cast<uint32_t>(col_tiles);
    if (access == kWordsAccess)
        ST_CUDA_TRY(launch_kernel(quantize_tiles_kernel<T, MODE, NROWS, kWordsAccess>, g, kTileThreads, 0, stream, p, ct));
    else if (access == kUnitAccess)
        ST_CUDA_TRY(launch_kernel(quantize_tiles_kernel<T, MODE, NROWS, kUnitAccess>, g, kTileThreads, 0, stream, p, ct));
    else
        ST_CUDA_TRY(launch_kernel(quantize_tiles_kernel<T, MODE, NROWS, kAnyAccess>, g, kTileThreads, 0, stream, p, ct));
    return checked("quantize_tiles_kernel");
}

template <typename T>
int launch_typed(const QuantizeArgs &p, cudaStream_t stream) {
    const bool unit = p.sa1 == 1 && p.sq1 == 1;
    const bool words = unit && reinterpret_cast<uintptr_t>(p.a) % 16 == 0 &&
                       (p.rows == 1 || p.sa0 * static_cast<int64_t>(sizeof(T)) % 16 == 0) &&
                       reinterpret_cast<uintptr_t>(p.q) % 8 == 0 && (p.rows == 1 || p.sq0 % 8 == 0);
    const int access = words ? kWordsAccess : unit ? kUnitAccess : kAnyAccess;
    if (p.block_rows == 1 && words) {
        const int64_t chunks = cdiv(p.cols, 256), units = cdiv(p.rows, 4) * chunks;
        if (units > INT32_MAX) return fail(ST_ERR_UNSUPPORTED, "quantize_fp8: too many blocks");
        const unsigned g = static_cast<unsigned>(cdiv(units, kRowThreads / 32));
        const uint32_t ch = static_cast<uint32_t>(chunks);
        if (p.e5m2) ST_CUDA_TRY(launch_kernel(quantize_rows_kernel<T, true>, g, kRowThreads, 0, stream, p, ch));
        else ST_CUDA_TRY(launch_kernel(quantize_rows_kernel<T, false>, g, kRowThreads, 0, stream, p, ch));
        return checked("quantize_rows_kernel");
    }
    if (p.block_rows == 1) return launch_tiles<T, kRowBlocks, 2>(p, access, stream);
    if (p.block_cols == 1) return launch_tiles<T, kColumnBlocks, 8>(p, access, stream);
    return launch_tiles<T, kSquareBlocks, 8>(p, access, stream);
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
