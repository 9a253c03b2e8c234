// gemm_fp8.cu -- matrix product of 8-bit operands with a scale for each
// block of 128 along the contraction.
//
//   C[m, n] = sum_b sa[m, b] * sb[b, n] * sum_{k in block b} A[m, k] * B[k, n]  (+ bias[n])
//
// A and B are e4m3 or e5m2, sa and sb float32.  The inner sum of a block is
// one K = 128 chain of tcgen05.mma (kind::f8f6f4) into a fresh TMEM
// accumulator; the epilogue warps read each block's accumulator, multiply by
// the block's two scales and add onto running sums in fp32 registers, while
// the tensor core works on the next blocks in the other TMEM accumulators.
// So the sum over blocks is a plain fp32 sum; the product of the two scales
// is one too, and has to stay within fp32's normal range.
//
//   warp 0      TMA producer: one 128-byte-swizzled box of each operand per block
//   warp 1      MMA issuer (owns the TMEM allocation)
//   warps 2..   scaling (4 warps, 8 from 64 columns on): TMEM -> registers,
//               scale, add; then bias and the store
//   last warp   the blocks' scales, ahead of their use, into shared memory
//
// The kernel knows a row operand (128 rows a tile, the MMA's M) and a column
// operand (BN columns, the MMA's N).  With up to 64 tokens the weights may
// become the row operand and the tokens the columns, so that a tile reads 128
// rows of weights against 16 to 64 tokens and nothing is padded to 128
// tokens; that is done where it is estimated to be faster (57 x 4109 x 4001
// keeps its tokens as rows, 71 of a tile's 128 empty).  When tiles alone would leave SMs idle, a cluster of up to 8 CTAs
// splits the blocks of one tile and adds its parts in a fixed order through
// distributed shared memory.  Bound by the weights' bytes with few tokens:
// 1 x 8192 x 8192 in 15.0 us (10.3 at the copy rate; about 5 us are launch,
// the first load's latency, the cluster's exchange and the store, whatever
// the size), 57 x 4109 x 4001 in 14.1, 1024^3 in 10.8 a call and 7.2 in a
// replayed graph.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.h"
#include "fp8.cuh"
#include "sm100.cuh"
#include "tensor_map.h"

namespace st {
namespace {

constexpr int kTileRows = 128;
constexpr int kBlockK = 128;  // bytes = elements: one scale block, one 128-byte swizzle span
constexpr int kMmaK = 32;
constexpr int kBarBytes = 1024;

struct Fp8Params {
    int rows, cols, k_blocks;  // row operand x column operand
    int tiles_r, tiles_c, split;
    const float *rs, *cs;            // scales of the row and the column operand
    int64_t rs_i, rs_b, cs_i, cs_b;  // strides: per index (row / column or their block of 128), per K block
    int rs_shift, cs_shift;          // 7: one scale for 128 rows / columns
    void *c;
    int64_t c_r, c_c;  // strides of C along the row and the column operand; one of them is 1
    int c_dtype;
    const void *bias;
    int bias_dtype;
    int bias_on_rows;  // B is the row operand: C's rows, contiguous, run along the tile's columns
    int staged;  // CTA pairs: C leaves by TMA stores
    uint32_t idesc;
    int *err;
    unsigned long long timeout_ns;
};

__device__ __forceinline__ uint32_t pack_16(float a, float b, int dtype) {
    if (dtype == ST_F16) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Load 8, 16 or 32 consecutive f32 columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_load_8(uint32_t taddr, uint32_t *r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void tmem_load_16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_load_x32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
template <int N>
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint32_t *r) {
    static_assert(N == 8 || N == 16 || N == 32, "one load");
    if constexpr (N == 8) tmem_load_8(taddr, r);
    else if constexpr (N == 16) tmem_load_16(taddr, r);
    else tmem_load_x32(taddr, r);
}

// Wait for every load so far; the registers pass through, so that nothing
// reads them before it.
template <int N>
__device__ __forceinline__ void tmem_loaded(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]));
#pragma unroll
    for (int i = 8; i < N; i += 8)
        asm volatile("" : "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]),
                          "+r"(r[i + 6]), "+r"(r[i + 7]));
}

// The four MMAs of a block, by one elected lane: descriptors of its first
// 32 elements along K, each next one a fixed step further in the address
// field (shared memory ends below 2^18, so the field does not overflow).
template <bool R_MN, bool C_MN, bool PAIR>
__device__ __forceinline__ void issue_block(uint32_t d_tmem, uint64_t dr, uint64_t dc, uint32_t idesc) {
    // K-major: 32 bytes further along the 128-byte span; otherwise 32 K rows of 128 bytes
    constexpr uint64_t kStepR = (R_MN ? kMmaK * 128 : kMmaK) >> 4, kStepC = (C_MN ? kMmaK * 128 : kMmaK) >> 4;
#pragma unroll
    for (int ks = 0; ks < kBlockK / kMmaK; ++ks) {
        if constexpr (PAIR) tc_mma_f8_pair(d_tmem, dr + ks * kStepR, dc + ks * kStepC, idesc, ks != 0 ? 1u : 0u);
        else tc_mma_f8(d_tmem, dr + ks * kStepR, dc + ks * kStepC, idesc, ks != 0 ? 1u : 0u);
    }
}

__device__ __forceinline__ void copy_4_async(uint32_t dst, const float *src, bool valid) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(valid ? 4 : 0) : "memory");
}

// One warp brings the scales of a tile's blocks, ROWS for its rows and COLS
// for its columns (CVEC), or one for each 128 columns, into a ring of shared
// memory ahead of their use: a load by the scaling warps themselves would
// cost them its latency in every block.  A slot holds the scales of kBatch
// blocks, so that a slot's two barriers are passed once in kBatch blocks.
constexpr int kBatch = 4;

template <int ROWS, int COLS, bool CVEC, int DEPTH>
struct ScaleRing {
    static constexpr int kDepth = DEPTH;
    static constexpr int kCols = CVEC ? COLS : (COLS + 127) / 128;
    static constexpr int kBlock = ROWS + (kCols + 3) / 4 * 4;  // floats; 16-byte aligned columns
    static constexpr int kBytes = DEPTH * kBatch * kBlock * 4;
    static constexpr int kBars = 2 * DEPTH;
    float *slots;
    uint32_t bar0;  // full[DEPTH], empty[DEPTH]
    __device__ __forceinline__ uint32_t full(int d) const { return bar0 + 8u * d; }
    __device__ __forceinline__ uint32_t empty(int d) const { return bar0 + 8u * (DEPTH + d); }
    __device__ __forceinline__ void init(int readers) const {
        for (int d = 0; d < DEPTH; ++d) {
            mbar_init(full(d), 32);
            mbar_init(empty(d), readers);
        }
    }
    __device__ __forceinline__ const float *rows(int d, int i) const { return slots + (d * kBatch + i) * kBlock; }
    __device__ __forceinline__ const float *cols(int d, int i) const { return rows(d, i) + ROWS; }
    // The scales of blocks b0, b0 + step, ... (count of them) of the tile at
    // row r0, column c0; false after an abort.
    __device__ __forceinline__ bool load(const Fp8Params &p, int r0, int c0, int b0, int step, int count, int lane, int &d,
                                         uint32_t &ph, const volatile int *abort_flag) const {
        const float *src_r[ROWS / 32], *src_c[(kCols + 31) / 32];
        bool ok_r[ROWS / 32], ok_c[(kCols + 31) / 32];
#pragma unroll
        for (int i = 0; i < ROWS / 32; ++i) {
            const int r = r0 + lane + 32 * i;
            ok_r[i] = r < p.rows;
            src_r[i] = p.rs + static_cast<int64_t>(ok_r[i] ? r >> p.rs_shift : 0) * p.rs_i;
        }
#pragma unroll
        for (int i = 0; i < (kCols + 31) / 32; ++i) {
            const int j = lane + 32 * i, c = c0 + (CVEC ? j : 128 * j);
            ok_c[i] = j < kCols && c < p.cols;
            src_c[i] = p.cs + static_cast<int64_t>(ok_c[i] ? c >> p.cs_shift : 0) * p.cs_i;
        }
        for (int done = 0; done < count; done += kBatch) {
            if (!__all_sync(0xffffffffu, mbar_wait(empty(d), ph ^ 1u, abort_flag, p.timeout_ns))) return false;
            const int n = count - done < kBatch ? count - done : kBatch;
            for (int k = 0; k < n; ++k) {
                const int b = b0 + (done + k) * step;
                const uint32_t to_r = smem_addr(rows(d, k)) + 4u * lane, to_c = to_r + 4u * ROWS;
#pragma unroll
                for (int i = 0; i < ROWS / 32; ++i) copy_4_async(to_r + 128u * i, src_r[i] + b * p.rs_b, ok_r[i]);
#pragma unroll
                for (int i = 0; i < (kCols + 31) / 32; ++i)
                    if (lane + 32 * i < kCols) copy_4_async(to_c + 128u * i, src_c[i] + b * p.cs_b, ok_c[i]);
            }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full(d)) : "memory");
            if (++d == DEPTH) {
                d = 0;
                ph ^= 1u;
            }
        }
        return true;
    }
};

// What a scaling warp carries from tile to tile: the next accumulator and ring slot.
struct ScalePosition {
    int a = 0, d = 0;
    uint32_t aph = 0, dph = 0;
};

// acc += the scaled sums of n blocks of a tile, for one row (TMEM lane) and
// COLS columns from accumulator column t on (accumulator a lies a * STRIDE
// further).  A warp passes every block, so a block's serial latency counts:
// STEP columns are added while the next STEP are read, and the first ones of
// the next block are asked for before the last ones of this block are added.
// The sums are added one by one: a packed multiply-add of two needs its
// operands in register pairs, and the moves that make them cost more than it
// saves (eight warps reading and adding 128 columns each: 292 cycles, packed
// 445).  released(a): accumulator a has been read.
template <int COLS, int STEP, bool CVEC, int ACCS, int STRIDE, typename Ring, typename Full, typename Released>
__device__ __forceinline__ bool scale_blocks(float (&acc)[COLS], int n, uint32_t t, int row, int col, const Ring &ring,
                                             ScalePosition &at, Full tfull, Released released, int lane,
                                             const volatile int *abort_flag, uint64_t limit_ns) {
    constexpr int kSteps = COLS / STEP;
    static_assert(kSteps % 2 == 0, "the two buffers keep their order from block to block");
    uint32_t v[2][STEP];
    auto arrived = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit_ns));
    };
    if (!arrived(tfull(at.a), at.aph)) return false;
    tc_fence_after_sync();
    tmem_load<STEP>(t + static_cast<uint32_t>(at.a * STRIDE), v[0]);
    for (int b = 0; b < n; ++b) {
        const int k = b % kBatch;
        if (k == 0 && !arrived(ring.full(at.d), at.dph)) {
            tmem_loaded<STEP>(v[0]);  // the load under way lands before its registers serve anything else
            return false;
        }
        const float *cols = ring.cols(at.d, k) + col;
        const float r_scale = ring.rows(at.d, k)[row];
        const float both = CVEC ? r_scale : r_scale * cols[0];
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            uint32_t *x = v[j & 1];
            // CVEC: the step's scales while its columns are on their way
            uint64_t scales[CVEC ? STEP / 2 : 1];
            if constexpr (CVEC) {
#pragma unroll
                for (int i = 0; i < STEP; i += 4) {
                    const float4 c = *reinterpret_cast<const float4 *>(cols + j * STEP + i);
                    scales[i / 2] = mul2(pack2(both, both), pack2(c.x, c.y));
                    scales[i / 2 + 1] = mul2(pack2(both, both), pack2(c.z, c.w));
                }
            }
            tmem_loaded<STEP>(x);
            if (j + 1 < kSteps) {
                tmem_load<STEP>(t + static_cast<uint32_t>(at.a * STRIDE + (j + 1) * STEP), v[(j + 1) & 1]);
            } else {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) released(at.a);
                if (++at.a == ACCS) {
                    at.a = 0;
                    at.aph ^= 1u;
                }
                if (b + 1 < n) {
                    if (!arrived(tfull(at.a), at.aph)) return false;
                    tc_fence_after_sync();
                    tmem_load<STEP>(t + static_cast<uint32_t>(at.a * STRIDE), v[0]);
                }
            }
            float *s = acc + j * STEP;
#pragma unroll
            for (int i = 0; i < STEP; ++i)
                s[i] = __fmaf_rn(__uint_as_float(x[i]), CVEC ? (i & 1 ? hi2(scales[i / 2]) : lo2(scales[i / 2])) : both, s[i]);
        }
        if (k == kBatch - 1 || b + 1 == n) {
            __syncwarp();
            if (lane == 0) mbar_arrive(ring.empty(at.d));
            if (++at.d == Ring::kDepth) {
                at.d = 0;
                at.dph ^= 1u;
            }
        }
    }
    return true;
}

// Load 32 columns of 16 TMEM lanes: lane l gets, for each 8 columns, columns
// 2 (l % 4) and + 1 of rows l / 4 and l / 4 + 8.
__device__ __forceinline__ void tmem_load_16x32(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.16x256b.x4.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// scale_blocks for scales that differ from column to column, with each
// lane on 4 rows (l / 4 + 8 q) and every fourth pair of columns instead of
// one row and all columns: then a lane needs a quarter of the column scales.
// (A 16-byte shared-memory read that all lanes share still takes four
// cycles: one row a lane, 8 warps reading 128 scales each kept shared memory
// busy for 1024 cycles a block beside the MMAs' 512, and a block took 1480.)
// Element (row l / 4 + 8 q, column 8 c + 2 (l % 4) + i) is acc[8 c + 2 q + i].
template <int COLS, int ACCS, int STRIDE, typename Ring, typename Full, typename Released>
__device__ __forceinline__ bool scale_blocks_by_column(float (&acc)[COLS], int n, uint32_t t, int row0, int col, const Ring &ring,
                                                       ScalePosition &at, Full tfull, Released released, int lane,
                                                       const volatile int *abort_flag, uint64_t limit_ns) {
    constexpr int kSteps = COLS / 32;
    static_assert(kSteps % 2 == 0, "the two buffers keep their order from block to block");
    uint32_t v[2][32];  // 16 lanes, then the other 16
    auto arrived = [&](uint32_t bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit_ns));
    };
    auto ask = [&](uint32_t from, uint32_t *to) {
        tmem_load_16x32(from, to);
        tmem_load_16x32(from + (16u << 16), to + 16);
    };
    if (!arrived(tfull(at.a), at.aph)) return false;
    tc_fence_after_sync();
    ask(t + static_cast<uint32_t>(at.a * STRIDE), v[0]);
    for (int b = 0; b < n; ++b) {
        const int k = b % kBatch;
        if (k == 0 && !arrived(ring.full(at.d), at.dph)) {
            tmem_loaded<32>(v[0]);  // as in scale_blocks
            return false;
        }
        const float2 *cols = reinterpret_cast<const float2 *>(ring.cols(at.d, k) + col) + (lane & 3);
        const float *rows = ring.rows(at.d, k) + row0 + (lane >> 2);
        uint64_t r[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) r[q] = pack2(rows[8 * q], rows[8 * q]);
#pragma unroll
        for (int j = 0; j < kSteps; ++j) {
            uint32_t *x = v[j & 1];
            tmem_loaded<32>(x);
            if (j + 1 < kSteps) {
                ask(t + static_cast<uint32_t>(at.a * STRIDE + (j + 1) * 32), v[(j + 1) & 1]);
            } else {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) released(at.a);
                if (++at.a == ACCS) {
                    at.a = 0;
                    at.aph ^= 1u;
                }
                if (b + 1 < n) {
                    if (!arrived(tfull(at.a), at.aph)) return false;
                    tc_fence_after_sync();
                    ask(t + static_cast<uint32_t>(at.a * STRIDE), v[0]);
                }
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // 8 columns
                const float2 pair = cols[4 * (4 * j + c)];
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const uint64_t scale = mul2(r[q], pack2(pair.x, pair.y));
                    const uint32_t *in = x + (q >> 1) * 16 + 4 * c + 2 * (q & 1);
                    float *s = acc + 8 * (4 * j + c) + 2 * q;
                    s[0] = __fmaf_rn(__uint_as_float(in[0]), lo2(scale), s[0]);
                    s[1] = __fmaf_rn(__uint_as_float(in[1]), hi2(scale), s[1]);
                }
            }
        }
        if (k == kBatch - 1 || b + 1 == n) {
            __syncwarp();
            if (lane == 0) mbar_arrive(ring.empty(at.d));
            if (++at.d == Ring::kDepth) {
                at.d = 0;
                at.dph ^= 1u;
            }
        }
    }
    return true;
}

// One scaling warp on its way out (st_check_device_wait): its accumulator is
// there, so its first columns are being read, and the block's scales never
// come.  It waits for the read, frees its TMEM and returns.
__device__ float g_checked_sum;  // so that what is read has a use

template <bool BY_COLUMN>
__global__ void __launch_bounds__(32) fp8_wait_check_kernel(uint64_t limit_ns, int *err) {
    constexpr int kCols = BY_COLUMN ? 128 : 16;
    using Ring = ScaleRing<kTileRows, kCols, true, 2>;
    __shared__ __align__(16) float slots[Ring::kBytes / 4];
    __shared__ __align__(8) uint64_t bars[1 + Ring::kBars];
    __shared__ uint32_t tmem_slot;
    __shared__ int abort_flag;
    const int lane = static_cast<int>(threadIdx.x);
    const uint32_t accumulated = smem_addr(bars);
    const Ring ring{slots, accumulated + 8u};
    if (lane == 0) {
        mbar_init(accumulated, 1);
        ring.init(1);
        abort_flag = 0;
        fence_barrier_init();
        mbar_arrive(accumulated);
    }
    __syncwarp();
    tmem_alloc(smem_addr(&tmem_slot), 128);
    tmem_relinquish();
    __syncwarp();
    const uint32_t t = *static_cast<volatile uint32_t *>(&tmem_slot);
    float acc[kCols];
#pragma unroll
    for (int j = 0; j < kCols; ++j) {
        acc[j] = 0.0f;
        asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(t + static_cast<uint32_t>(j)), "r"(0) : "memory");
    }
    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
    ScalePosition at;
    auto full = [&](int) { return accumulated; };
    auto released = [](int) {};
    bool ok;
    if constexpr (BY_COLUMN)
        ok = scale_blocks_by_column<kCols, 1, kCols>(acc, 1, t, 0, 0, ring, at, full, released, lane, &abort_flag, limit_ns);
    else
        ok = scale_blocks<kCols, 8, true, 1, kCols>(acc, 1, t, lane, 0, ring, at, full, released, lane, &abort_flag, limit_ns);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < kCols; ++j) sum += acc[j];
    if (ok) g_checked_sum = sum;
    if (!ok && lane == 0) {
        abort_flag = 1;
        atomicExch(err, kDevAbortGemmEpilogue);
    }
    __syncwarp();
    tmem_dealloc(t, 128);
}

__device__ __forceinline__ void copies_done() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// ---------------------------------------------------------------- one CTA, 128 x BN tiles

template <int BN, bool CVEC>
struct Fp8Cfg {
    // warps 0 TMA, 1 MMA, 2.. scaling, the last one scales; two scaling warps
    // share a quarter of the lanes where a tile has the columns for both
    static constexpr int kScaleWarps = BN >= 64 ? 8 : 4;
    static constexpr int kWarpCols = BN / (kScaleWarps / 4);
    static constexpr int kThreads = 32 * (3 + kScaleWarps);
    static constexpr int kRowBytes = kTileRows * kBlockK;
    static constexpr int kColBytes = BN * kBlockK;
    static constexpr int kStageBytes = kRowBytes + kColBytes;
    // Stage and accumulator of a block have one index: the commit that hands
    // over the accumulator frees the stage as well.  BN 128 fills an SM's
    // TMEM (4 x 128 columns) alone; narrower tiles leave room for two CTAs.
    static constexpr int kStages = BN >= 64 ? 4 : 5;
    static constexpr int kTmemCols = BN == 16 ? 128 : BN == 32 ? 256 : kStages * BN;  // powers of two
    static_assert(kStages * BN <= kTmemCols, "the accumulators fit");
    using Ring = ScaleRing<kTileRows, BN, CVEC, 2>;
    static constexpr int kSmemBytes = kStages * kStageBytes + kBarBytes + Ring::kBytes + 1024;
    static_assert(kSmemBytes <= (BN == 128 ? 232448 : 115712), "shared memory of one (two) CTAs per SM");
    static_assert(kStages * kStageBytes >= kTileRows * (BN + 4 * 8) * 4, "the ring holds eight parts' sums of its columns");
};

// Thread `first` of THREADS: its share of 128 rows x `own` columns (a power
// of two, 4 at least), added over the parts of sums [part][row][own + 4].
// By rows, the same 4 columns of every (4 THREADS / own)th row; else every
// (THREADS / 128)th 4 columns of one row.
template <typename T, int THREADS>
__device__ __forceinline__ void store_sums(const Fp8Params &p, const float4 *sums, int first, int own, int own_shift,
                                           int parts, int r0, int col0) {
    const int quads = own / 4, pitch = own / 4 + 1;
    const bool by_rows = !p.bias_on_rows;  // not c_c == 1: a C of one row may have unit strides both ways
    const int quad0 = by_rows ? first & (quads - 1) : first >> 7, r_first = by_rows ? first >> (own_shift - 2) : first & 127;
    const int dr = by_rows ? 4 * THREADS / own : 0, dq = by_rows ? 0 : THREADS / 128;
    T *c = static_cast<T *>(p.c) + (r0 + r_first) * p.c_r + (col0 + 4 * quad0) * p.c_c;
    const int64_t dc = by_rows ? dr * p.c_r : 4 * dq * p.c_c;
    const int left = p.cols - col0 - 4 * quad0;  // columns from this thread's first on
    const bool four = by_rows && left >= 4 && reinterpret_cast<uintptr_t>(p.c) % (4 * sizeof(T)) == 0 && p.c_r % 4 == 0 &&
                      col0 % 4 == 0;
    // one bias for each column of a quad, or one for the row
    float add[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.bias != nullptr) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int i = p.bias_on_rows ? r0 + r_first : col0 + 4 * quad0 + k;
            if (i < (p.bias_on_rows ? p.rows : p.cols)) add[k] = load_any(p.bias, p.bias_dtype, i);
        }
    }
#pragma unroll 2
    for (int i = 0;; ++i, c += dc) {
        const int r = r_first + i * dr, quad = quad0 + i * dq;
        if (r >= kTileRows || quad >= quads || r0 + r >= p.rows) break;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int q = 0; q < parts; ++q) {
            const float4 x = sums[(q * kTileRows + r) * pitch + quad];
            v.x += x.x;
            v.y += x.y;
            v.z += x.z;
            v.w += x.w;
        }
        if (p.bias != nullptr) {
            v.x += add[0];
            v.y += add[1];
            v.z += add[2];
            v.w += add[3];
        }
        T o[4];
        from_float(v.x, o[0]);
        from_float(v.y, o[1]);
        from_float(v.z, o[2]);
        from_float(v.w, o[3]);
        if (four) {
            struct alignas(4 * sizeof(T)) Four {
                T v[4];
            };
            *reinterpret_cast<Four *>(c) = Four{{o[0], o[1], o[2], o[3]}};
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (k < left - 4 * i * dq) c[k * p.c_c] = o[k];
        }
    }
}

// R_MN / C_MN: the operand is stored with its rows (columns) contiguous
// instead of K.  CVEC: the column scale differs inside the tile.
template <int BN, bool R_MN, bool C_MN, bool CVEC>
__global__ void __launch_bounds__(Fp8Cfg<BN, CVEC>::kThreads, BN == 128 ? 1 : 2)
    gemm_fp8_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ CUtensorMap tmap_c,
                    const Fp8Params p) {
    using Cfg = Fp8Cfg<BN, CVEC>;
    using Ring = typename Cfg::Ring;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Cfg::kStages * Cfg::kStageBytes);
    constexpr int kBars = 3 * Cfg::kStages + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars + Ring::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };                        // loads landed
    auto done_bar = [&](int s) { return bar0 + 8u * (Cfg::kStages + s); };       // MMAs done: stage free, accumulator full
    auto empty_bar = [&](int s) { return bar0 + 8u * (2 * Cfg::kStages + s); };  // accumulator read
    const uint32_t drain_bar = bar0 + 8u * (kBars - 1);
    const Ring ring{reinterpret_cast<float *>(smem + Cfg::kStages * Cfg::kStageBytes + kBarBytes), bar0 + 8u * kBars};

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(done_bar(s), 1);
            mbar_init(empty_bar(s), Cfg::kScaleWarps);
        }
        mbar_init(drain_bar, 1);
        ring.init(Cfg::kScaleWarps);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_map(&tmap_r);
        tma_prefetch_map(&tmap_c);
    }
    if (warp == 1) {
        tmem_alloc(smem_addr(tmem_slot), Cfg::kTmemCols);
        tmem_relinquish();
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    pdl_begin();  // nothing above touches global memory

    const int split = p.split;
    const int part = split > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int tile = static_cast<int>(blockIdx.x) / split;
    // neighbouring CTAs walk the row tiles of one column tile
    const int r0 = (tile % p.tiles_r) * kTileRows;
    const int c0 = (tile / p.tiles_r) * BN;
    // blocks part, part + split, ...: a cluster's loads of a row lie next to each other
    const int blocks = (p.k_blocks - part + split - 1) / split;

    // scaling warps: TMEM lane = row of the tile
    constexpr int kWarpCols = Cfg::kWarpCols;
    const int g = warp & 3, col_in_tile = ((warp - 2) >> 2) * kWarpCols;
    const int row_in_tile = g * 32 + lane;
    float acc[kWarpCols];

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            // rows that one column tile reads pass through L2 once
            const uint64_t pol = l2_policy_evict_last(), row_pol = p.tiles_c > 1 ? pol : l2_policy_evict_first();
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int b = part; b < p.k_blocks; b += split, ++issued) {
                if (!mbar_wait(done_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                    ok = false;
                    break;
                }
                mbar_arrive_expect_tx(full_bar(s), Cfg::kStageBytes);
                const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes);
                const uint32_t sc = sr + Cfg::kRowBytes;
                const int k0 = b * kBlockK;
                if constexpr (R_MN) tma_load_2d(sr, &tmap_r, full_bar(s), r0, k0, row_pol);
                else tma_load_2d(sr, &tmap_r, full_bar(s), k0, r0, row_pol);
                if constexpr (C_MN) tma_load_2d(sc, &tmap_c, full_bar(s), c0, k0, pol);
                else tma_load_2d(sc, &tmap_c, full_bar(s), k0, c0, pol);
                if (++s == Cfg::kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
            if (!ok) {
                *abort_flag = 1;
                atomicExch(p.err, kDevAbortGemmProducer);
            }
            drain_ring(issued, Cfg::kStages, full_bar, p.timeout_ns);
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        const uint64_t dr0 = smem_desc_sw128(smem_addr(smem), R_MN ? 128 * 128 : 16, 1024);
        const uint64_t dc0 = smem_desc_sw128(smem_addr(smem) + Cfg::kRowBytes, C_MN ? 128 * 128 : 16, 1024);
        for (int b = 0; b < blocks; ++b) {
            const bool ready = mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns) &&
                               mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns);
            if (!__all_sync(0xffffffffu, ready)) {
                ok = false;
                break;
            }
            tc_fence_after_sync();
            if (elect_one()) {
                const uint64_t step = static_cast<uint64_t>(s) * (Cfg::kStageBytes >> 4);
                issue_block<R_MN, C_MN, false>(tmem_base + static_cast<uint32_t>(s * BN), dr0 + step, dc0 + step, p.idesc);
                tc_commit(done_bar(s));
            }
            __syncwarp();
            if (++s == Cfg::kStages) {
                s = 0;
                ph ^= 1u;
            }
        }
        if (!ok) {
            *abort_flag = 1;
            atomicExch(p.err, kDevAbortGemmMma);
        }
        if (elect_one()) tc_commit(drain_bar);
        __syncwarp();
        drain_ring(1, 1, [&](int) { return drain_bar; }, p.timeout_ns);  // the MMAs read shared memory and write TMEM
    } else if (warp == 2 + Cfg::kScaleWarps) {
        // ------------------------------------------------ scales
        int d = 0;
        uint32_t dph = 0;
        if (!ring.load(p, r0, c0, part, split, blocks, lane, d, dph, abort_flag)) *abort_flag = 1;
        copies_done();
    } else {
        // ------------------------------------------------ scaling
#pragma unroll
        for (int j = 0; j < kWarpCols; ++j) acc[j] = 0.0f;
        ScalePosition at;
        const bool ok = scale_blocks<kWarpCols, (kWarpCols >= 64 ? (CVEC ? 16 : 32) : BN == 32 ? 16 : 8), CVEC, Cfg::kStages, BN>(
            acc, blocks, tmem_base + (static_cast<uint32_t>(g * 32) << 16) + static_cast<uint32_t>(col_in_tile), row_in_tile,
            CVEC ? col_in_tile : 0, ring, at, done_bar,
            [&](int a) { mbar_arrive_relaxed(empty_bar(a)); }, lane, abort_flag, p.timeout_ns);
        if (!ok) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(p.err, kDevAbortGemmEpilogue);
        }
    }

    // ------------------------------------------------ C
    const bool scaler = warp >= 2 && warp < 2 + Cfg::kScaleWarps;
    const int es = p.c_dtype == ST_F32 ? 4 : 2;
    const bool wide = split == 1 && p.c_c == 1 && p.cols - c0 >= BN && p.bias == nullptr &&
                      (reinterpret_cast<uintptr_t>(p.c) & 15u) == 0 && (p.c_r * es) % 16 == 0;
    if (wide) {  // whole 16-byte pieces of each row, straight from registers
        const int row = r0 + row_in_tile;
        if (scaler && row < p.rows) {
            uint8_t *dst = static_cast<uint8_t *>(p.c) + (row * p.c_r + c0 + col_in_tile) * es;
            if (p.c_dtype == ST_F32) {
#pragma unroll
                for (int j = 0; j < kWarpCols; j += 4)
                    reinterpret_cast<float4 *>(dst)[j / 4] = make_float4(acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            } else {
#pragma unroll
                for (int j = 0; j < kWarpCols; j += 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = pack_16(acc[j + 2 * i], acc[j + 2 * i + 1], p.c_dtype);
                    reinterpret_cast<uint4 *>(dst)[j / 8] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    } else {
        // A part owns `own` columns of the tile (with many parts, the last
        // ones none): every CTA sends its sums to their owners' rings, once
        // all of the cluster's MMAs have read them, as [part][row][own + 4
        // columns]; the owner adds its columns over the parts in order, a
        // warp's lanes along C's contiguous dimension.  (Stores do not wait;
        // reading the others' parts cost a remote round trip for every few
        // values.)
        const int own = BN / split < 4 ? 4 : BN / split, own_shift = 31 - __clz(own);  // split is a power of two
        const int stride = own + 4;  // floats; rows on different banks
        __syncwarp();
        if (split > 1) cluster_sync();
        if (scaler) {
            const uint32_t mine = smem_addr(smem) + 4u * static_cast<uint32_t>((part * kTileRows + row_in_tile) * stride);
#pragma unroll
            for (int j = 0; j < kWarpCols; j += 4) {
                const int col = col_in_tile + j;
                const uint32_t to = (split == 1 ? mine : map_to_rank(mine, static_cast<uint32_t>(col >> own_shift))) +
                                    4u * static_cast<uint32_t>(col & (own - 1));
                st_cluster_v4(to, acc[j], acc[j + 1], acc[j + 2], acc[j + 3]);
            }
        }
        __syncwarp();
        if (split > 1) cluster_sync();
        else __syncthreads();
        if (scaler && part * own < BN) {
            const float4 *sums = reinterpret_cast<const float4 *>(smem);
            const int first = (warp - 2) * 32 + lane;
            const int col0 = c0 + part * own;
            if (p.c_dtype == ST_F32) store_sums<float, 32 * Cfg::kScaleWarps>(p, sums, first, own, own_shift, split, r0, col0);
            else if (p.c_dtype == ST_F16) store_sums<__half, 32 * Cfg::kScaleWarps>(p, sums, first, own, own_shift, split, r0, col0);
            else store_sums<__nv_bfloat16, 32 * Cfg::kScaleWarps>(p, sums, first, own, own_shift, split, r0, col0);
        }
    }
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, Cfg::kTmemCols);
    }
}

// ---------------------------------------------------------------- CTA pairs, 256 x 256 tiles
// The large products.  A pair of CTAs (cta_group::2) computes 256 x 256 of C:
// each holds 128 rows of the row operand and 128 columns of the column
// operand, so a block of K costs an SM 32 KB of loads for 512 cycles of its
// tensor core, half of what 128 x 128 tiles of one CTA take.  A block's
// accumulator is 256 TMEM columns, two of them alternate.  (Two halves of 128
// columns with four buffers would be handed over more finely, but a block's
// four MMAs of 128 columns take 369 cycles for the 256 of their arithmetic.)  Eight scaling warps per CTA, two for each
// quarter of the lanes, hold 128 columns of running sums each in registers.
// What bounds it is not the MMAs but reading their sums: 128 KB of TMEM a
// block take eight warps 137 cycles alone and about 750 while the next
// block's MMAs run, against the MMAs' 512; why they slow down is not known.
// Calls back to back: 8192^3 in 605 us (1820 TFLOP/s), 4096 x 4096 x 16384
// with a scale for each column in 462 (1190).
//
// full[s] lives in the even CTA and counts both CTAs' loads; the even CTA's
// MMA warp commits empty[s] and tfull[a] to both CTAs; tempty[a] lives in
// the even CTA and counts the pair's 16 scaling warps.
constexpr int kPairScaleWarps = 8;
constexpr int kPairThreads = 128 + 32 * kPairScaleWarps;  // warps 0 TMA, 1 MMA, 2 scales, 3 idle, 4.. scaling
// 128 running sums and their temporaries do not fit the 168 registers that
// 384 threads get each: the feeding warpgroup hands its own over,
// 56 + 2 * 224 = 3 * 168.
constexpr int kPairFeedRegs = 56, kPairScaleRegs = 224;
constexpr int kPairCols = 256;
constexpr int kPairWarpCols = 128;  // columns of a scaling warp
constexpr int kBoxBytes = 32 * 128;
constexpr int kPairRingDepth = 2;

template <bool CVEC>
struct PairCfg {
    static constexpr int kRowBytes = kTileRows * kBlockK;
    static constexpr int kColBytes = 128 * kBlockK;
    static constexpr int kStageBytes = kRowBytes + kColBytes;
    static constexpr int kStages = 4;
    static constexpr int kAccs = 2;
    static constexpr int kTmemCols = kAccs * kPairCols;
    static constexpr int kStoreBytes = kPairScaleWarps * 2 * kBoxBytes;
    using Ring = ScaleRing<kTileRows, kPairCols, CVEC, kPairRingDepth>;
    static constexpr int kSmemBytes = kStages * kStageBytes + kBarBytes + kStoreBytes + Ring::kBytes + 1024;
    static_assert(kSmemBytes <= 232448, "over the per-block shared memory limit");
};

// One lane's 128-byte row of a 32-row box in the 128-byte swizzle.
__device__ __forceinline__ void put_box_row(uint32_t box, int lane, const uint32_t (&w)[32]) {
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const uint32_t at = box + static_cast<uint32_t>(lane * 128 + ((q ^ (lane & 7)) << 4));
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[4 * q]), "r"(w[4 * q + 1]),
                     "r"(w[4 * q + 2]), "r"(w[4 * q + 3])
                     : "memory");
    }
}

// 8 (4) bytes at byte `at` of a row of such a box.
__device__ __forceinline__ void put_box_8(uint32_t box, int row, int at, uint32_t a, uint32_t b) {
    const uint32_t to = box + static_cast<uint32_t>(row * 128 + (((at >> 4) ^ (row & 7)) << 4) + (at & 15));
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(a), "r"(b) : "memory");
}
__device__ __forceinline__ void put_box_4(uint32_t box, int row, int at, uint32_t a) {
    const uint32_t to = box + static_cast<uint32_t>(row * 128 + (((at >> 4) ^ (row & 7)) << 4) + (at & 15));
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(to), "r"(a) : "memory");
}

// Row and column tile of tile t: 8 row tiles of a column tile after another,
// so that the tiles in flight share their operands in L2.
__device__ __forceinline__ void pair_tile(const Fp8Params &p, int t, int &tr, int &tc) {
    constexpr int kGroup = 8;
    const int in_group = kGroup * p.tiles_c;
    const int first = t / in_group * kGroup;
    const int rows = p.tiles_r - first < kGroup ? p.tiles_r - first : kGroup;
    tr = first + (t % in_group) % rows;
    tc = (t % in_group) / rows;
}

template <bool R_MN, bool C_MN, bool CVEC>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kPairThreads, 1)
    gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ CUtensorMap tmap_c,
                         const __grid_constant__ CUtensorMap tmap_out, const Fp8Params p) {
    using Cfg = PairCfg<CVEC>;
    using Ring = typename Cfg::Ring;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *boxes = smem + Cfg::kStages * Cfg::kStageBytes;
    uint64_t *bars = reinterpret_cast<uint64_t *>(boxes + Cfg::kStoreBytes);
    constexpr int kBars = 2 * Cfg::kStages + 2 * Cfg::kAccs + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars + Ring::kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
    const int tiles = p.tiles_r * p.tiles_c;
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (Cfg::kStages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * Cfg::kStages + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * Cfg::kStages + Cfg::kAccs + a); };
    const uint32_t drain_bar = bar0 + 8u * (kBars - 1);
    const Ring ring{reinterpret_cast<float *>(boxes + Cfg::kStoreBytes + kBarBytes), bar0 + 8u * kBars};

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < Cfg::kAccs; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 2 * kPairScaleWarps);
        }
        mbar_init(drain_bar, 1);
        ring.init(kPairScaleWarps);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_map(&tmap_r);
        tma_prefetch_map(&tmap_c);
        tma_prefetch_map(&tmap_out);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_addr(tmem_slot), Cfg::kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    cluster_sync();
    tc_fence_after_sync();
    const uint32_t tmem_base = *tmem_slot;
    pdl_begin();  // nothing above touches global memory

    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kPairFeedRegs));
        if (warp == 0) {
            // -------------------------------------------- TMA producer (both CTAs)
            if (lane == 0) {
                const uint64_t pol = l2_policy_evict_last();
                const uint32_t even_full0 = map_to_rank(full_bar(0), 0);
                int s = 0, issued = 0;
                uint32_t ph = 0;
                bool ok = true;
                for (int t = pair; ok && t < tiles; t += pairs) {
                    int tr, tc;
                    pair_tile(p, t, tr, tc);
                    const int r0 = tr * 2 * kTileRows + static_cast<int>(rank) * kTileRows;
                    const int c0 = tc * kPairCols + static_cast<int>(rank) * 128;
                    for (int b = 0; b < p.k_blocks; ++b, ++issued) {
                        if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                            ok = false;
                            break;
                        }
                        if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * Cfg::kStageBytes);
                        const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes);
                        const uint32_t sc = sr + Cfg::kRowBytes;
                        const uint32_t fb = even_full0 + 8u * s;
                        const int k0 = b * kBlockK;
                        if constexpr (R_MN) tma_load_2d_pair(sr, &tmap_r, fb, r0, k0, pol);
                        else tma_load_2d_pair(sr, &tmap_r, fb, k0, r0, pol);
                        if constexpr (C_MN) tma_load_2d_pair(sc, &tmap_c, fb, c0, k0, pol);
                        else tma_load_2d_pair(sc, &tmap_c, fb, k0, c0, pol);
                        if (++s == Cfg::kStages) {
                            s = 0;
                            ph ^= 1u;
                        }
                    }
                }
                if (!ok) {
                    *abort_flag = 1;
                    atomicExch(p.err, kDevAbortGemmProducer);
                }
                if (rank == 0) drain_ring(issued, Cfg::kStages, full_bar, p.timeout_ns);  // both CTAs' copies
                else drain_ring(issued, Cfg::kStages, empty_bar, p.timeout_ns);  // the even CTA's arrivals here
            }
        } else if (warp == 1) {
            // -------------------------------------------- MMA issuer (even CTA)
            if (rank == 0) {
                int s = 0, a = 0;
                uint32_t ph = 0, aph = 0;
                bool ok = true;
                const uint64_t dr0 = smem_desc_sw128(smem_addr(smem), R_MN ? 128 * 128 : 16, 1024);
                const uint64_t dc0 = smem_desc_sw128(smem_addr(smem) + Cfg::kRowBytes, C_MN ? 128 * 128 : 16, 1024);
                for (int t = pair; ok && t < tiles; t += pairs) {
                    for (int b = 0; b < p.k_blocks; ++b) {
                        const bool ready = mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns) &&
                                           mbar_wait(tempty_bar(a), aph ^ 1u, abort_flag, p.timeout_ns);
                        if (!__all_sync(0xffffffffu, ready)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                        if (elect_one()) {
                            const uint64_t step = static_cast<uint64_t>(s) * (Cfg::kStageBytes >> 4);
                            issue_block<R_MN, C_MN, true>(tmem_base + static_cast<uint32_t>(a * kPairCols), dr0 + step,
                                                          dc0 + step, p.idesc);
                            tc_commit_pair_multicast(tfull_bar(a), 3);
                            tc_commit_pair_multicast(empty_bar(s), 3);
                        }
                        __syncwarp();
                        if (++s == Cfg::kStages) {
                            s = 0;
                            ph ^= 1u;
                        }
                        if (++a == Cfg::kAccs) {
                            a = 0;
                            aph ^= 1u;
                        }
                    }
                }
                if (!ok) {
                    *abort_flag = 1;
                    atomicExch(p.err, kDevAbortGemmMma);
                }
                if (elect_one()) tc_commit_pair(drain_bar);
                __syncwarp();
                drain_ring(1, 1, [&](int) { return drain_bar; }, p.timeout_ns);  // the MMAs read shared memory and write TMEM
            }
        } else if (warp == 2) {
            // -------------------------------------------- scales (both CTAs)
            int d = 0;
            uint32_t dph = 0;
            for (int t = pair; t < tiles; t += pairs) {
                int tr, tc;
                pair_tile(p, t, tr, tc);
                if (!ring.load(p, tr * 2 * kTileRows + static_cast<int>(rank) * kTileRows, tc * kPairCols, 0, 1,
                               p.k_blocks, lane, d, dph, abort_flag)) {
                    *abort_flag = 1;
                    break;
                }
            }
            copies_done();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kPairScaleRegs));
        // ------------------------------------------------ scaling warps (both CTAs)
        const int g = warp & 3, e = warp - 4;
        const int half = e >> 2;
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(g * 32) << 16) + static_cast<uint32_t>(half * kPairWarpCols);
        const uint32_t even_tempty0 = map_to_rank(tempty_bar(0), 0);
        uint8_t *my_boxes = boxes + e * 2 * kBoxBytes;
        int box = 0;
        ScalePosition at;
        bool ok = true;
        for (int t = pair; t < tiles; t += pairs) {
            float acc[kPairWarpCols];
#pragma unroll
            for (int j = 0; j < kPairWarpCols; ++j) acc[j] = 0.0f;
            auto released = [&](int a) {
                if (rank == 0) mbar_arrive_relaxed(tempty_bar(a));
                else mbar_arrive_cluster_relaxed(even_tempty0 + 8u * a);
            };
            if constexpr (CVEC)
                ok = scale_blocks_by_column<kPairWarpCols, Cfg::kAccs, kPairCols>(acc, p.k_blocks, t_lane, g * 32,
                                                                                  half * kPairWarpCols, ring, at, tfull_bar,
                                                                                  released, lane, abort_flag, p.timeout_ns);
            else
                ok = scale_blocks<kPairWarpCols, 32, false, Cfg::kAccs, kPairCols>(acc, p.k_blocks, t_lane, g * 32 + lane, half,
                                                                                   ring, at, tfull_bar, released, lane,
                                                                                   abort_flag, p.timeout_ns);
            if (!ok) {
                *abort_flag = 1;
                if (lane == 0) atomicExch(p.err, kDevAbortGemmEpilogue);
                break;
            }
            // ---- bias, conversion, and out through the warp's two boxes of 32 rows x 128 bytes
            int tr, tc;
            pair_tile(p, t, tr, tc);
            const int row0 = tr * 2 * kTileRows + static_cast<int>(rank) * kTileRows + g * 32;
            const int col0 = tc * kPairCols + half * kPairWarpCols;
            if (row0 >= p.rows) continue;
            // CVEC: this lane's element e of 8 columns c lies at (row_of(e), col_of(c, e)); otherwise row `lane`, all columns
            auto row_of = [&](int e) { return (lane >> 2) + 8 * (e >> 1); };
            auto col_of = [&](int c, int e) { return 8 * c + 2 * (lane & 3) + (e & 1); };
            if (p.bias != nullptr) {
#pragma unroll
                for (int j = 0; j < kPairWarpCols; ++j) {
                    const int c = col0 + (CVEC ? col_of(j / 8, j % 8) : j);
                    acc[j] += c < p.cols ? load_any(p.bias, p.bias_dtype, c) : 0.0f;
                }
            }
            if (p.staged) {
#pragma unroll
                for (int h = 0; h < kPairWarpCols / 32; ++h) {  // a box: 32 columns of fp32, 64 of 16 bits
                    if (p.c_dtype != ST_F32 && (h & 1)) continue;
                    if (col0 + 32 * h >= p.cols) continue;
                    if (lane == 0) bulk_wait_group_read<1>();  // the store that last used this box has read it
                    __syncwarp();
                    const uint32_t at_box = smem_addr(my_boxes + box * kBoxBytes);
                    if constexpr (CVEC) {
                        if (p.c_dtype == ST_F32) {
#pragma unroll
                            for (int c = 0; c < 4; ++c)
#pragma unroll
                                for (int e = 0; e < 8; e += 2)
                                    put_box_8(at_box, row_of(e), 4 * (8 * c + 2 * (lane & 3)),
                                              __float_as_uint(acc[32 * h + 8 * c + e]), __float_as_uint(acc[32 * h + 8 * c + e + 1]));
                        } else {
#pragma unroll
                            for (int c = 0; c < 8; ++c)
#pragma unroll
                                for (int e = 0; e < 8; e += 2) {
                                    const int j = (32 * h + 8 * c + e) % kPairWarpCols;
                                    put_box_4(at_box, row_of(e), 2 * (8 * c + 2 * (lane & 3)), pack_16(acc[j], acc[j + 1], p.c_dtype));
                                }
                        }
                    } else {
                        uint32_t w[32];
                        if (p.c_dtype == ST_F32) {
#pragma unroll
                            for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(acc[32 * h + i]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; ++i) {
                                const int j = (32 * h + 2 * i) % kPairWarpCols;
                                w[i] = pack_16(acc[j], acc[j + 1], p.c_dtype);
                            }
                        }
                        put_box_row(at_box, lane, w);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {  // TMA clips the box at C's extents
                        tma_store_2d(&tmap_out, at_box, col0 + 32 * h, row0);
                        bulk_commit_group();
                    }
                    box ^= 1;
                }
            } else {  // 32 columns at a time through both boxes, then a row at a time with a lane per column
                float *m = reinterpret_cast<float *>(my_boxes);
                const int n = p.rows - row0 < 32 ? p.rows - row0 : 32;
#pragma unroll
                for (int h = 0; h < kPairWarpCols / 32; ++h) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        m[CVEC ? row_of(i % 8) * 33 + col_of(i / 8, i % 8) : lane * 33 + i] = acc[32 * h + i];
                    __syncwarp();
                    const int c = col0 + 32 * h + lane;
                    if (c < p.cols)
                        for (int r = 0; r < n; ++r) store_any(p.c, p.c_dtype, (row0 + r) * p.c_r + c, m[r * 33 + lane]);
                    __syncwarp();
                }
            }
        }
        if (lane == 0) bulk_wait_group_all();  // every store of C has landed
    }

    tc_fence_before_sync();
    __syncwarp();
    cluster_sync();  // all MMAs retired, all TMEM reads done, no remote arrival pending
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc_pair(tmem_base, Cfg::kTmemCols);
    }
}

// Dense copy of a strided 8-bit [rows, cols] matrix, rows of `ld` bytes (a
// multiple of 16).  Whole 16-byte pieces are written, so the padding gets
// bytes of no meaning; the tensor map ends at cols.  Unit column stride: 16 bytes
// a thread, put together from the aligned words that hold them.
__global__ void __launch_bounds__(256) repack_8_kernel(const uint8_t *__restrict__ src, int64_t s0, int64_t s1,
                                                       int64_t rows, int64_t cols, uint8_t *__restrict__ dst, int64_t ld) {
    pdl_wait();
    const int64_t per_row = ld / 16, total = rows * per_row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = i / per_row, c = (i - r * per_row) * 16;
        const int n = cols - c < 16 ? static_cast<int>(cols - c) : 16;
        uint32_t w[4] = {0, 0, 0, 0};
        if (s1 == 1) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(src + r * s0 + c);
            const uint32_t *words = reinterpret_cast<const uint32_t *>(at & ~uintptr_t(3));
            const int shift = static_cast<int>(at & 3) * 8, have = (static_cast<int>(at & 3) + n + 3) / 4;
            uint32_t x[5];
#pragma unroll
            for (int j = 0; j < 5; ++j) x[j] = j < have ? words[j] : 0u;  // only words with a byte of the row
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(x[j], x[j + 1], shift);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
                if (j < n) w[j / 4] |= static_cast<uint32_t>(src[r * s0 + (c + j) * s1]) << (8 * (j % 4));
        }
        *reinterpret_cast<uint4 *>(dst + r * ld + c) = make_uint4(w[0], w[1], w[2], w[3]);
    }
    pdl_trigger();
}

__global__ void __launch_bounds__(256) fill_bias_kernel(void *c, int64_t ldc, int c_dtype, const void *bias,
                                                        int bias_dtype, int64_t m, int64_t n) {
    pdl_wait();
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < m * n;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t r = i / n, q = i - r * n;
        store_any(c, c_dtype, r * ldc + q, bias ? load_any(bias, bias_dtype, q) : 0.0f);
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- host side
// 128-byte-swizzled box of 128 bytes x `box_rows` of a byte matrix whose rows are `ld` bytes apart
int make_map_8(CUtensorMap *map, const void *base, int64_t inner, int64_t outer, int64_t ld, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {128, static_cast<cuuint32_t>(box_rows)};
    return make_tensor_map(map, "an 8-bit operand", CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box);
}

template <int BN, bool R_MN, bool C_MN, bool CVEC>
int launch_instance(const CUtensorMap &mr, const CUtensorMap &mc, const Fp8Params &p, cudaStream_t stream) {
    using Cfg = Fp8Cfg<BN, CVEC>;
    auto kern = gemm_fp8_kernel<BN, R_MN, C_MN, CVEC>;
    static uint64_t attr_set = 0;  // one bit per device ordinal
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(p.tiles_r) * p.tiles_c * p.split));
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (p.split > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(p.split);
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    ST_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, mr, mc, p));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "gemm_fp8_kernel launch");
}

template <int BN>
int launch_narrow(const CUtensorMap &mr, const CUtensorMap &mc, const Fp8Params &p, bool r_mn, cudaStream_t stream) {
    return r_mn ? launch_instance<BN, true, false, true>(mr, mc, p, stream)
                : launch_instance<BN, false, false, true>(mr, mc, p, stream);
}

template <bool CVEC>
int launch_wide(const CUtensorMap &mr, const CUtensorMap &mc, const Fp8Params &p, bool r_mn, bool c_mn,
                cudaStream_t stream) {
    if (r_mn)
        return c_mn ? launch_instance<128, true, true, CVEC>(mr, mc, p, stream)
                    : launch_instance<128, true, false, CVEC>(mr, mc, p, stream);
    return c_mn ? launch_instance<128, false, true, CVEC>(mr, mc, p, stream)
                : launch_instance<128, false, false, CVEC>(mr, mc, p, stream);
}

template <bool R_MN, bool C_MN, bool CVEC>
int launch_pair_instance(const CUtensorMap &mr, const CUtensorMap &mc, const CUtensorMap &mo, const Fp8Params &p,
                         int sm_count, cudaStream_t stream) {
    auto kern = gemm_fp8_pair_kernel<R_MN, C_MN, CVEC>;
    static uint64_t attr_set = 0;  // one bit per device ordinal
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, PairCfg<CVEC>::kSmemBytes));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    const int64_t tiles = static_cast<int64_t>(p.tiles_r) * p.tiles_c;
    const int64_t pairs = tiles < sm_count / 2 ? tiles : sm_count / 2;
    ST_CUDA_TRY(launch_kernel(kern, static_cast<unsigned>(2 * pairs), kPairThreads, PairCfg<CVEC>::kSmemBytes, stream, mr, mc, mo, p));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "gemm_fp8_pair_kernel launch");
}

template <bool CVEC>
int launch_pair(const CUtensorMap &mr, const CUtensorMap &mc, const CUtensorMap &mo, const Fp8Params &p, bool r_mn,
                bool c_mn, int sm_count, cudaStream_t stream) {
    if (r_mn)
        return c_mn ? launch_pair_instance<true, true, CVEC>(mr, mc, mo, p, sm_count, stream)
                    : launch_pair_instance<true, false, CVEC>(mr, mc, mo, p, sm_count, stream);
    return c_mn ? launch_pair_instance<false, true, CVEC>(mr, mc, mo, p, sm_count, stream)
                : launch_pair_instance<false, false, CVEC>(mr, mc, mo, p, sm_count, stream);
}

// 32-row box of 128 bytes of C
int make_map_out(CUtensorMap *map, const GemmFp8Args &g) {
    auto fn = tensor_map_encoder();
    if (!fn) return fail(ST_ERR_CUDA, "cuTensorMapEncodeTiled is not available from the driver");
    const int es = static_cast<int>(dtype_size(g.c_dtype));
    const CUtensorMapDataType dt = g.c_dtype == ST_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : g.c_dtype == ST_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                         : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    cuuint64_t dims[2] = {static_cast<cuuint64_t>(g.b.rows), static_cast<cuuint64_t>(g.a.rows)};
    cuuint64_t strides[1] = {static_cast<cuuint64_t>(g.ldc) * es};
    cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / es), 32};
    cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, dt, 2, g.c, dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS)
        return fail(ST_ERR_INVALID_ARGUMENT, "cuTensorMapEncodeTiled rejected C (error " +
                                                 std::to_string(static_cast<int>(r)) + ")");
    return ST_OK;
}

// How TMA can read a [rows, k] operand: directly along K or along its rows,
// or after a copy (the overlapping rows of a broadcast or a window among the
// copies).
struct Access {
    bool mn;     // rows contiguous
    bool copy;   // through the workspace
    int64_t ld;  // bytes between rows (K-major) or between K indices (mn)
};

Access access_of(const Fp8Operand &o) {
    const bool base = (reinterpret_cast<uintptr_t>(o.data) & 15u) == 0;
    auto fits = [&](int64_t unit, int64_t unit_extent, int64_t ld, int64_t outer) {
        return base && (unit == 1 || unit_extent == 1) &&
               (outer == 1 || (ld >= unit_extent && ld % 16 == 0 && ld < (int64_t(1) << 40)));
    };
    auto stride = [](int64_t ld, int64_t outer, int64_t extent) { return outer == 1 ? (extent + 15) / 16 * 16 : ld; };
    if (fits(o.s_k, o.k, o.s_row, o.rows)) return {false, false, stride(o.s_row, o.rows, o.k)};
    if (fits(o.s_row, o.rows, o.s_k, o.k)) return {true, false, stride(o.s_k, o.k, o.rows)};
    const bool mn = o.s_row == 1 && o.s_k != 1;
    return {mn, true, ((mn ? o.rows : o.k) + 15) / 16 * 16};
}

// Tile shape and split of a product of one orientation: the least estimated
// time.  A wave of CTAs costs its blocks of K and what a CTA spends outside
// them; the figures are SM cycles fitted to B200 timings of 1 x 1024 x 4096 to
// 8192^3 (within 10 % of most; e.g. 64 x 8192 x 8192 estimated 19.4 us on 128
// columns and two parts, 21.3 on 64 columns and four, measured 20.6 and 22.7).
struct Fp8Plan {
    bool pair = false;
    int bn = 128, split = 1;
    double cycles = 1e300;
};

Fp8Plan plan_fp8(int64_t rows, int64_t cols, int64_t k_blocks, bool k_major, bool column_scales, int sm_count) {
    Fp8Plan best;
    auto offer = [&](bool pair, int bn, int split, int64_t ctas, int64_t slots, double block, double ends) {
        const double t = static_cast<double>(cdiv(ctas, slots)) * (static_cast<double>(cdiv(k_blocks, split)) * block + ends);
        if (t < best.cycles) best = Fp8Plan{pair, bn, split, t};
    };
    struct Shape {
        int bn;
        double block, two, ends, join[3];  // a block alone on an SM, and beside another CTA; extra for 2, 4 and 8 parts
    };
    const Shape shapes[] = {{16, 600, 1000, 12000, {0, 0, 0}},
                            {32, 700, 1050, 14000, {0, 0, 0}},
                            {64, 1050, 1340, 18000, {0, 0, 5000}},
                            {128, column_scales ? 890.0 : 620.0, 0, 9000, {7000, 11700, 16000}}};
    for (const Shape &s : shapes) {
        if (s.bn < 128 && (!k_major || s.bn < (cols < 64 ? cols : 64))) continue;  // narrow boxes are K-major
        const int64_t tiles = cdiv(rows, kTileRows) * cdiv(cols, s.bn);
        const int per_sm = s.bn == 128 ? 1 : 2;
        for (int parts = 0; parts <= 3 && (1 << parts) <= k_blocks; ++parts) {
            const int64_t ctas = tiles << parts;
            offer(false, s.bn, 1 << parts, ctas, static_cast<int64_t>(sm_count) * per_sm,
                  ctas > sm_count && per_sm == 2 ? s.two : s.block, s.ends + (parts > 0 ? s.join[parts - 1] : 0));
        }
    }
    if (cols > 64)
        offer(true, 128, 1, cdiv(rows, 256) * cdiv(cols, 256), sm_count / 2, column_scales ? 1400 : 980, 11400);
    return best;
}

int64_t copy_bytes(const Fp8Operand &o, const Access &a) {
    return a.copy ? ((a.mn ? o.k : o.rows) * a.ld + 255) / 256 * 256 : 0;
}

int copy_operand(const Fp8Operand &o, const Access &a, uint8_t *dst, int sm_count, cudaStream_t stream) {
    const int64_t outer = a.mn ? o.k : o.rows, inner = a.mn ? o.rows : o.k;
    const int64_t s0 = a.mn ? o.s_k : o.s_row, s1 = a.mn ? o.s_row : o.s_k;
    return launch_repack_8(o.data, s0, s1, outer, inner, dst, a.ld, sm_count, stream);
}

}  // namespace

int launch_repack_8(const void *src, int64_t s0, int64_t s1, int64_t rows, int64_t cols, void *dst, int64_t ld,
                    int sm_count, cudaStream_t stream) {
    int64_t grid = cdiv(rows * (ld / 16), 256);
    if (grid > static_cast<int64_t>(sm_count) * 8) grid = static_cast<int64_t>(sm_count) * 8;
    ST_CUDA_TRY(launch_kernel(repack_8_kernel, static_cast<unsigned>(grid), 256, 0, stream, static_cast<const uint8_t *>(src), s0,
                              cols == 1 ? int64_t(1) : s1, rows, cols, static_cast<uint8_t *>(dst), ld));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "repack_8_kernel");
}

int launch_fill_bias(void *c, int64_t ldc, int c_dtype, const void *bias, int bias_dtype, int64_t m, int64_t n, int sm_count,
                     cudaStream_t stream) {
    ST_CUDA_TRY(launch_kernel(fill_bias_kernel, static_cast<unsigned>(sm_count), 256, 0, stream, c, ldc, c_dtype, bias, bias_dtype, m, n));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "fill_bias_kernel");
}

int launch_fp8_wait_check(bool by_column, uint64_t limit_ns, int *dev_err, cudaStream_t stream) {
    if (by_column) fp8_wait_check_kernel<true><<<1, 32, 0, stream>>>(limit_ns, dev_err);
    else fp8_wait_check_kernel<false><<<1, 32, 0, stream>>>(limit_ns, dev_err);
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "fp8_wait_check_kernel launch");
}

int64_t gemm_fp8_workspace_bytes(const Fp8Operand &a, const Fp8Operand &b) {
    if (a.rows == 0 || b.rows == 0 || a.k == 0) return 0;
    return copy_bytes(a, access_of(a)) + copy_bytes(b, access_of(b));
}

int launch_gemm_fp8(const GemmFp8Args &g, void *workspace, int sm_count, int *dev_err, uint64_t timeout_ns,
                    cudaStream_t stream) {
    const int64_t m = g.a.rows, n = g.b.rows, k = g.a.k;
    if (m == 0 || n == 0) return ST_OK;
    if (k == 0) {
        return launch_fill_bias(g.c, g.ldc, g.c_dtype, g.bias, g.bias_dtype, m, n, sm_count, stream);
    }
    Fp8Operand op[2] = {g.a, g.b};
    Access acc[2] = {access_of(g.a), access_of(g.b)};
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    for (int i = 0; i < 2; ++i) {
        if (!acc[i].copy) continue;
        ST_TRY(copy_operand(op[i], acc[i], ws, sm_count, stream));
        op[i].data = ws;
        ws += copy_bytes(op[i], acc[i]);
    }
    // A becomes the row operand; or B does, where few rows of A then make a
    // narrow tile's columns.
    const int64_t k_blocks = cdiv(k, kBlockK);
    Fp8Plan plan = plan_fp8(m, n, k_blocks, !acc[1].mn, g.b.scale_shift == 0, sm_count);
    bool swap = false;
    if (m <= 64 && !acc[0].mn) {
        const Fp8Plan other = plan_fp8(n, m, k_blocks, true, true, sm_count);
        swap = other.cycles < plan.cycles;
        if (swap) plan = other;
    }
    const int ri = swap ? 1 : 0, ci = swap ? 0 : 1;
    const Fp8Operand &r = op[ri], &c = op[ci];
    const bool pair = plan.pair;
    const int bn = plan.bn;
    Fp8Params p{};
    p.rows = static_cast<int>(r.rows);
    p.cols = static_cast<int>(c.rows);
    p.k_blocks = static_cast<int>(k_blocks);
    p.tiles_r = static_cast<int>(cdiv(r.rows, pair ? 2 * kTileRows : kTileRows));
    p.tiles_c = static_cast<int>(cdiv(c.rows, pair ? kPairCols : bn));
    p.split = plan.split;
    const int64_t tiles = static_cast<int64_t>(p.tiles_r) * p.tiles_c;
    if (tiles * p.split > INT32_MAX) return fail(ST_ERR_UNSUPPORTED, "matmul_fp8: too many output tiles");
    p.rs = static_cast<const float *>(r.scale);
    p.rs_i = r.scale_row;
    p.rs_b = r.scale_k;
    p.rs_shift = r.scale_shift;
    p.cs = static_cast<const float *>(c.scale);
    p.cs_i = c.scale_row;
    p.cs_b = c.scale_k;
    p.cs_shift = c.scale_shift;
    p.c = g.c;
    p.c_r = swap ? 1 : g.ldc;
    p.c_c = swap ? g.ldc : 1;
    p.c_dtype = g.c_dtype;
    p.bias = g.bias;
    p.bias_dtype = g.bias_dtype;
    p.bias_on_rows = swap;
    p.idesc = mma_idesc_f8(r.e5m2, c.e5m2, acc[ri].mn, acc[ci].mn, pair ? 2 * kTileRows : kTileRows,
                           static_cast<uint32_t>(pair ? kPairCols : bn));
    p.err = dev_err;
    p.timeout_ns = timeout_ns;
    CUtensorMap mr, mc;
    if (acc[ri].mn) ST_TRY(make_map_8(&mr, r.data, r.rows, k, acc[ri].ld, kBlockK));
    else ST_TRY(make_map_8(&mr, r.data, k, r.rows, acc[ri].ld, kTileRows));
    if (acc[ci].mn) ST_TRY(make_map_8(&mc, c.data, c.rows, k, acc[ci].ld, kBlockK));
    else ST_TRY(make_map_8(&mc, c.data, k, c.rows, acc[ci].ld, bn));
    if (pair) {
        CUtensorMap mo = mr;  // unused where C leaves by plain stores
        // a TMA store writes whole 16-byte pieces: not where a row of C ends inside one
        const int64_t es = static_cast<int64_t>(dtype_size(g.c_dtype));
        p.staged = reinterpret_cast<uintptr_t>(g.c) % 16 == 0 && g.ldc * es % 16 == 0 && n * es % 16 == 0;
        if (p.staged) ST_TRY(make_map_out(&mo, g));
        return p.cs_shift == 7 ? launch_pair<false>(mr, mc, mo, p, acc[ri].mn, acc[ci].mn, sm_count, stream)
                               : launch_pair<true>(mr, mc, mo, p, acc[ri].mn, acc[ci].mn, sm_count, stream);
    }
    switch (bn) {
    case 16: return launch_narrow<16>(mr, mc, p, acc[ri].mn, stream);
    case 32: return launch_narrow<32>(mr, mc, p, acc[ri].mn, stream);
    case 64: return launch_narrow<64>(mr, mc, p, acc[ri].mn, stream);
    default: break;
    }
    return p.cs_shift == 7 ? launch_wide<false>(mr, mc, p, acc[ri].mn, acc[ci].mn, stream)
                           : launch_wide<true>(mr, mc, p, acc[ri].mn, acc[ci].mn, stream);
}

}  // namespace st
