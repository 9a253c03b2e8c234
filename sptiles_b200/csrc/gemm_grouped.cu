// gemm_grouped.cu -- matrix products by groups of rows, for layers of which
// each token meets one of several weight matrices.
//
//   rows      C[r, n]    = sum_k A[r, k] B[g, k, n]               for the rows r of group g
//   weights   D[g, k, n] = sum over the rows r of group g of A[r, k] C[r, n]
//
// Group g is rows [ends[g - 1], ends[g]); the ends lie on the device, and no
// host code waits for them: every CTA reads them and works out which tiles
// there are.  An end below the one before it, or beyond the rows, is taken as
// that bound, so that whatever the ends hold nothing outside of A, C and D is
// touched.  f16 or bf16 operands, fp32 sums (tcgen05.mma into TMEM).
//
//   warp 0      TMA producer
//   warp 1      MMA issuer (owns the TMEM allocation)
//   warps 2-9   C: TMEM -> registers -> columns of a tile, while the MMAs of
//               the next tile fill the other accumulator
//
// The kernels know a row operand (the MMA's M) and a column operand (its N).
//
// First form: B's columns are the rows of a tile and the group's rows its
// columns, 16 to 256 of them: N is a field of the MMA's descriptor, so a group
// is cut into tiles of equal size in steps of 16 (32 for a pair of CTAs, whose
// M = 256 takes no other) and nothing is padded to 128 or 256 rows (16384 rows on 32 groups of 4096 x 4096, between 60 and 2400
// rows each: 647 us with a group's rows as M).  The last columns of a tile may
// be rows of the next group, or what an earlier tile left in shared memory:
// columns of a product do not mix, and those are not stored.
//
// Second form: the rows are what is summed over, and a group's last, shorter
// step of n < 64 rows brings rows of the next group too.  It takes ceil(n / 16)
// MMAs of 16 rows, and of the last one's rows those behind the group are set to
// zero in shared memory first, in both operands (a product with a NaN is one).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <utility>

#include "common.h"
#include "fp8.cuh"
#include "sm100.cuh"
#include "tensor_map.h"

namespace st {
namespace {

// Measured, bf16: one group of 16384 rows of 4096 x 4096 340 to 400 us (1370 to
// 1618 TFLOP/s), 32 unequal groups of them 410 to 470 over 20 calls and 510 to 545
// over seconds under the power cap (the tensor pipe 85 % busy); 64 rows on 64
// groups of 2048 x 4096 98 us, bound by the weights' bytes (92 at the copy rate);
// the gradient of 32 x 2048 x 4096 from 16384 rows in f32 295 on a cool card to 400
// (194), in bf16 235 to 260 (165: the products), bound by its stores beside the loads.
constexpr int kMaxGroups = kGroupedMaxGroups;
constexpr int kBK = 64;  // elements of the contraction a stage: 128 bytes, one swizzle span
constexpr int kMmaK = 16;
constexpr int kBarBytes = 512;
constexpr int kOutWarps = 8;  // warps that take C out, two for each quarter of the TMEM lanes

struct GroupedParams {
    const int *ends;
    int groups;
    int rows, k, n;      // A [rows, k]; n columns of C
    int tiles_r;         // along the row operand
    int tiles_c;         // weights: along the column operand
    int b_groups;        // 0: one B for every group
    void *c;
    int64_t c_g, ldc;    // weights: D's strides of groups and rows
    int c_dtype;
    int zero_rest;       // rows of no group are set to 0
    int split;           // CTAs of a cluster that share a tile
    int r_by_64, c_by_64;  // the operand's map splits its columns in 64s, so that one box holds two of them
    int reads;           // there is something to sum over: the maps are valid
    uint32_t idesc;
    int *err;
    unsigned long long timeout_ns;
};

// Maps of the column operand with boxes of 32, 64, 96 and 128 rows: a stage's
// rows come in one box.  (Four boxes of 32 cost more than one of 128: 16384 x
// 4096 x 4096 421 us against 355.)  The second form uses the first one only.
struct ColumnMaps {
    CUtensorMap by32[4];
};

// ends[g] clipped to [ends[g - 1], rows], and the tiles up to and with group g.
struct GroupTable {
    int row_end[kMaxGroups];
    int tile_end[kMaxGroups];
};

// By one warp: 32 groups at a time, a running maximum and a running sum.
// COLS: the most columns of a tile.
template <bool WEIGHTS, int COLS>
__device__ __forceinline__ void build_table(GroupTable &t, const GroupedParams &p, int lane) {
    int last_end = 0, last_tile = 0;
    for (int g0 = 0; g0 < p.groups; g0 += 32) {
        const int g = g0 + lane;
        int end = g < p.groups ? p.ends[g] : 0;
        end = end < 0 ? 0 : end > p.rows ? p.rows : end;
        if (end < last_end) end = last_end;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, end, o);
            if (lane >= o && x > end) end = x;
        }
        int begin = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) begin = last_end;
        int tiles = p.tiles_r * (WEIGHTS ? p.tiles_c : (end - begin + COLS - 1) / COLS);
        if (g >= p.groups) tiles = 0;
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int x = __shfl_up_sync(0xffffffffu, tiles, o);
            if (lane >= o) tiles += x;
        }
        tiles += last_tile;
        if (g < p.groups) {
            t.row_end[g] = end;
            t.tile_end[g] = tiles;
        }
        last_end = __shfl_sync(0xffffffffu, end, 31);
        last_tile = __shfl_sync(0xffffffffu, tiles, 31);
    }
}

// One output tile.
struct Tile {
    int group;
    int r0, c0, cols;  // first row and column, columns inside (c0: a row of A in the first form)
    int first, rows;   // the group's rows (second form)
    int blocks;        // steps of the contraction
};

// Tiles in order; each role walks them for itself.  ROWS, COLS: a tile's most.
template <bool WEIGHTS, int ROWS, int COLS>
struct TileWalk {
    static constexpr int kStep = ROWS == 256 ? 32 : 16;  // of the MMA's N
    static __device__ __forceinline__ uint32_t idesc_n(int cols) { return static_cast<uint32_t>((cols + kStep - 1) / kStep * (kStep / 8)) << 17; }
    int t, step, g = 0;
    __device__ __forceinline__ TileWalk(int first, int step) : t(first), step(step) {}
    __device__ __forceinline__ bool next(const GroupTable &table, const GroupedParams &p, Tile &out) {
        while (g < p.groups && t >= table.tile_end[g]) ++g;
        if (g >= p.groups) return false;
        const int begin = g > 0 ? table.row_end[g - 1] : 0, end = table.row_end[g], rows = end - begin;
        const int i = t - (g > 0 ? table.tile_end[g - 1] : 0);
        const int tiles_c = WEIGHTS ? p.tiles_c : (rows + COLS - 1) / COLS;
        // eight column tiles of a row tile after another, so that tiles in flight share their operands in L2
        constexpr int kBand = 8;
        const int in_band = kBand * p.tiles_r, band = i / in_band * kBand;
        const int high = tiles_c - band < kBand ? tiles_c - band : kBand;
        const int c = band + i % in_band % high;
        out.group = g;
        out.r0 = i % in_band / high * ROWS;
        out.first = begin;
        out.rows = rows;
        if constexpr (WEIGHTS) {
            out.c0 = c * COLS;
            out.cols = p.k - out.c0 < COLS ? p.k - out.c0 : COLS;
            out.blocks = (rows + kBK - 1) / kBK;
        } else {
            const int even = ((rows + tiles_c - 1) / tiles_c + kStep - 1) / kStep * kStep;  // columns of the group's tiles
            out.c0 = begin + c * even;
            out.cols = rows - c * even < even ? rows - c * even : even;
            out.blocks = (p.k + kBK - 1) / kBK;
        }
        t += step;
        return true;
    }
};

// The step's rows that belong to the group, and whether its last MMA meets others.
struct Step {
    int mmas;
    bool mixed;
    __device__ __forceinline__ explicit Step(int left) : mmas(left < kBK ? (left + kMmaK - 1) / kMmaK : kBK / kMmaK), mixed(left < kBK && left % kMmaK != 0) {}
};

// By a warp: rows from `left` on of its last MMA become 0 in a stage, 2 x 128
// columns in 64s of 64 rows, and the tensor core sees it.  (A swizzled row's
// units stay within its 128 bytes.)
__device__ __forceinline__ void zero_behind(uint32_t stage, int left, int lane) {
    const int units = (kMmaK - left % kMmaK) * 4 * 8;  // of 16 bytes
    for (int i = lane; i < units; i += 32) {
        const int line = i >> 3, row = left + (line >> 2);
        asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(stage + (line & 3) * (64 * 128) + row * 128 + (i & 7) * 16), "r"(0) : "memory");
    }
    fence_proxy_async_smem();
    __syncwarp();
}

// 128 columns (64s of a swizzle span each) x 64 rows of an operand that lies
// along its columns.  y and z: the map's other coordinates.  (Two boxes a
// stage and operand instead of one: weights of 4096 x 4096 from 16384 rows
// 433 us, in one 367.)
template <bool PAIR>
__device__ __forceinline__ void load_columns(uint32_t dst, const CUtensorMap *map, uint32_t bar, int col, int y, int z, bool by_64,
                                             uint64_t pol) {
    if (by_64) {
        if constexpr (PAIR) tma_load_4d_pair(dst, map, bar, 0, y, z, col / 64, pol);
        else tma_load_4d(dst, map, bar, 0, y, z, col / 64, pol);
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if constexpr (PAIR) tma_load_3d_pair(dst + i * 64 * 128, map, bar, col + 64 * i, y, z, pol);
            else tma_load_3d(dst + i * 64 * 128, map, bar, col + 64 * i, y, z, pol);
        }
    }
}

// ---- C.  The TMEM lanes lie along C's rows and the columns are rows of C, so
// that a register of a warp is 32 neighbouring elements, stored as they are, at
// any alignment.  (An earlier form of the kernels stored through shared memory, by
// TMA or 16 bytes a lane, for no gain; that was within what boxes differ by and has
// not been tried in this form.)
//
// A warp's share (every other 32) of `cols` columns of 32 TMEM lanes.  at: the element of C of lane 0 and column 0; `lanes` of the lanes are inside.  zero:
// there was nothing to sum.  released(): the accumulator has been read.
template <typename T, typename Released>
__device__ __forceinline__ void store_tile(const GroupedParams &p, int64_t at, uint32_t taddr, int lanes, int cols, bool zero,
                                           int lane, Released released) {
    if (lanes <= 0) cols = 0;
    const int half = (static_cast<int>(threadIdx.x >> 5) - 2) >> 2;  // of the two warps of a quarter
    for (int c = 32 * half; c < cols; c += 64) {
        uint32_t v[32];
        if (!zero) {
            tmem_load_32(taddr + static_cast<uint32_t>(c), v);
            tmem_load_wait();
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        if (c + 64 >= cols) released();
        if (lane < lanes) {
            T *to = static_cast<T *>(p.c) + at + c * p.ldc + lane;
            if (cols - c >= 32) {
#pragma unroll
                for (int i = 0; i < 32; ++i, to += p.ldc) from_float(__uint_as_float(v[i]), *to);
            } else {
#pragma unroll
                for (int i = 0; i < 32; ++i, to += p.ldc)
                    if (i < cols - c) from_float(__uint_as_float(v[i]), *to);
            }
        }
        __syncwarp();  // TMEM is read by whole warps
    }
    if (32 * half >= cols) released();  // no share in this tile
}

template <typename Released>
__device__ __forceinline__ void store_any_tile(const GroupedParams &p, int64_t at, uint32_t taddr, int lanes, int cols, bool zero,
                                               int lane, Released released) {
    if (p.c_dtype == ST_F32) store_tile<float>(p, at, taddr, lanes, cols, zero, lane, released);
    else if (p.c_dtype == ST_F16) store_tile<__half>(p, at, taddr, lanes, cols, zero, lane, released);
    else store_tile<__nv_bfloat16>(p, at, taddr, lanes, cols, zero, lane, released);
}

// Rows [first, p.rows) of C, which belong to no group, become 0: a row a CTA.
template <int THREADS>
__device__ __forceinline__ void zero_rows(const GroupedParams &p, int first, int thread) {
    const int es = p.c_dtype == ST_F32 ? 4 : 2;
    const bool wide = reinterpret_cast<uintptr_t>(p.c) % 16 == 0 && p.ldc * es % 16 == 0;
    for (int64_t r = first + static_cast<int64_t>(blockIdx.x); r < p.rows; r += gridDim.x) {
        uint8_t *row = static_cast<uint8_t *>(p.c) + r * p.ldc * es;
        const int64_t bytes = static_cast<int64_t>(p.n) * es, whole = wide ? bytes / 16 * 16 : 0;
        for (int64_t i = 16 * thread; i < whole; i += 16 * THREADS) *reinterpret_cast<uint4 *>(row + i) = make_uint4(0, 0, 0, 0);
        for (int64_t i = whole + 2 * thread; i < bytes; i += 2 * THREADS) *reinterpret_cast<uint16_t *>(row + i) = 0;
    }
}

// ---------------------------------------------------------------- one CTA, 128 x BN tiles
template <int BN>
struct GroupedCfg {
    static constexpr int kRows = 128;
    static constexpr int kThreads = 32 * (2 + kOutWarps);
    static constexpr int kRowBytes = kRows * kBK * 2;
    static constexpr int kColBytes = BN * kBK * 2;
    static constexpr int kStageBytes = kRowBytes + kColBytes;
    static constexpr int kStages = BN == 128 ? 6 : 9;
    static constexpr int kTmemCols = 2 * BN;
    static constexpr int kSmemBytes =
        kStages * kStageBytes + static_cast<int>(sizeof(GroupTable)) + kBarBytes + 1024;
    static_assert(kSmemBytes <= 232448, "over the per-block shared memory limit");
    static_assert(kStages * kStageBytes >= kRows * (BN + 4 * 8) * 4, "the ring holds eight parts' sums of its columns");
};

// SPLIT: a cluster of p.split CTAs takes one tile, each every split-th step of
// its contraction; the sums are added in order through distributed shared memory.
template <int BN, bool WEIGHTS, bool R_MN, bool SPLIT>
__global__ void __launch_bounds__(GroupedCfg<BN>::kThreads, 1)
    gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ ColumnMaps maps_c,
                        const GroupedParams p) {
    using Cfg = GroupedCfg<BN>;
    static_assert(!WEIGHTS || R_MN, "both operands of the second form lie along their columns");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    GroupTable &table = *reinterpret_cast<GroupTable *>(smem + Cfg::kStages * Cfg::kStageBytes);
    uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(&table) + sizeof(GroupTable));
    constexpr int kBars = 2 * Cfg::kStages + 5;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);  // uniform registers for what follows from it
    const int lane = threadIdx.x & 31;
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (Cfg::kStages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * Cfg::kStages + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * Cfg::kStages + 2 + a); };
    const uint32_t drain_bar = bar0 + 8u * (kBars - 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), kOutWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0 && p.reads) {
        tma_prefetch_map(&tmap_r);
        tma_prefetch_map(&maps_c.by32[0]);
    }
    if (warp == 1) {
        tmem_alloc(smem_addr(tmem_slot), Cfg::kTmemCols);
        tmem_relinquish();
    }
    pdl_begin();  // nothing above touches global memory
    if (warp == 0) build_table<WEIGHTS, BN>(table, p, lane);
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    const int split = SPLIT ? p.split : 1, part = SPLIT ? static_cast<int>(cluster_rank()) : 0;
    using Walk = TileWalk<WEIGHTS, Cfg::kRows, BN>;
    Walk walk(static_cast<int>(blockIdx.x) / split, static_cast<int>(gridDim.x) / split);
    Tile tile;
    auto my_blocks = [&](const Tile &of) { return SPLIT ? (of.blocks - part + split - 1) / split : of.blocks; };
    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_last();
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            while (ok && walk.next(table, p, tile)) {
                const int high = (tile.cols + 31) / 32;  // rows of the column operand's box, in 32
                for (int b = part; b < tile.blocks; b += split, ++issued) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = full_bar(s);
                    const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                    if constexpr (WEIGHTS) {
                        mbar_arrive_expect_tx(fb, Cfg::kStageBytes);
                        static_assert(!WEIGHTS || BN == 128, "columns in two 64s");
                        load_columns<false>(sr, &tmap_r, fb, tile.r0, tile.first + b * kBK, 0, p.r_by_64, pol);
                        load_columns<false>(sc, &maps_c.by32[0], fb, tile.c0, tile.first + b * kBK, 0, p.c_by_64, pol);
                    } else {
                        mbar_arrive_expect_tx(fb, static_cast<uint32_t>(Cfg::kRowBytes + high * 32 * 128));
                        const int g = p.b_groups ? tile.group : 0;
                        if constexpr (R_MN) {
                            load_columns<false>(sr, &tmap_r, fb, tile.r0, b * kBK, g, p.r_by_64, pol);
                        } else {
                            tma_load_3d(sr, &tmap_r, fb, b * kBK, tile.r0, g, pol);
                        }
                        tma_load_2d(sc, &maps_c.by32[high - 1], fb, b * kBK, tile.c0, pol);
                    }
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
            drain_ring(issued, Cfg::kStages, full_bar, p.timeout_ns);
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer
        int s = 0, a = 0;
        uint32_t ph = 0, aph = 0;
        bool ok = true;
        while (ok && walk.next(table, p, tile)) {
            const int blocks = my_blocks(tile);
            if (blocks == 0) continue;
            const uint32_t idesc = p.idesc | Walk::idesc_n(WEIGHTS ? BN : tile.cols);
            if (!__all_sync(0xffffffffu, mbar_wait(tempty_bar(a), aph ^ 1u, abort_flag, p.timeout_ns))) {
                ok = false;
                break;
            }
            for (int b = 0; b < blocks; ++b) {
                if (!__all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns))) {
                    ok = false;
                    break;
                }
                const Step step(WEIGHTS ? tile.rows - (part + b * split) * kBK : kBK);
                if (WEIGHTS && step.mixed) zero_behind(smem_addr(smem + s * Cfg::kStageBytes), tile.rows % kBK, lane);
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                    const uint64_t dr = smem_desc_sw128(sr, R_MN ? 64 * 128 : 16, 1024);
                    const uint64_t dc = smem_desc_sw128(sc, WEIGHTS ? 64 * 128 : 16, 1024);
#pragma unroll
                    for (int j = 0; j < kBK / kMmaK; ++j)
                        if (!WEIGHTS || j < step.mmas)
                            tc_mma<false>(tmem_base + static_cast<uint32_t>(a * BN), dr + j * ((R_MN ? kMmaK * 128 : 32) >> 4),
                                          dc + j * ((WEIGHTS ? kMmaK * 128 : 32) >> 4), idesc, (b | j) != 0 ? 1u : 0u);
                    tc_commit(empty_bar(s));
                    if (b + 1 == blocks) tc_commit(tfull_bar(a));
                }
                __syncwarp();
                if (++s == Cfg::kStages) {
                    s = 0;
                    ph ^= 1u;
                }
            }
            if (++a == 2) {
                a = 0;
                aph ^= 1u;
            }
        }
        if (!ok) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(p.err, kDevAbortGemmMma);
        }
        if (elect_one()) tc_commit(drain_bar);
        __syncwarp();
        drain_ring(1, 1, [&](int) { return drain_bar; }, p.timeout_ns);  // the MMAs read shared memory and write TMEM
    } else if constexpr (!SPLIT) {
        // ------------------------------------------------ C
        const int g = warp & 3;
        int a = 0;
        uint32_t aph = 0;
        while (walk.next(table, p, tile)) {
            const bool zero = tile.blocks == 0;
            if (!zero) {
                if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(a), aph, abort_flag, p.timeout_ns))) {
                    *abort_flag = 1;
                    if (lane == 0) atomicExch(p.err, kDevAbortGemmEpilogue);
                    break;
                }
                tc_fence_after_sync();
            }
            const int r = tile.r0 + 32 * g;
            const int64_t at = (WEIGHTS ? tile.group * p.c_g : 0) + tile.c0 * p.ldc + r;
            store_any_tile(p, at, tmem_base + (static_cast<uint32_t>(g * 32) << 16) + static_cast<uint32_t>(a * BN), p.n - r,
                           tile.cols, zero, lane, [&] {
                               if (zero) return;
                               tc_fence_before_sync();
                               __syncwarp();
                               if (lane == 0) mbar_arrive(tempty_bar(a));
                           });
            if (!zero && ++a == 2) {
                a = 0;
                aph ^= 1u;
            }
        }
    }
    if constexpr (SPLIT) {
        // ------------------------------------------------ C of the cluster's tile
        Walk again(static_cast<int>(blockIdx.x) / split, static_cast<int>(gridDim.x) / split);
        const bool any = again.next(table, p, tile);
        const int g = warp & 3, half = (warp - 2) >> 2;
        const bool out = warp >= 2, zero = !any || my_blocks(tile) == 0;
        if (out && !zero) {
            if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(0), 0, abort_flag, p.timeout_ns))) {
                *abort_flag = 1;
                if (lane == 0) atomicExch(p.err, kDevAbortGemmEpilogue);
            }
            tc_fence_after_sync();
        }
        __syncwarp();
        cluster_sync();  // every MMA of the cluster has read its ring
        // A part owns `own` columns of the tile and gets them as [part][128 lanes][own + 4 columns].  (As [column][lane],
        // one value a lane and store, the exchange of 64 columns between two parts took 5 us more.)
        const int own = BN / split, own_shift = 31 - __clz(own), pitch = own + 4;  // split is a power of two
        if (out && any) {
            const uint32_t mine = smem_addr(smem) + 4u * static_cast<uint32_t>((part * 128 + 32 * g + lane) * pitch);
            for (int c = 32 * half; c < tile.cols; c += 64) {
                uint32_t v[32];
                if (!zero) {
                    tmem_load_32(tmem_base + (static_cast<uint32_t>(g * 32) << 16) + static_cast<uint32_t>(c), v);
                    tmem_load_wait();
                } else {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] = 0u;
                }
#pragma unroll
                for (int i = 0; i < 32; i += 4) {
                    const int col = c + i;
                    st_cluster_v4(map_to_rank(mine, static_cast<uint32_t>(col >> own_shift)) + 4u * static_cast<uint32_t>(col & (own - 1)),
                                  __uint_as_float(v[i]), __uint_as_float(v[i + 1]), __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
                }
                __syncwarp();
            }
        }
        __syncwarp();
        cluster_sync();
        if (out && any) {
            const int id = (warp - 2) * 32 + lane, n = tile.r0 + (id & 127);
            const float *sums = reinterpret_cast<const float *>(smem) + (id & 127) * pitch;
            const int64_t at = (WEIGHTS ? tile.group * p.c_g : 0) + tile.c0 * p.ldc + n;
            if (n < p.n)
                for (int j = 4 * (id >> 7); j < own && part * own + j < tile.cols; j += kOutWarps) {
                    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (int q = 0; q < split; ++q) {
                        const float4 x = *reinterpret_cast<const float4 *>(sums + q * 128 * pitch + j);
                        v[0] += x.x;
                        v[1] += x.y;
                        v[2] += x.z;
                        v[3] += x.w;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (part * own + j + i >= tile.cols) break;
                        const int64_t to = at + (part * own + j + i) * p.ldc;
                        if (p.c_dtype == ST_F32) static_cast<float *>(p.c)[to] = v[i];
                        else if (p.c_dtype == ST_F16) from_float(v[i], static_cast<__half *>(p.c)[to]);
                        else from_float(v[i], static_cast<__nv_bfloat16 *>(p.c)[to]);
                    }
                }
        }
    }
    if (!WEIGHTS && p.zero_rest && warp >= 2)
        zero_rows<32 * kOutWarps>(p, p.groups > 0 ? table.row_end[p.groups - 1] : 0, (warp - 2) * 32 + lane);
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after_sync();
        tmem_dealloc(tmem_base, Cfg::kTmemCols);
    }
}

// ---------------------------------------------------------------- CTA pairs, 256 x 256 tiles
// Groups of many rows.  A pair of CTAs (cta_group::2) computes 256 x 256 of C:
// each holds 128 rows of A and 128 columns of B, half of the loads per SM and
// MMA that 128 x 128 tiles of one CTA take.
//
// full[s] lives in the even CTA and counts both CTAs' loads; the even CTA's
// MMA warp commits empty[s] and tfull[a] to both CTAs; tempty[a] lives in the
// even CTA and counts the pair's warps that read accumulators.  A step whose
// rows are mixed (second form): the odd CTA's loads complete its own landed[s],
// its second warp sets the rows behind the group to zero and arrives at the even
// CTA's cleared[s].
struct GroupedPairCfg {
    static constexpr int kRows = 256, kCols = 256;
    static constexpr int kThreads = 32 * (2 + kOutWarps);
    static constexpr int kRowBytes = 128 * kBK * 2;
    static constexpr int kColBytes = 128 * kBK * 2;
    static constexpr int kStageBytes = kRowBytes + kColBytes;
    static constexpr int kStages = 6;
    static constexpr int kTmemCols = 2 * kCols;
    static constexpr int kSmemBytes =
        kStages * kStageBytes + static_cast<int>(sizeof(GroupTable)) + kBarBytes + 1024;
    static_assert(kSmemBytes <= 232448, "over the per-block shared memory limit");
};

template <bool WEIGHTS, bool R_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GroupedPairCfg::kThreads, 1)
    gemm_grouped_pair_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ ColumnMaps maps_c,
                             const GroupedParams p) {
    using Cfg = GroupedPairCfg;
    static_assert(!WEIGHTS || R_MN, "both operands of the second form lie along their columns");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    GroupTable &table = *reinterpret_cast<GroupTable *>(smem + Cfg::kStages * Cfg::kStageBytes);
    uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(&table) + sizeof(GroupTable));
    constexpr int kBars = 4 * Cfg::kStages + 5;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (Cfg::kStages + s); };
    auto tfull_bar = [&](int a) { return bar0 + 8u * (2 * Cfg::kStages + a); };
    auto tempty_bar = [&](int a) { return bar0 + 8u * (2 * Cfg::kStages + 2 + a); };
    auto landed_bar = [&](int s) { return bar0 + 8u * (2 * Cfg::kStages + 4 + s); };
    auto cleared_bar = [&](int s) { return bar0 + 8u * (3 * Cfg::kStages + 4 + s); };
    const uint32_t drain_bar = bar0 + 8u * (kBars - 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
            mbar_init(landed_bar(s), 1);
            mbar_init(cleared_bar(s), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), 2 * kOutWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0 && p.reads) {
        tma_prefetch_map(&tmap_r);
        tma_prefetch_map(&maps_c.by32[0]);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_addr(tmem_slot), Cfg::kTmemCols);
        tmem_relinquish_pair();
    }
    pdl_begin();  // nothing above touches global memory
    if (warp == 0) build_table<WEIGHTS, Cfg::kCols>(table, p, lane);
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);

    using Walk = TileWalk<WEIGHTS, Cfg::kRows, Cfg::kCols>;
    Walk walk(static_cast<int>(blockIdx.x >> 1), static_cast<int>(gridDim.x >> 1));
    Tile tile;
    if (warp == 0) {
        // ------------------------------------------------ TMA producer (both CTAs)
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_last();
            const uint32_t even_full0 = map_to_rank(full_bar(0), 0);
            const int half = static_cast<int>(rank) * 128;
            int s = 0, issued = 0;
            uint32_t ph = 0, uses = 0, landed_ph = 0;  // a bit for each landed[s]: waited for, and its next parity
            bool ok = true;
            while (ok && walk.next(table, p, tile)) {
                // each CTA brings half of the tile's columns (rows of A)
                const int half_c = (tile.cols + 31) / 32 * 16, high = (half_c + 31) / 32;
                for (int b = 0; b < tile.blocks; ++b, ++issued) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = even_full0 + 8u * s;
                    const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                    if constexpr (WEIGHTS) {
                        const Step step(tile.rows - b * kBK);
                        const int y = tile.first + b * kBK;
                        uint32_t bar = fb;
                        if (rank == 0) {
                            mbar_arrive_expect_tx(full_bar(s), step.mixed ? Cfg::kStageBytes : 2 * Cfg::kStageBytes);
                        } else if (step.mixed) {
                            bar = landed_bar(s);
                            mbar_arrive_expect_tx(bar, Cfg::kStageBytes);
                            uses |= 1u << s;
                            landed_ph ^= 1u << s;
                        }
                        load_columns<true>(sr, &tmap_r, bar, tile.r0 + half, y, 0, p.r_by_64, pol);
                        load_columns<true>(sc, &maps_c.by32[0], bar, tile.c0 + half, y, 0, p.c_by_64, pol);
                    } else {
                        if (rank == 0)
                            mbar_arrive_expect_tx(full_bar(s), static_cast<uint32_t>(2 * (Cfg::kRowBytes + high * 32 * 128)));
                        const int g = p.b_groups ? tile.group : 0;
                        if constexpr (R_MN) {
                            load_columns<true>(sr, &tmap_r, fb, tile.r0 + half, b * kBK, g, p.r_by_64, pol);
                        } else {
                            tma_load_3d_pair(sr, &tmap_r, fb, b * kBK, tile.r0 + half, g, pol);
                        }
                        tma_load_2d_pair(sc, &maps_c.by32[high - 1], fb, b * kBK, tile.c0 + static_cast<int>(rank) * half_c, pol);
                    }
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
            if constexpr (WEIGHTS) {
                const volatile int never = 0;
                for (int i = 0; i < Cfg::kStages; ++i)  // copies that landed[i] counts
                    if (uses >> i & 1u) (void)mbar_wait(landed_bar(i), (landed_ph >> i & 1u) ^ 1u, &never, p.timeout_ns);
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer (even CTA)
        if (rank == 0) {
            int s = 0, a = 0;
            uint32_t ph = 0, aph = 0, cleared_ph = 0;  // a bit for each cleared[s]
            bool ok = true;
            while (ok && walk.next(table, p, tile)) {
                if (tile.blocks == 0) continue;
                const uint32_t idesc = p.idesc | Walk::idesc_n(WEIGHTS ? Cfg::kCols : tile.cols);
                if (!__all_sync(0xffffffffu, mbar_wait(tempty_bar(a), aph ^ 1u, abort_flag, p.timeout_ns))) {
                    ok = false;
                    break;
                }
                for (int b = 0; b < tile.blocks; ++b) {
                    if (!__all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns))) {
                        ok = false;
                        break;
                    }
                    const Step step(WEIGHTS ? tile.rows - b * kBK : kBK);
                    if (WEIGHTS && step.mixed) {
                        zero_behind(smem_addr(smem + s * Cfg::kStageBytes), tile.rows % kBK, lane);
                        if (!__all_sync(0xffffffffu, mbar_wait_cluster(cleared_bar(s), cleared_ph >> s & 1u, abort_flag, p.timeout_ns))) {
                            ok = false;
                            break;
                        }
                        cleared_ph ^= 1u << s;
                    }
                    tc_fence_after_sync();
                    if (elect_one()) {
                        const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                        const uint64_t dr = smem_desc_sw128(sr, R_MN ? 64 * 128 : 16, 1024);
                        const uint64_t dc = smem_desc_sw128(sc, WEIGHTS ? 64 * 128 : 16, 1024);
#pragma unroll
                        for (int j = 0; j < kBK / kMmaK; ++j)
                            if (!WEIGHTS || j < step.mmas)
                                tc_mma_pair<false>(tmem_base + static_cast<uint32_t>(a * Cfg::kCols),
                                                   dr + j * ((R_MN ? kMmaK * 128 : 32) >> 4),
                                                   dc + j * ((WEIGHTS ? kMmaK * 128 : 32) >> 4), idesc, (b | j) != 0 ? 1u : 0u);
                        tc_commit_pair_multicast(empty_bar(s), 3);
                        if (b + 1 == tile.blocks) tc_commit_pair_multicast(tfull_bar(a), 3);
                    }
                    __syncwarp();
                    if (++s == Cfg::kStages) {
                        s = 0;
                        ph ^= 1u;
                    }
                }
                if (++a == 2) {
                    a = 0;
                    aph ^= 1u;
                }
            }
            if (!ok) {
                *abort_flag = 1;
                if (lane == 0) atomicExch(p.err, kDevAbortGemmMma);
            }
            if (elect_one()) tc_commit_pair(drain_bar);
            __syncwarp();
            drain_ring(1, 1, [&](int) { return drain_bar; }, p.timeout_ns);  // the MMAs read shared memory and write TMEM
        } else if constexpr (WEIGHTS) {
            // -------------------------------------------- zeros behind a group's last rows (odd CTA)
            const uint32_t even_cleared0 = map_to_rank(cleared_bar(0), 0);
            int s = 0;
            uint32_t landed_ph = 0;
            bool ok = true;
            while (ok && walk.next(table, p, tile)) {
                for (int b = 0; b < tile.blocks; ++b) {
                    if (Step(tile.rows - b * kBK).mixed) {
                        if (!__all_sync(0xffffffffu, mbar_wait(landed_bar(s), landed_ph >> s & 1u, abort_flag, p.timeout_ns))) {
                            ok = false;
                            break;
                        }
                        landed_ph ^= 1u << s;
                        zero_behind(smem_addr(smem + s * Cfg::kStageBytes), tile.rows % kBK, lane);
                        if (lane == 0) mbar_arrive_cluster_release(even_cleared0 + 8u * s);
                    }
                    if (++s == Cfg::kStages) s = 0;
                }
            }
            if (!ok) {
                *abort_flag = 1;
                if (lane == 0) atomicExch(p.err, kDevAbortGemmMma);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------------------------ C (both CTAs)
        const int g = warp & 3, row = static_cast<int>(rank) * 128 + 32 * g;
        const uint32_t even_tempty0 = map_to_rank(tempty_bar(0), 0);
        int a = 0;
        uint32_t aph = 0;
        while (walk.next(table, p, tile)) {
            const bool zero = tile.blocks == 0;
            if (!zero) {
                if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(a), aph, abort_flag, p.timeout_ns))) {
                    *abort_flag = 1;
                    if (lane == 0) atomicExch(p.err, kDevAbortGemmEpilogue);
                    break;
                }
                tc_fence_after_sync();
            }
            const int r = tile.r0 + row;
            const int64_t at = (WEIGHTS ? tile.group * p.c_g : 0) + tile.c0 * p.ldc + r;
            store_any_tile(p, at, tmem_base + (static_cast<uint32_t>(g * 32) << 16) + static_cast<uint32_t>(a * Cfg::kCols), p.n - r,
                           tile.cols, zero, lane, [&] {
                               if (zero) return;
                               tc_fence_before_sync();
                               __syncwarp();
                               if (lane == 0) {
                                   if (rank == 0) mbar_arrive(tempty_bar(a));
                                   else mbar_arrive_cluster(even_tempty0 + 8u * a);
                               }
                           });
            if (!zero && ++a == 2) {
                a = 0;
                aph ^= 1u;
            }
        }
        if (!WEIGHTS && p.zero_rest)
            zero_rows<32 * kOutWarps>(p, p.groups > 0 ? table.row_end[p.groups - 1] : 0, (warp - 2) * 32 + lane);
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

// Dense copy of strided 16-bit matrices, one for each group, into rows of `ld`
// elements (a multiple of 8), padding columns zeroed: 8 elements a thread, put
// together from the aligned words that hold them where they lie together.
struct Repack {
    const uint16_t *src;
    int64_t sg, s0, s1;  // element strides of groups, rows and columns
    int64_t groups, rows, cols;
    uint16_t *dst;
    int64_t ld;
};
// Both operands' copies in one launch, one for each blockIdx.y (1003 rows on 7 groups of 1001 x 515, both off their
// boundaries: 19.4 us a call in two launches, 18.5 in one).
struct Repacks {
    Repack of[2];
};

__global__ void __launch_bounds__(256) repack_groups_kernel(const __grid_constant__ Repacks both) {
    pdl_wait();
    const Repack &m = both.of[blockIdx.y];
    const int64_t per_row = m.ld / 8, total = m.groups * m.rows * per_row;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t line = i / per_row, c = (i - line * per_row) * 8, g = line / m.rows, r = line - g * m.rows;
        const uint16_t *from = m.src + g * m.sg + r * m.s0 + c * m.s1;
        const int n = m.cols - c < 8 ? static_cast<int>(m.cols - c) : 8;
        uint32_t w[4] = {0, 0, 0, 0};
        if (m.s1 == 1) {
            const uint32_t *words = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(from) & ~uintptr_t(3));
            const int odd = static_cast<int>(reinterpret_cast<uintptr_t>(from) >> 1) & 1, have = (odd + n + 1) / 2;
            uint32_t x[5];
#pragma unroll
            for (int j = 0; j < 5; ++j) x[j] = j < have ? __ldg(words + j) : 0u;  // only words with an element of the row
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                w[j] = __funnelshift_r(x[j], x[j + 1], 16 * odd);
                if (2 * j + 1 >= n) w[j] = 2 * j < n ? w[j] & 0xffffu : 0u;
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < n) w[j / 2] |= static_cast<uint32_t>(__ldg(from + j * m.s1)) << (16 * (j % 2));
        }
        reinterpret_cast<uint4 *>(m.dst)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- host side
int checked(const char *what) {
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), what);
}

// Matrices [groups][outer][inner] as TMA reads them: the inner dimension
// contiguous, everything on 16-byte boundaries, no two rows sharing memory;
// any other is copied first.
struct Matrices {
    const void *data;
    int64_t groups, outer, inner;
    int64_t sg, so, si;  // element strides
    bool copy = false;
    int64_t copied() const { return copy ? (groups * outer * ((inner + 7) / 8 * 8) * 2 + 255) / 256 * 256 : 0; }
};

Matrices layout(const void *data, int64_t groups, int64_t outer, int64_t inner, int64_t sg, int64_t so, int64_t si) {
    Matrices m{data, groups, outer, inner, sg, so, si};
    auto fits = [](int64_t stride, int64_t extent, int64_t least) {
        return extent == 1 || (stride >= least && stride % 8 == 0 && stride < (int64_t(1) << 38));
    };
    m.copy = !(reinterpret_cast<uintptr_t>(data) % 16 == 0 && (si == 1 || inner == 1) && fits(so, outer, inner) &&
               fits(sg, groups, 8));
    return m;
}

// The operands as the maps take them, copied where they have to be.
int copy_in(Matrices &a, Matrices &b, uint8_t *ws, int sm_count, cudaStream_t stream) {
    Repacks copies{};
    int n = 0;
    int64_t work = 0;
    for (Matrices *m : {&a, &b}) {
        if (m->copy) {
            const int64_t ld = (m->inner + 7) / 8 * 8, mine = cdiv(m->groups * m->outer * (ld / 8), 256);
            copies.of[n++] = Repack{static_cast<const uint16_t *>(m->data), m->sg, m->so, m->si, m->groups, m->outer, m->inner,
                                    reinterpret_cast<uint16_t *>(ws), ld};
            work = mine > work ? mine : work;
            m->data = ws;
            ws += m->copied();
            m->so = ld;
            m->sg = m->outer * ld;
        }
        m->si = 1;
        // strides that are never used still have to be valid ones
        if (m->outer == 1) m->so = (m->inner + 7) / 8 * 8;
        if (m->groups == 1) m->sg = (m->outer * m->so + 7) / 8 * 8;
    }
    if (n == 0) return ST_OK;
    const int64_t most = static_cast<int64_t>(sm_count) * 8;
    const dim3 grid(static_cast<unsigned>(work < most ? work : most), static_cast<unsigned>(n));
    ST_CUDA_TRY(launch_kernel(repack_groups_kernel, grid, 256, 0, stream, copies));
    return checked("repack_groups_kernel");
}

struct Operands {
    Matrices a, b;
    bool b_mn;
    int b_groups;
};

Operands operands_of(const GroupedArgs &g) {
    Operands o{};
    if (g.weights) {
        o.a = layout(g.a, 1, g.rows, g.k, 0, g.a_s0, g.a_s1);
        o.b = layout(g.b, 1, g.rows, g.n, 0, g.b_s0, g.b_s1);
        o.b_mn = true;
        return o;
    }
    o.a = layout(g.a, 1, g.rows, g.k, 0, g.a_s0, g.a_s1);
    o.b_groups = g.b_g != 0 && g.groups > 1;
    const int64_t groups = o.b_groups ? g.groups : 1;
    // along K or along N, whichever needs no copy; else along whichever is contiguous
    const Matrices by_k = layout(g.b, groups, g.n, g.k, g.b_g, g.b_s1, g.b_s0), by_n = layout(g.b, groups, g.k, g.n, g.b_g, g.b_s0, g.b_s1);
    o.b_mn = by_k.copy && (!by_n.copy || g.b_s1 == 1);
    o.b = o.b_mn ? by_n : by_k;
    return o;
}

int make_map_16(CUtensorMap *map, int dtype, const char *what, int rank, const void *data, int64_t d0, int64_t d1, int64_t d2,
                int64_t s1, int64_t s2, int b0, int b1) {
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(d0), static_cast<cuuint64_t>(d1), static_cast<cuuint64_t>(d2)};
    const cuuint64_t strides[2] = {static_cast<cuuint64_t>(s1 * 2), static_cast<cuuint64_t>(s2 * 2)};
    const cuuint32_t box[3] = {static_cast<cuuint32_t>(b0), static_cast<cuuint32_t>(b1), 1};
    return make_tensor_map(map, what, dtype == ST_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank,
                           data, dims, strides, box);
}

// (column, y, z) for load_columns: whole 64s as (column in a 64, y, z, 64), any other as three dimensions.
int make_map_columns(CUtensorMap *map, int *by_64, int dtype, const char *what, const void *data, int64_t cols, int64_t y, int64_t z,
                     int64_t sy, int64_t sz) {
    *by_64 = cols % 64 == 0;
    if (!*by_64) return make_map_16(map, dtype, what, 3, data, cols, y, z, sy, sz, 64, kBK);
    const cuuint64_t dims[4] = {64, static_cast<cuuint64_t>(y), static_cast<cuuint64_t>(z), static_cast<cuuint64_t>(cols / 64)};
    const cuuint64_t strides[3] = {static_cast<cuuint64_t>(sy * 2), static_cast<cuuint64_t>(sz * 2), 128};
    const cuuint32_t box[4] = {64, kBK, 1, 2};
    return make_tensor_map(map, what, dtype == ST_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, data,
                           dims, strides, box);
}

template <int BN, bool WEIGHTS, bool R_MN, bool SPLIT>
int launch_instance(const CUtensorMap &mr, const ColumnMaps &mc, const GroupedParams &p, int64_t most_tiles, int sm_count,
                    cudaStream_t stream) {
    using Cfg = GroupedCfg<BN>;
    auto kern = gemm_grouped_kernel<BN, WEIGHTS, R_MN, SPLIT>;
    static uint64_t attr_set = 0;  // one bit per device ordinal
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    const int64_t tiles = most_tiles < 1 ? 1 : most_tiles;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(SPLIT ? tiles * p.split : tiles < sm_count ? tiles : sm_count));
    cfg.blockDim = dim3(Cfg::kThreads);
    cfg.dynamicSmemBytes = Cfg::kSmemBytes;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (pdl_enabled()) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (SPLIT) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = static_cast<unsigned>(p.split);
        attr[n].val.clusterDim.y = 1;
        attr[n++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    ST_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, mr, mc, p));
    return checked("gemm_grouped_kernel");
}

template <int BN, bool WEIGHTS, bool R_MN>
int launch_single(const CUtensorMap &mr, const ColumnMaps &mc, const GroupedParams &p, int64_t most_tiles, int sm_count,
                  cudaStream_t stream) {
    return p.split > 1 ? launch_instance<BN, WEIGHTS, R_MN, true>(mr, mc, p, most_tiles, sm_count, stream)
                       : launch_instance<BN, WEIGHTS, R_MN, false>(mr, mc, p, most_tiles, sm_count, stream);
}

template <bool WEIGHTS, bool R_MN>
int launch_pair_instance(const CUtensorMap &mr, const ColumnMaps &mc, const GroupedParams &p, int64_t most_tiles, int sm_count,
                         cudaStream_t stream) {
    using Cfg = GroupedPairCfg;
    auto kern = gemm_grouped_pair_kernel<WEIGHTS, R_MN>;
    static uint64_t attr_set = 0;  // one bit per device ordinal
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    const int64_t pairs = most_tiles < 1 ? 1 : most_tiles < sm_count / 2 ? most_tiles : sm_count / 2;
    ST_CUDA_TRY(launch_kernel(kern, static_cast<unsigned>(2 * pairs), Cfg::kThreads, Cfg::kSmemBytes, stream, mr, mc, p));
    return checked("gemm_grouped_pair_kernel");
}

// Most tiles that there can be, however the ends divide the rows: m groups of a
// row each, and a tile more for each `cols` of the other rows.
int64_t most_tiles(const GroupedArgs &g, int64_t tiles_r, int cols) {
    if (g.weights) return tiles_r * g.groups * cdiv(g.k, cols);
    const int64_t m = g.groups < g.rows ? g.groups : g.rows;
    return tiles_r * ((g.rows - m) / cols + m);
}

// Tile shape and split: the least estimated time for groups of equal size (what
// the ends hold is not known here).  The figures are microseconds fitted to
// B200 timings of 1 x 4096 x 1024 to 16384 rows on 32 groups of 4096 x 4096: a
// stage of 64 along the contraction, which few columns of a tile leave bound by
// the SM's loads; a tile's way out, beside the next tile's stages; the join of
// parts.  (32 rows of 8192 x 512, in a replayed graph: 33 us on 32 columns, with
// 8 parts estimated 10.8, measured 10.3.)
struct GroupedPlan {
    bool pair = false;
    int cols = 128;  // most columns of a tile
    int split = 1;
    double us = 1e300;
};

GroupedPlan plan_grouped(const GroupedArgs &g, int sm_count) {
    const int64_t met = g.groups < 1 ? 1 : !g.weights && g.rows < g.groups ? (g.rows > 0 ? g.rows : 1) : g.groups;
    const int64_t per_group = cdiv(g.rows > 0 ? g.rows : 1, met), blocks = cdiv(g.weights ? per_group : g.k, kBK);
    constexpr double kLaunch = 2.5;
    GroupedPlan best;
    auto offer = [&](bool pair, int cols, int split) {
        const int64_t extent = g.weights ? g.k : per_group, tiles_c = cdiv(extent, cols), tiles_r = cdiv(g.n, pair ? 256 : 128);
        const double c = g.weights ? cols : static_cast<double>(cdiv(cdiv(extent, tiles_c), pair ? 32 : 16) * (pair ? 32 : 16));
        const double stage = pair ? (c > 168 ? 0.00125 * c : 0.21) : 0.235 + 0.0004 * c, out = pair ? 0.5 + 0.006 * c : 0.4 + 0.006 * c;
        const double sums = static_cast<double>(cdiv(blocks, split)) * stage;
        double us;
        if (split > 1) {  // every tile that there can be has a cluster, met or not
            const double join[2][3] = {{3.8, 4.5, 4.5}, {6.2, 6.2, 7.5}};
            const int64_t at_once = split == 8 ? 120 : split == 4 ? 140 : sm_count, ctas = most_tiles(g, tiles_r, cols) * split;
            if (split > blocks || ctas > 4 * at_once) return;
            us = static_cast<double>(cdiv(ctas, at_once)) * (kLaunch + sums + join[cols == 128][split == 2 ? 0 : split == 4 ? 1 : 2]);
        } else {
            us = kLaunch + static_cast<double>(cdiv(met * tiles_c * tiles_r, pair ? sm_count / 2 : sm_count)) * (sums > out ? sums : out) + out;
        }
        if (us < best.us) best = GroupedPlan{pair, cols, split, us};
    };
    for (int split = 1; split <= 8; split *= 2) {
        if (!g.weights) offer(false, 32, split);
        offer(false, 128, split);
    }
    offer(true, GroupedPairCfg::kCols, 1);
    return best;
}

}  // namespace

int64_t gemm_grouped_workspace_bytes(const GroupedArgs &g) {
    if (g.rows == 0 || g.k == 0 || g.n == 0 || g.groups == 0) return 0;
    const Operands o = operands_of(g);
    return o.a.copied() + o.b.copied();
}

int launch_gemm_grouped(const GroupedArgs &g, void *workspace, int sm_count, int *dev_err, uint64_t timeout_ns,
                        cudaStream_t stream) {
    if (g.n == 0 || (g.weights ? g.k == 0 || g.groups == 0 : g.rows == 0)) return ST_OK;
    GroupedParams p{};
    p.ends = g.ends;
    p.groups = static_cast<int>(g.groups);
    p.rows = static_cast<int>(g.rows);
    p.k = static_cast<int>(g.k);
    p.n = static_cast<int>(g.n);
    p.c = g.c;
    p.c_g = g.c_g;
    p.ldc = g.ldc;
    p.c_dtype = g.c_dtype;
    p.zero_rest = g.zero_rest;
    p.err = dev_err;
    p.timeout_ns = timeout_ns;
    const GroupedPlan plan = plan_grouped(g, sm_count);
    const bool pair = plan.pair;
    const int rows = pair ? GroupedPairCfg::kRows : 128, cols = plan.cols;
    p.tiles_r = static_cast<int>(cdiv(g.n, rows));
    p.tiles_c = static_cast<int>(cdiv(g.k, cols));
    p.split = plan.split;
    const int64_t most = most_tiles(g, p.tiles_r, cols);
    if (most > INT32_MAX / 2) return fail(ST_ERR_UNSUPPORTED, "matmul_grouped: too many output tiles");
    CUtensorMap mr{};
    ColumnMaps mc{};
    Operands o{};
    o.b_mn = g.weights;
    // with nothing to sum over (k = 0, no groups, or no rows) no operand is read
    if (g.rows > 0 && g.k > 0 && g.groups > 0) {
        o = operands_of(g);
        ST_TRY(copy_in(o.a, o.b, static_cast<uint8_t *>(workspace), sm_count, stream));
        if (g.weights) {
            ST_TRY(make_map_columns(&mr, &p.r_by_64, g.dtype, "C", o.b.data, g.n, g.rows, 1, o.b.so, o.b.sg));
            ST_TRY(make_map_columns(&mc.by32[0], &p.c_by_64, g.dtype, "A", o.a.data, g.k, g.rows, 1, o.a.so, o.a.sg));
        } else {
            for (int i = 0; i < 4; ++i)
                ST_TRY(make_map_16(&mc.by32[i], g.dtype, "A", 2, o.a.data, g.k, g.rows, 1, o.a.so, 0, kBK, 32 * (i + 1)));
            if (o.b_mn) ST_TRY(make_map_columns(&mr, &p.r_by_64, g.dtype, "B", o.b.data, g.n, g.k, o.b.groups, o.b.so, o.b.sg));
            else ST_TRY(make_map_16(&mr, g.dtype, "B", 3, o.b.data, g.k, g.n, o.b.groups, o.b.so, o.b.sg, kBK, 128));
        }
        p.b_groups = o.b_groups;
        p.reads = 1;
    }
    p.idesc = mma_idesc(g.dtype == ST_F16 ? 0 : 1, o.b_mn, g.weights, static_cast<uint32_t>(rows), 0);
    if (pair) {
        if (g.weights) return launch_pair_instance<true, true>(mr, mc, p, most, sm_count, stream);
        return o.b_mn ? launch_pair_instance<false, true>(mr, mc, p, most, sm_count, stream)
                      : launch_pair_instance<false, false>(mr, mc, p, most, sm_count, stream);
    }
    if (g.weights) return launch_single<128, true, true>(mr, mc, p, most, sm_count, stream);
    if (cols == 32)
        return o.b_mn ? launch_single<32, false, true>(mr, mc, p, most, sm_count, stream)
                      : launch_single<32, false, false>(mr, mc, p, most, sm_count, stream);
    return o.b_mn ? launch_single<128, false, true>(mr, mc, p, most, sm_count, stream)
                  : launch_single<128, false, false>(mr, mc, p, most, sm_count, stream);
}

}  // namespace st
