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
//   warps 2-5   C: TMEM -> registers -> shared memory -> rows of C, while the
//               MMAs of the next tile fill the other accumulator
//
// The kernels know a row operand (the MMA's M) and a column operand (its N).
//
// First form: B's columns are the rows of a tile and the group's rows its
// columns, 16 to 256 of them: N is a field of the MMA's descriptor, so a group
// is cut into tiles of equal size in steps of 16 and nothing is padded to 128
// or 256 rows (16384 rows on 32 groups of 4096 x 4096, between 60 and 2400
// rows each: 647 us with a group's rows as M).  The last columns of a tile may
// be rows of the next group, or what an earlier tile left in shared memory:
// columns of a product do not mix, and those are not stored.
//
// Second form: the rows are what is summed over, so a group's last, shorter
// step must read zeros beside its own rows: the row dimension of the tensor
// map is split in two of equal stride, (position in the step, first row of the
// step), and a step of n < 64 rows starts at position n - 64, whose first
// 64 - n rows lie outside of the map and read as zeros.
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

constexpr int kMaxGroups = kGroupedMaxGroups;
constexpr int kBK = 64;  // elements of the contraction a stage: 128 bytes, one swizzle span
constexpr int kMmaK = 16;
constexpr int kBarBytes = 512;
constexpr int kPitch = 36;  // floats of a staged row of 32: 16-byte reads and writes without bank conflicts

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
    int reads;           // there is something to sum over: the maps are valid
    uint32_t idesc;
    int *err;
    unsigned long long timeout_ns;
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
            out.cols = p.n - out.c0 < COLS ? p.n - out.c0 : COLS;
            out.blocks = (rows + kBK - 1) / kBK;
        } else {
            const int even = ((rows + tiles_c - 1) / tiles_c + 15) / 16 * 16;  // columns of the group's tiles
            out.c0 = begin + c * even;
            out.cols = rows - c * even < even ? rows - c * even : even;
            out.blocks = (p.k + kBK - 1) / kBK;
        }
        t += step;
        return true;
    }
};

// A warp's 32 x 32 values, staged [row][kPitch], to C: `rows` x `cols` of them
// are inside.  c points at the first one.  16-byte pieces where C allows.
template <typename T>
__device__ __forceinline__ void store_box(T *c, int64_t ldc, const float *box, int rows, int cols, bool wide, int lane) {
    constexpr int kPer = 16 / static_cast<int>(sizeof(T)), kLanes = 32 / kPer;  // elements a piece, pieces a row
    if (wide && cols >= 32) {
        const int piece = lane % kLanes;
#pragma unroll
        for (int r = lane / kLanes; r < 32; r += 32 / kLanes) {
            if (r >= rows) break;
            alignas(16) T o[kPer];
#pragma unroll
            for (int i = 0; i < kPer; i += 4) {
                const float4 v = *reinterpret_cast<const float4 *>(box + r * kPitch + piece * kPer + i);
                from_float(v.x, o[i]);
                from_float(v.y, o[i + 1]);
                from_float(v.z, o[i + 2]);
                from_float(v.w, o[i + 3]);
            }
            *reinterpret_cast<uint4 *>(c + r * ldc + piece * kPer) = *reinterpret_cast<const uint4 *>(o);
        }
    } else if (lane < cols) {
        for (int r = 0; r < rows && r < 32; ++r) from_float(box[r * kPitch + lane], c[r * ldc + lane]);
    }
}

// A warp's 32 TMEM lanes, `cols` columns of them, to C.  ACROSS: the lanes lie
// along C's rows (n) and the columns are rows of C; else the lanes are rows of C.
// `at`: the element of lane 0 and column 0; `lanes` of the lanes are inside C.
// zero: there was nothing to sum.
template <bool ACROSS>
__device__ __forceinline__ void store_tile(const GroupedParams &p, int64_t at, uint32_t taddr, float *box, int lanes, int cols,
                                           bool zero, int lane) {
    const int es = p.c_dtype == ST_F32 ? 4 : 2;
    const int64_t next = (ACROSS ? 32 * p.ldc : 32) * es;  // bytes from 32 columns to the next
    uint8_t *base = static_cast<uint8_t *>(p.c) + at * es;
    const bool wide = reinterpret_cast<uintptr_t>(base) % 16 == 0 && p.ldc * es % 16 == 0;
#pragma unroll 1
    for (int c = 0; c < cols; c += 32, base += next) {
        uint32_t v[32];
        if (!zero) {
            tmem_load_32(taddr + static_cast<uint32_t>(c), v);
            tmem_load_wait();
        } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = 0u;
        }
        __syncwarp();  // the last 32 columns have left the box
        if constexpr (ACROSS) {
#pragma unroll
            for (int i = 0; i < 32; ++i) box[i * kPitch + lane] = __uint_as_float(v[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
                *reinterpret_cast<uint4 *>(box + lane * kPitch + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        __syncwarp();
        const int rows = ACROSS ? cols - c : lanes, width = ACROSS ? lanes : cols - c;
        if (p.c_dtype == ST_F32) store_box(reinterpret_cast<float *>(base), p.ldc, box, rows, width, wide, lane);
        else if (p.c_dtype == ST_F16) store_box(reinterpret_cast<__half *>(base), p.ldc, box, rows, width, wide, lane);
        else store_box(reinterpret_cast<__nv_bfloat16 *>(base), p.ldc, box, rows, width, wide, lane);
    }
}

// Rows [first, p.rows) of C, which belong to no group, become 0.
template <int THREADS>
__device__ __forceinline__ void zero_rows(const GroupedParams &p, int first, int thread) {
    const int64_t total = static_cast<int64_t>(p.rows - first) * p.n;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * THREADS + thread; i < total; i += static_cast<int64_t>(gridDim.x) * THREADS) {
        const int64_t at = (first + i / p.n) * p.ldc + i % p.n;
        if (p.c_dtype == ST_F32) static_cast<float *>(p.c)[at] = 0.0f;
        else static_cast<uint16_t *>(p.c)[at] = 0;
    }
}

// ---------------------------------------------------------------- one CTA, 128 x BN tiles
template <int BN>
struct GroupedCfg {
    static constexpr int kRows = 128;
    static constexpr int kOutWarps = 4;
    static constexpr int kThreads = 32 * (2 + kOutWarps);
    static constexpr int kRowBytes = kRows * kBK * 2;
    static constexpr int kColBytes = BN * kBK * 2;
    static constexpr int kStageBytes = kRowBytes + kColBytes;
    static constexpr int kStages = BN == 128 ? 6 : 9;
    static constexpr int kTmemCols = 2 * BN;
    static constexpr int kBoxBytes = 32 * kPitch * 4;
    static constexpr int kSmemBytes =
        kStages * kStageBytes + kOutWarps * kBoxBytes + static_cast<int>(sizeof(GroupTable)) + kBarBytes + 1024;
    static_assert(kSmemBytes <= 232448, "over the per-block shared memory limit");
};

template <int BN, bool WEIGHTS, bool R_MN>
__global__ void __launch_bounds__(GroupedCfg<BN>::kThreads, 1)
    gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ CUtensorMap tmap_c,
                        const GroupedParams p) {
    using Cfg = GroupedCfg<BN>;
    static_assert(!WEIGHTS || R_MN, "both operands of the second form lie along their columns");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *boxes = smem + Cfg::kStages * Cfg::kStageBytes;
    GroupTable &table = *reinterpret_cast<GroupTable *>(boxes + Cfg::kOutWarps * Cfg::kBoxBytes);
    uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(&table) + sizeof(GroupTable));
    constexpr int kBars = 2 * Cfg::kStages + 5;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
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
            mbar_init(tempty_bar(a), Cfg::kOutWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0 && p.reads) {
        tma_prefetch_map(&tmap_r);
        tma_prefetch_map(&tmap_c);
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
    const uint32_t tmem_base = *tmem_slot;

    TileWalk<WEIGHTS, Cfg::kRows, BN> walk(static_cast<int>(blockIdx.x), static_cast<int>(gridDim.x));
    Tile tile;
    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_last();
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            while (ok && walk.next(table, p, tile)) {
                const int boxes_c = (tile.cols + 31) / 32;
                for (int b = 0; b < tile.blocks; ++b, ++issued) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = full_bar(s);
                    const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                    if constexpr (WEIGHTS) {
                        mbar_arrive_expect_tx(fb, Cfg::kStageBytes);
                        const int left = tile.rows - b * kBK, y = left < kBK ? left - kBK : 0, z = tile.first + b * kBK;
#pragma unroll
                        for (int i = 0; i < Cfg::kRows / 64; ++i)
                            tma_load_3d(sr + i * 64 * 128, &tmap_r, fb, tile.r0 + 64 * i, y, z, pol);
#pragma unroll
                        for (int i = 0; i < BN / 64; ++i) tma_load_3d(sc + i * 64 * 128, &tmap_c, fb, tile.c0 + 64 * i, y, z, pol);
                    } else {
                        mbar_arrive_expect_tx(fb, static_cast<uint32_t>(Cfg::kRowBytes + boxes_c * 32 * 128));
                        const int g = p.b_groups ? tile.group : 0;
                        if constexpr (R_MN) {
#pragma unroll
                            for (int i = 0; i < Cfg::kRows / 64; ++i)
                                tma_load_3d(sr + i * 64 * 128, &tmap_r, fb, tile.r0 + 64 * i, b * kBK, g, pol);
                        } else {
                            tma_load_3d(sr, &tmap_r, fb, b * kBK, tile.r0, g, pol);
                        }
                        for (int i = 0; i < boxes_c; ++i) tma_load_2d(sc + i * 32 * 128, &tmap_c, fb, b * kBK, tile.c0 + 32 * i, pol);
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
            if (tile.blocks == 0) continue;
            const uint32_t idesc = p.idesc | static_cast<uint32_t>(WEIGHTS ? BN / 8 : (tile.cols + 15) / 16 * 2) << 17;
            if (!__all_sync(0xffffffffu, mbar_wait(tempty_bar(a), aph ^ 1u, abort_flag, p.timeout_ns))) {
                ok = false;
                break;
            }
            for (int b = 0; b < tile.blocks; ++b) {
                if (!__all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns))) {
                    ok = false;
                    break;
                }
                tc_fence_after_sync();
                if (elect_one()) {
                    const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                    const uint64_t dr = smem_desc_sw128(sr, R_MN ? 64 * 128 : 16, 1024);
                    const uint64_t dc = smem_desc_sw128(sc, WEIGHTS ? 64 * 128 : 16, 1024);
#pragma unroll
                    for (int j = 0; j < kBK / kMmaK; ++j)
                        tc_mma<false>(tmem_base + static_cast<uint32_t>(a * BN), dr + j * ((R_MN ? kMmaK * 128 : 32) >> 4),
                                      dc + j * ((WEIGHTS ? kMmaK * 128 : 32) >> 4), idesc, (b | j) != 0 ? 1u : 0u);
                    tc_commit(empty_bar(s));
                    if (b + 1 == tile.blocks) tc_commit(tfull_bar(a));
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
    } else {
        // ------------------------------------------------ C
        const int g = warp & 3;
        float *box = reinterpret_cast<float *>(boxes + g * Cfg::kBoxBytes);
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
            const int lanes = (WEIGHTS ? p.k : p.n) - tile.r0 - 32 * g;
            const int64_t at = WEIGHTS ? tile.group * p.c_g + (tile.r0 + 32 * g) * p.ldc + tile.c0
                                       : tile.c0 * p.ldc + tile.r0 + 32 * g;
            if (lanes > 0)
                store_tile<!WEIGHTS>(p, at, tmem_base + (static_cast<uint32_t>(g * 32) << 16) + static_cast<uint32_t>(a * BN), box,
                                     lanes < 32 ? lanes : 32, tile.cols, zero, lane);
            if (!zero) {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(tempty_bar(a));
                if (++a == 2) {
                    a = 0;
                    aph ^= 1u;
                }
            }
        }
        if (!WEIGHTS && p.zero_rest)
            zero_rows<32 * Cfg::kOutWarps>(p, p.groups > 0 ? table.row_end[p.groups - 1] : 0, (warp - 2) * 32 + lane);
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
// Groups of many rows.  A pair of CTAs (cta_group::2) computes 256 x 256 of C:
// each holds 128 rows of A and 128 columns of B, half of the loads per SM and
// MMA that 128 x 128 tiles of one CTA take.
//
// full[s] lives in the even CTA and counts both CTAs' loads; the even CTA's
// MMA warp commits empty[s] and tfull[a] to both CTAs; tempty[a] lives in the
// even CTA and counts the pair's warps that read accumulators.
struct GroupedPairCfg {
    static constexpr int kRows = 256, kCols = 256;
    static constexpr int kOutWarps = 4;
    static constexpr int kThreads = 32 * (2 + kOutWarps);
    static constexpr int kRowBytes = 128 * kBK * 2;
    static constexpr int kColBytes = 128 * kBK * 2;
    static constexpr int kStageBytes = kRowBytes + kColBytes;
    static constexpr int kStages = 6;
    static constexpr int kTmemCols = 2 * kCols;
    static constexpr int kBoxBytes = 32 * kPitch * 4;
    static constexpr int kSmemBytes =
        kStages * kStageBytes + kOutWarps * kBoxBytes + static_cast<int>(sizeof(GroupTable)) + kBarBytes + 1024;
    static_assert(kSmemBytes <= 232448, "over the per-block shared memory limit");
};

template <bool WEIGHTS, bool R_MN>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GroupedPairCfg::kThreads, 1)
    gemm_grouped_pair_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ CUtensorMap tmap_c,
                             const GroupedParams p) {
    using Cfg = GroupedPairCfg;
    static_assert(!WEIGHTS || R_MN, "both operands of the second form lie along their columns");
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t *boxes = smem + Cfg::kStages * Cfg::kStageBytes;
    GroupTable &table = *reinterpret_cast<GroupTable *>(boxes + Cfg::kOutWarps * Cfg::kBoxBytes);
    uint64_t *bars = reinterpret_cast<uint64_t *>(reinterpret_cast<uint8_t *>(&table) + sizeof(GroupTable));
    constexpr int kBars = 2 * Cfg::kStages + 5;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
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
            mbar_init(tempty_bar(a), 2 * Cfg::kOutWarps);
        }
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0 && p.reads) {
        tma_prefetch_map(&tmap_r);
        tma_prefetch_map(&tmap_c);
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
    const uint32_t tmem_base = *tmem_slot;

    TileWalk<WEIGHTS, Cfg::kRows, Cfg::kCols> walk(static_cast<int>(blockIdx.x >> 1), static_cast<int>(gridDim.x >> 1));
    Tile tile;
    if (warp == 0) {
        // ------------------------------------------------ TMA producer (both CTAs)
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_last();
            const uint32_t even_full0 = map_to_rank(full_bar(0), 0);
            const int half = static_cast<int>(rank) * 128;
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            while (ok && walk.next(table, p, tile)) {
                // each CTA brings half of the tile's columns (rows of A), in boxes of 32
                const int half_c = (tile.cols + 15) / 16 * 8, boxes_c = (half_c + 31) / 32;
                for (int b = 0; b < tile.blocks; ++b, ++issued) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    const uint32_t fb = even_full0 + 8u * s;
                    const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                    if constexpr (WEIGHTS) {
                        if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * Cfg::kStageBytes);
                        const int left = tile.rows - b * kBK, y = left < kBK ? left - kBK : 0, z = tile.first + b * kBK;
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            tma_load_3d_pair(sr + i * 64 * 128, &tmap_r, fb, tile.r0 + half + 64 * i, y, z, pol);
                            tma_load_3d_pair(sc + i * 64 * 128, &tmap_c, fb, tile.c0 + half + 64 * i, y, z, pol);
                        }
                    } else {
                        if (rank == 0)
                            mbar_arrive_expect_tx(full_bar(s), static_cast<uint32_t>(2 * (Cfg::kRowBytes + boxes_c * 32 * 128)));
                        const int g = p.b_groups ? tile.group : 0;
                        if constexpr (R_MN) {
#pragma unroll
                            for (int i = 0; i < 2; ++i)
                                tma_load_3d_pair(sr + i * 64 * 128, &tmap_r, fb, tile.r0 + half + 64 * i, b * kBK, g, pol);
                        } else {
                            tma_load_3d_pair(sr, &tmap_r, fb, b * kBK, tile.r0 + half, g, pol);
                        }
                        const int c0 = tile.c0 + static_cast<int>(rank) * half_c;
                        for (int i = 0; i < boxes_c; ++i)
                            tma_load_2d_pair(sc + i * 32 * 128, &tmap_c, fb, b * kBK, c0 + 32 * i, pol);
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
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer (even CTA)
        if (rank == 0) {
            int s = 0, a = 0;
            uint32_t ph = 0, aph = 0;
            bool ok = true;
            while (ok && walk.next(table, p, tile)) {
                if (tile.blocks == 0) continue;
                const uint32_t idesc = p.idesc | static_cast<uint32_t>(WEIGHTS ? Cfg::kCols / 8 : (tile.cols + 15) / 16 * 2) << 17;
                if (!__all_sync(0xffffffffu, mbar_wait(tempty_bar(a), aph ^ 1u, abort_flag, p.timeout_ns))) {
                    ok = false;
                    break;
                }
                for (int b = 0; b < tile.blocks; ++b) {
                    if (!__all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    if (elect_one()) {
                        const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                        const uint64_t dr = smem_desc_sw128(sr, R_MN ? 64 * 128 : 16, 1024);
                        const uint64_t dc = smem_desc_sw128(sc, WEIGHTS ? 64 * 128 : 16, 1024);
#pragma unroll
                        for (int j = 0; j < kBK / kMmaK; ++j)
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
        }
    } else {
        // ------------------------------------------------ C (both CTAs)
        const int g = warp & 3, row = static_cast<int>(rank) * 128 + 32 * g;
        const uint32_t even_tempty0 = map_to_rank(tempty_bar(0), 0);
        float *box = reinterpret_cast<float *>(boxes + g * Cfg::kBoxBytes);
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
            const int lanes = (WEIGHTS ? p.k : p.n) - tile.r0 - row;
            const int64_t at = WEIGHTS ? tile.group * p.c_g + (tile.r0 + row) * p.ldc + tile.c0 : tile.c0 * p.ldc + tile.r0 + row;
            if (lanes > 0)
                store_tile<!WEIGHTS>(p, at, tmem_base + (static_cast<uint32_t>(g * 32) << 16) + static_cast<uint32_t>(a * Cfg::kCols),
                                     box, lanes < 32 ? lanes : 32, tile.cols, zero, lane);
            if (!zero) {
                tc_fence_before_sync();
                __syncwarp();
                if (lane == 0) {
                    if (rank == 0) mbar_arrive(tempty_bar(a));
                    else mbar_arrive_cluster(even_tempty0 + 8u * a);
                }
                if (++a == 2) {
                    a = 0;
                    aph ^= 1u;
                }
            }
        }
        if (!WEIGHTS && p.zero_rest)
            zero_rows<32 * Cfg::kOutWarps>(p, p.groups > 0 ? table.row_end[p.groups - 1] : 0, (warp - 2) * 32 + lane);
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

// Dense copy of strided 16-bit matrices, one for each group: rows of `ld`
// elements (a multiple of 8), padding columns zeroed.
__global__ void __launch_bounds__(256) repack_groups_kernel(const uint16_t *__restrict__ src, int64_t sg, int64_t s0, int64_t s1,
                                                            int64_t groups, int64_t rows, int64_t cols, uint16_t *__restrict__ dst,
                                                            int64_t ld) {
    pdl_wait();
    const int64_t per_group = rows * ld, total = groups * per_group;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * 256) {
        const int64_t g = i / per_group, j = i - g * per_group, r = j / ld, c = j - r * ld;
        dst[i] = c < cols ? src[g * sg + r * s0 + c * s1] : static_cast<uint16_t>(0);
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

int copy_in(Matrices &m, uint8_t *&ws, int sm_count, cudaStream_t stream) {
    if (m.copy) {
        const int64_t ld = (m.inner + 7) / 8 * 8, total = m.groups * m.outer * ld;
        const int64_t grid = cdiv(total, 256 * 8) < sm_count * 8 ? cdiv(total, 256 * 8) : sm_count * 8;
        ST_CUDA_TRY(launch_kernel(repack_groups_kernel, static_cast<unsigned>(grid), 256, 0, stream,
                                  static_cast<const uint16_t *>(m.data), m.sg, m.so, m.si, m.groups, m.outer, m.inner,
                                  reinterpret_cast<uint16_t *>(ws), ld));
        ST_TRY(checked("repack_groups_kernel"));
        m.data = ws;
        ws += m.copied();
        m.so = ld;
        m.sg = m.outer * ld;
    }
    m.si = 1;
    // strides that are never used still have to be valid ones
    if (m.outer == 1) m.so = (m.inner + 7) / 8 * 8;
    if (m.groups == 1) m.sg = (m.outer * m.so + 7) / 8 * 8;
    return ST_OK;
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

template <int BN, bool WEIGHTS, bool R_MN>
int launch_instance(const CUtensorMap &mr, const CUtensorMap &mc, const GroupedParams &p, int64_t most_tiles, int sm_count,
                    cudaStream_t stream) {
    using Cfg = GroupedCfg<BN>;
    auto kern = gemm_grouped_kernel<BN, WEIGHTS, R_MN>;
    static uint64_t attr_set = 0;  // one bit per device ordinal
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg::kSmemBytes));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    const int64_t ctas = most_tiles < 1 ? 1 : most_tiles < sm_count ? most_tiles : sm_count;
    ST_CUDA_TRY(launch_kernel(kern, static_cast<unsigned>(ctas), Cfg::kThreads, Cfg::kSmemBytes, stream, mr, mc, p));
    return checked("gemm_grouped_kernel");
}

template <bool WEIGHTS, bool R_MN>
int launch_pair_instance(const CUtensorMap &mr, const CUtensorMap &mc, const GroupedParams &p, int64_t most_tiles, int sm_count,
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
    // rows of the group, on average: the columns of a tile
    const int64_t per_group = cdiv(g.rows, g.groups > 0 ? g.groups : 1), extent_r = g.weights ? g.k : g.n;
    const bool pair = extent_r > 128 && (g.weights ? g.n > 128 : per_group > 64);
    const int rows = pair ? GroupedPairCfg::kRows : 128;
    const int cols = pair ? GroupedPairCfg::kCols : g.weights || per_group > 32 ? 128 : 32;
    p.tiles_r = static_cast<int>(cdiv(extent_r, rows));
    p.tiles_c = static_cast<int>(cdiv(g.n, cols));
    const int64_t most = g.weights ? g.groups * p.tiles_r * p.tiles_c
                                   : (cdiv(g.rows, cols) + (g.groups < g.rows ? g.groups : g.rows)) * p.tiles_r;
    if (most > INT32_MAX / 2) return fail(ST_ERR_UNSUPPORTED, "matmul_grouped: too many output tiles");
    CUtensorMap mr{}, mc{};
    Operands o{};
    o.b_mn = g.weights;
    // with nothing to sum over (k = 0, no groups, or no rows) no operand is read
    if (g.rows > 0 && g.k > 0 && g.groups > 0) {
        o = operands_of(g);
        uint8_t *ws = static_cast<uint8_t *>(workspace);
        ST_TRY(copy_in(o.a, ws, sm_count, stream));
        ST_TRY(copy_in(o.b, ws, sm_count, stream));
        if (g.weights) {
            // (column, position in a step of 64 rows, the step's first row): positions reach behind the last
            // row in the map's extents, but no step's box does
            ST_TRY(make_map_16(&mr, g.dtype, "A", 3, o.a.data, g.k, kBK, g.rows, o.a.so, o.a.so, 64, kBK));
            ST_TRY(make_map_16(&mc, g.dtype, "C", 3, o.b.data, g.n, kBK, g.rows, o.b.so, o.b.so, 64, kBK));
        } else {
            ST_TRY(make_map_16(&mc, g.dtype, "A", 2, o.a.data, g.k, g.rows, 1, o.a.so, 0, kBK, 32));
            if (o.b_mn) ST_TRY(make_map_16(&mr, g.dtype, "B", 3, o.b.data, g.n, g.k, o.b.groups, o.b.so, o.b.sg, 64, kBK));
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
    if (g.weights) return launch_instance<128, true, true>(mr, mc, p, most, sm_count, stream);
    if (cols == 32)
        return o.b_mn ? launch_instance<32, false, true>(mr, mc, p, most, sm_count, stream)
                      : launch_instance<32, false, false>(mr, mc, p, most, sm_count, stream);
    return o.b_mn ? launch_instance<128, false, true>(mr, mc, p, most, sm_count, stream)
                  : launch_instance<128, false, false>(mr, mc, p, most, sm_count, stream);
}

}  // namespace st
