// gemm_fp4.cu -- matrix product of 4-bit operands (e2m1) with a scale for
// each 16 (e4m3) or 32 (e8m0) elements along the contraction.
//
//   C[m, n] = ta tb sum_k (sa[m, k / block] A[m, k]) (sb[n, k / block] B[k, n])  (+ bias[n])
//
// The tensor core multiplies the scales in (tcgen05.mma with block_scale, 64
// elements an instruction): they travel from shared memory to TMEM by
// tcgen05.cp ahead of the MMAs that read them, in the order in which the
// quantiser writes them, so that a stage's scales are one contiguous copy.
// Sums are fp32; ta, tb and the bias are applied in fp32 on the way out.
//
//   warp 0      TMA producer: 256 elements (128 bytes) of K of each operand a stage, and their scales
//   warp 1      MMA issuer (owns the TMEM allocation)
//   warps 2..   C: TMEM -> registers, scale, bias, store
//
// CTA pairs on 256 x 256 tiles, unless there are few rows of A or few tiles of
// a long K: then 128 x 16, 32 or 64 tiles of one CTA, two of them on an SM,
// and a cluster of up to 8 that splits the K of a tile.  8192^3 in 197 us over 20
// calls (5580 TFLOP/s) and 229 to 243 over seconds, under the power cap; 1024^3 in
// 5.6 in a replayed graph, 1 x 8192 x 8192 in 8.4 to 9.7 (5.8 at the copy rate).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <utility>

#include "common.h"
#include "fp8.cuh"
#include "sm100.cuh"
#include "tensor_map.h"

namespace st {
namespace {

constexpr int kTileRows = 128;
constexpr int kBlockK = 128;     // bytes: 256 elements, one 128-byte swizzle span
constexpr int kChunks = 4;       // MMAs of 64 elements in it
constexpr int kAtomBytes = 512;  // scales of 128 rows and four blocks
constexpr int kBarBytes = 512;

struct Fp4Params {
    int rows, cols;     // row operand x column operand
    int k_blocks;       // of 256 elements
    int k_chunks;       // of 64 elements
    int quads;          // groups of four blocks: atoms of a row of tiles
    int tiles_r, tiles_c, split;
    const uint8_t *rs, *cs;    // scales of the row and the column operand
    const float *ta, *tb;      // tensor scales, or null
    void *c;
    int64_t c_r, c_c;  // strides of C along the row and the column operand; one of them is 1
    int c_dtype;
    const void *bias;
    int bias_dtype;
    int bias_on_rows;  // B is the row operand: C's rows, contiguous, run along the tile's columns
    uint32_t idesc[2];  // blocks of 32: the MMA of the lower and the upper two scales of a word
    int *err;
    unsigned long long timeout_ns;
};

// The tensor scales' product, by which sums are multiplied.  Where it leaves
// fp32's normal range, a result need not: then one scale after the other,
// first the one that leads away from that end of the range.
struct Alpha {
    float first, second;
};
__device__ __forceinline__ Alpha alpha_of(const float *ta, const float *tb) {
    const float a = ta != nullptr ? *ta : 1.0f, b = tb != nullptr ? *tb : 1.0f, both = fabsf(a * b);
    if (both >= 0x1p-126f && both < INFINITY) return Alpha{1.0f, a * b};
    const bool a_first = (fabsf(a) > fabsf(b)) == (both < 1.0f);
    return a_first ? Alpha{a, b} : Alpha{b, a};
}

// Load 16 consecutive f32 columns of this thread's TMEM lane and wait for them.
__device__ __forceinline__ void tmem_read_16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}

// ---------------------------------------------------------------- one CTA, 128 x BN tiles
template <int BN>
struct Fp4Cfg {
    static constexpr int kOutWarps = 4;
    static constexpr int kThreads = 32 * (2 + kOutWarps);
    static constexpr int kRowBytes = kTileRows * kBlockK;
    static constexpr int kColBytes = BN * kBlockK;
    static constexpr int kScaleBytes = kChunks * kAtomBytes;  // of each operand (blocks of 32 use half)
    static constexpr int kStageBytes = kRowBytes + kColBytes + 2 * kScaleBytes;
    static constexpr int kStages = BN == 64 ? 3 : BN == 32 ? 4 : 5;
    // A stage's scales have TMEM columns of their own: they are overwritten
    // only after the MMAs that read them have freed the stage.
    static constexpr int kStageCols = 2 * 4 * kChunks;
    static constexpr int kScaleCol = BN;
    static constexpr int kTmemCols = 256;
    static_assert(kScaleCol + kStages * kStageCols <= kTmemCols, "the accumulator and the scales fit");
    static constexpr int kSmemBytes = kStages * kStageBytes + kBarBytes + 1024;
    static_assert(kSmemBytes <= 115712, "shared memory of two CTAs per SM");
    static_assert(kStages * kStageBytes >= kTileRows * (BN + 4 * 8) * 4, "the ring holds eight parts' sums of its columns");
};

// Thread `first` of THREADS: its share of 128 rows x `own` columns (a power
// of two, 4 at least), added over the parts of sums [part][row][own + 4],
// times alpha.  By rows, the same 4 columns of every (4 THREADS / own)th row;
// else every (THREADS / 128)th 4 columns of one row.
template <typename T, int THREADS>
__device__ __forceinline__ void store_parts(const Fp4Params &p, const float4 *sums, const Alpha &alpha, int first, int own,
                                            int own_shift, int parts, int r0, int col0) {
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
        T o[4];
        from_float(__fmaf_rn(v.x * alpha.first, alpha.second, add[0]), o[0]);
        from_float(__fmaf_rn(v.y * alpha.first, alpha.second, add[1]), o[1]);
        from_float(__fmaf_rn(v.z * alpha.first, alpha.second, add[2]), o[2]);
        from_float(__fmaf_rn(v.w * alpha.first, alpha.second, add[3]), o[3]);
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

template <int BN, bool WIDE>
__global__ void __launch_bounds__(Fp4Cfg<BN>::kThreads, 2)
    gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ CUtensorMap tmap_c,
                    const Fp4Params p) {
    using Cfg = Fp4Cfg<BN>;
    constexpr int kAtoms = WIDE ? 2 : 4;  // of a stage and an operand
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Cfg::kStages * Cfg::kStageBytes);
    constexpr int kBars = 2 * Cfg::kStages + 1;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };                   // loads landed
    auto empty_bar = [&](int s) { return bar0 + 8u * (Cfg::kStages + s); };  // MMAs done
    const uint32_t done_bar = bar0 + 8u * (kBars - 1);                       // all of the tile's MMAs done

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
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
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    pdl_begin();  // nothing above touches global memory

    const int split = p.split;
    const int part = split > 1 ? static_cast<int>(cluster_rank()) : 0;
    const int tile = static_cast<int>(blockIdx.x) / split;
    // neighbouring CTAs walk the row tiles of one column tile
    const int tr = tile % p.tiles_r, tc = tile / p.tiles_r;
    const int r0 = tr * kTileRows, c0 = tc * BN;
    // blocks part, part + split, ...: a cluster's loads of a row lie next to each other
    const int blocks = (p.k_blocks - part + split - 1) / split;

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0) {
            // rows that one column tile reads pass through L2 once
            const uint64_t pol = l2_policy_evict_last(), row_pol = p.tiles_c > 1 ? pol : l2_policy_evict_first();
            const uint8_t *rs = p.rs + static_cast<int64_t>(tr) * p.quads * kAtomBytes;
            const uint8_t *cs = p.cs + static_cast<int64_t>(c0 / 128) * p.quads * kAtomBytes;
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int b = part; b < p.k_blocks; b += split, ++issued) {
                if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                    ok = false;
                    break;
                }
                const int left = p.quads - b * kAtoms;
                const uint32_t scale_bytes = static_cast<uint32_t>(left < kAtoms ? left : kAtoms) * kAtomBytes;
                mbar_arrive_expect_tx(full_bar(s), Cfg::kRowBytes + Cfg::kColBytes + 2 * scale_bytes);
                const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes);
                const uint32_t sc = sr + Cfg::kRowBytes, ss = sc + Cfg::kColBytes;
                tma_load_2d(sr, &tmap_r, full_bar(s), b * kBlockK, r0, row_pol);
                tma_load_2d(sc, &tmap_c, full_bar(s), b * kBlockK, c0, pol);
                bulk_load(ss, rs + static_cast<int64_t>(b) * kAtoms * kAtomBytes, scale_bytes, full_bar(s));
                bulk_load(ss + Cfg::kScaleBytes, cs + static_cast<int64_t>(b) * kAtoms * kAtomBytes, scale_bytes, full_bar(s));
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
        // ------------------------------------------------ MMA issuer (see the pair's)
        const uint32_t ring = smem_addr(smem), scales = ring + Cfg::kRowBytes + Cfg::kColBytes;
        const uint64_t dr0 = smem_desc_sw128(ring, 16, 1024), dc0 = smem_desc_sw128(ring + Cfg::kRowBytes, 16, 1024);
        const uint64_t drs0 = smem_desc_scales(scales), dcs0 = smem_desc_scales(scales + Cfg::kScaleBytes);
        // a tile of 64 columns may begin in the middle of 128 columns' scales: two TMEM columns of 32 further
        const uint32_t middle = BN == 64 && (c0 & 64) ? 2u : 0u;
        int s = 0;
        uint32_t ph = 0;
        bool ok = true;
        for (int i = 0; i < blocks; ++i) {
            if (!__all_sync(0xffffffffu, mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns))) {
                ok = false;
                break;
            }
            tc_fence_after_sync();
            if (elect_one()) {
                const int left = p.k_chunks - (part + i * split) * kChunks;
                const uint64_t step = static_cast<uint64_t>(s) * (Cfg::kStageBytes >> 4);
                const uint32_t tr_s = tmem_base + static_cast<uint32_t>(Cfg::kScaleCol + s * Cfg::kStageCols);
                const uint32_t tc_s = tr_s + 4 * kChunks;
#pragma unroll
                for (uint32_t a = 0; a < kAtoms; ++a) {  // the last block's may be stale: no MMA reads those
                    tmem_copy_scales(tr_s + 4 * a, drs0 + step + a * (kAtomBytes >> 4));
                    tmem_copy_scales(tc_s + 4 * a, dcs0 + step + a * (kAtomBytes >> 4));
                }
#pragma unroll
                for (int j = 0; j < kChunks; ++j) {
                    const uint32_t atom = static_cast<uint32_t>(WIDE ? j / 2 : j);
                    if (j == 0 || j < left)
                        tc_mma_fp4<WIDE ? 2 : 4>(tmem_base, dr0 + step + j * 2u, dc0 + step + j * 2u, p.idesc[WIDE ? j % 2 : 0],
                                                 tr_s + 4 * atom, tc_s + middle + 4 * atom, i + j != 0 ? 1u : 0u);
                }
                tc_commit(empty_bar(s));
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
        if (elect_one()) tc_commit(done_bar);
        __syncwarp();
        drain_ring(1, 1, [&](int) { return done_bar; }, p.timeout_ns);  // the MMAs read shared memory and write TMEM
    }

    // ------------------------------------------------ C
    const int g = warp & 3, row_in_tile = g * 32 + lane;
    const bool out = warp >= 2;
    if (out) {
        if (!__all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort_flag, p.timeout_ns))) {
            *abort_flag = 1;
            if (lane == 0) atomicExch(p.err, kDevAbortGemmEpilogue);
        }
        tc_fence_after_sync();
    }
    const Alpha alpha = alpha_of(p.ta, p.tb);
    const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(g * 32) << 16);
    // A part owns `own` columns of the tile (with many parts, the last ones
    // none): every CTA sends its sums to their owners' rings, once all of the
    // cluster's MMAs have read them, as [part][row][own + 4 columns]; the
    // owner adds its columns over the parts in order, a warp's lanes along C's
    // contiguous dimension.
    const int own = BN / split < 4 ? 4 : BN / split, own_shift = 31 - __clz(own);  // split is a power of two
    const int stride = own + 4;  // floats; rows on different banks
    __syncwarp();
    if (split > 1) cluster_sync();
    if (out) {
        const uint32_t mine = smem_addr(smem) + 4u * static_cast<uint32_t>((part * kTileRows + row_in_tile) * stride);
#pragma unroll
        for (int c = 0; c < BN; c += 16) {
            uint32_t v[16];
            tmem_read_16(t_lane + static_cast<uint32_t>(c), v);
#pragma unroll
            for (int j = 0; j < 16; j += 4) {
                const int col = c + j;
                const uint32_t to = (split == 1 ? mine : map_to_rank(mine, static_cast<uint32_t>(col >> own_shift))) +
                                    4u * static_cast<uint32_t>(col & (own - 1));
                st_cluster_v4(to, __uint_as_float(v[j]), __uint_as_float(v[j + 1]), __uint_as_float(v[j + 2]),
                              __uint_as_float(v[j + 3]));
            }
        }
    }
    __syncwarp();
    if (split > 1) cluster_sync();
    else __syncthreads();
    if (out && part * own < BN) {
        const float4 *sums = reinterpret_cast<const float4 *>(smem);
        const int first = (warp - 2) * 32 + lane;
        const int col0 = c0 + part * own;
        constexpr int kOut = 32 * Cfg::kOutWarps;
        if (p.c_dtype == ST_F32) store_parts<float, kOut>(p, sums, alpha, first, own, own_shift, split, r0, col0);
        else if (p.c_dtype == ST_F16) store_parts<__half, kOut>(p, sums, alpha, first, own, own_shift, split, r0, col0);
        else store_parts<__nv_bfloat16, kOut>(p, sums, alpha, first, own, own_shift, split, r0, col0);
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
// The large products.  A pair of CTAs (cta_group::2) computes 256 x 256 of C,
// B's columns as its rows, so that the TMEM lanes lie along C's rows and C is
// stored from registers as it is: each CTA holds 128 rows of the row operand
// and 128 of the column operand, and the scales of its rows and of all columns.
//
// TMEM: a tile's sums take 256 columns, the scales of each stage 48 of their
// own behind them (so that they are written again only after the MMAs that read
// them have freed the stage).  There is no room for a second accumulator: eight
// warps take a tile's sums into registers at once, and the next tile's MMAs
// start when they have.
//
// What bounds the kernel is the warp that issues: a stage's 12 scale copies, 4
// MMAs and their barriers take it about as long as the 512 cycles of the MMAs.
// So it keeps together, its operands in uniform registers (the warp's index and
// the TMEM address are broadcast for that), and asks for the next stage's
// barrier before it issues this one's MMAs.
//
// full[s] lives in the even CTA and counts both CTAs' loads; the even CTA's
// MMA warp commits empty[s] and tfull to both CTAs; tfree lives in the even CTA
// and counts the pair's warps that have taken a tile's sums.
struct Fp4PairCfg {
    static constexpr int kRows = 256, kCols = 256;
    static constexpr int kOutWarps = 8;
    static constexpr int kThreads = 32 * (2 + kOutWarps);
    static constexpr int kRowBytes = 128 * kBlockK;
    static constexpr int kColBytes = 128 * kBlockK;
    static constexpr int kRowScaleBytes = kChunks * kAtomBytes;
    static constexpr int kColScaleBytes = 2 * kChunks * kAtomBytes;
    static constexpr int kStageBytes = kRowBytes + kColBytes + kRowScaleBytes + kColScaleBytes;
    static constexpr int kStages = 5;
    static constexpr int kScaleCol = kCols, kScaleCols = 12 * kChunks;
    static constexpr int kTmemCols = 512;
    static_assert(kScaleCol + kStages * kScaleCols <= kTmemCols, "the accumulator and the scales fit");
    static constexpr int kSmemBytes = kStages * kStageBytes + kBarBytes + 1024;
    static_assert(kSmemBytes <= 232448, "over the per-block shared memory limit");
};

// First row and column of tile t: 8 column tiles of a row tile after another,
// so that the tiles in flight share their operands in L2.
__device__ __forceinline__ void pair_tile(const Fp4Params &p, int t, int &r0, int &c0) {
    constexpr int kBand = 8;
    const int in_band = kBand * p.tiles_r;
    const int first = t / in_band * kBand;
    const int high = p.tiles_c - first < kBand ? p.tiles_c - first : kBand;
    c0 = (first + t % in_band % high) * Fp4PairCfg::kCols;
    r0 = t % in_band / high * Fp4PairCfg::kRows;
}

// 32 columns (rows of C) of a warp's lanes (its columns): alpha, bias, store.
template <typename T>
__device__ __forceinline__ void store_columns(T *to, int64_t ldc, const uint32_t (&v)[32], int cols, float alpha, float add) {
    if (cols >= 32) {
#pragma unroll
        for (int i = 0; i < 32; ++i, to += ldc) from_float(__fmaf_rn(__uint_as_float(v[i]), alpha, add), *to);
    } else {
#pragma unroll
        for (int i = 0; i < 32; ++i, to += ldc)
            if (i < cols) from_float(__fmaf_rn(__uint_as_float(v[i]), alpha, add), *to);
    }
}

template <bool WIDE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(Fp4PairCfg::kThreads, 1)
    gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tmap_r, const __grid_constant__ CUtensorMap tmap_c,
                         const __grid_constant__ CUtensorMap tmap_rs, const __grid_constant__ CUtensorMap tmap_cs,
                         const Fp4Params p) {
    using Cfg = Fp4PairCfg;
    constexpr int kAtoms = WIDE ? 2 : 4;  // of a stage and 128 rows
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + Cfg::kStages * Cfg::kStageBytes);
    constexpr int kBars = 2 * Cfg::kStages + 3;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + kBars);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(tmem_slot + 1);

    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
    const int lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = static_cast<int>(blockIdx.x >> 1), pairs = static_cast<int>(gridDim.x >> 1);
    const int tiles = p.tiles_r * p.tiles_c;
    const uint32_t bar0 = smem_addr(bars);
    auto full_bar = [&](int s) { return bar0 + 8u * s; };
    auto empty_bar = [&](int s) { return bar0 + 8u * (Cfg::kStages + s); };
    const uint32_t tfull_bar = bar0 + 8u * (2 * Cfg::kStages), tfree_bar = tfull_bar + 8u;
    const uint32_t drain_bar = bar0 + 8u * (kBars - 1);

    if (threadIdx.x == 0) {
        for (int s = 0; s < Cfg::kStages; ++s) {
            mbar_init(full_bar(s), 1);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(tfull_bar, 1);
        mbar_init(tfree_bar, 2 * Cfg::kOutWarps);
        mbar_init(drain_bar, 1);
        *abort_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        tma_prefetch_map(&tmap_r);
        tma_prefetch_map(&tmap_c);
        tma_prefetch_map(&tmap_rs);
        tma_prefetch_map(&tmap_cs);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_addr(tmem_slot), Cfg::kTmemCols);
        tmem_relinquish_pair();
    }
    tc_fence_before_sync();
    __syncthreads();
    cluster_sync();
    tc_fence_after_sync();
    const uint32_t tmem_base = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    pdl_begin();  // nothing above touches global memory

    if (warp == 0) {
        // ------------------------------------------------ TMA producer (both CTAs)
        if (lane == 0) {
            const uint64_t pol = l2_policy_evict_last();
            const uint32_t even_full0 = map_to_rank(full_bar(0), 0);
            constexpr uint32_t kBytes = Cfg::kRowBytes + Cfg::kColBytes + 3 * kAtoms * kAtomBytes;
            int s = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = pair; ok && t < tiles; t += pairs) {
                int r0, c0;
                pair_tile(p, t, r0, c0);
                const int half = static_cast<int>(rank) * 128;
                for (int b = 0; b < p.k_blocks; ++b, ++issued) {
                    if (!mbar_wait(empty_bar(s), ph ^ 1u, abort_flag, p.timeout_ns)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * kBytes);
                    const uint32_t sr = smem_addr(smem + s * Cfg::kStageBytes), sc = sr + Cfg::kRowBytes;
                    const uint32_t srs = sc + Cfg::kColBytes, scs = srs + Cfg::kRowScaleBytes, fb = even_full0 + 8u * s;
                    tma_load_2d_pair(sr, &tmap_r, fb, b * kBlockK, r0 + half, pol);
                    tma_load_2d_pair(sc, &tmap_c, fb, b * kBlockK, c0 + half, pol);
                    tma_load_3d_pair(srs, &tmap_rs, fb, 0, b * kAtoms, (r0 + half) / 128, pol);
                    tma_load_3d_pair(scs, &tmap_cs, fb, 0, b * kAtoms, c0 / 128, pol);
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
        // ------------------------------------------------ MMA issuer (even CTA)
        if (rank == 0) {
            const uint32_t ring = smem_addr(smem);
            const uint64_t dr0 = smem_desc_sw128(ring, 16, 1024), dc0 = smem_desc_sw128(ring + Cfg::kRowBytes, 16, 1024);
            const uint64_t drs0 = smem_desc_scales(ring + Cfg::kRowBytes + Cfg::kColBytes);
            const uint64_t dcs0 = smem_desc_scales(ring + Cfg::kRowBytes + Cfg::kColBytes + Cfg::kRowScaleBytes);
            int s = 0;
            uint32_t ph = 0, fph = 0;
            bool ok = true, there = false;  // there: this lane has seen stage s filled
            for (int t = pair; ok && t < tiles; t += pairs) {
                // the last tile's sums have been taken
                if (!__all_sync(0xffffffffu, mbar_wait(tfree_bar, fph ^ 1u, abort_flag, p.timeout_ns))) {
                    ok = false;
                    break;
                }
                fph ^= 1u;
                for (int b = 0; b < p.k_blocks; ++b) {
                    if (!__all_sync(0xffffffffu, there || mbar_wait(full_bar(s), ph, abort_flag, p.timeout_ns))) {
                        ok = false;
                        break;
                    }
                    tc_fence_after_sync();
                    const int next = s + 1 == Cfg::kStages ? 0 : s + 1;
                    const uint32_t next_ph = next == 0 ? ph ^ 1u : ph;
                    there = mbar_try_now(full_bar(next), next_ph);
                    if (elect_one()) {
                        const int left = p.k_chunks - b * kChunks;
                        const uint64_t step = static_cast<uint64_t>(s) * (Cfg::kStageBytes >> 4);
                        const uint32_t tr_s = tmem_base + static_cast<uint32_t>(Cfg::kScaleCol + s * Cfg::kScaleCols);
                        const uint32_t tc_s = tr_s + 4 * kChunks;
#pragma unroll
                        for (uint32_t i = 0; i < kAtoms; ++i) {
                            tmem_copy_scales_pair(tr_s + 4 * i, drs0 + step + i * (kAtomBytes >> 4));
                            tmem_copy_scales_pair(tc_s + 8 * i, dcs0 + step + i * (kAtomBytes >> 4));
                            tmem_copy_scales_pair(tc_s + 8 * i + 4, dcs0 + step + (kAtoms + i) * (kAtomBytes >> 4));
                        }
#pragma unroll
                        for (int j = 0; j < kChunks; ++j) {
                            const uint32_t atom = static_cast<uint32_t>(WIDE ? j / 2 : j);
                            if (j == 0 || j < left)
                                tc_mma_fp4_pair<WIDE ? 2 : 4>(tmem_base, dr0 + step + j * 2u, dc0 + step + j * 2u,
                                                              p.idesc[WIDE ? j % 2 : 0], tr_s + 4 * atom, tc_s + 8 * atom,
                                                              j != 0 || b != 0 ? 1u : 0u);
                        }
                        tc_commit_pair_multicast(empty_bar(s), 3);
                        if (b + 1 == p.k_blocks) tc_commit_pair_multicast(tfull_bar, 3);
                    }
                    __syncwarp();
                    s = next;
                    ph = next_ph;
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
        const int g = warp & 3, side = (warp - 2) >> 2;  // two warps for each quarter of the lanes
        const uint32_t even_tfree = map_to_rank(tfree_bar, 0);
        const uint32_t t_lane = tmem_base + (static_cast<uint32_t>(g * 32) << 16);
        const Alpha alpha = alpha_of(p.ta, p.tb);
        uint32_t fph = 0;
        for (int t = pair; t < tiles; t += pairs, fph ^= 1u) {
            int r0, c0;
            pair_tile(p, t, r0, c0);
            if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar, fph, abort_flag, p.timeout_ns))) {
                *abort_flag = 1;
                if (lane == 0) atomicExch(p.err, kDevAbortGemmEpilogue);
                break;
            }
            tc_fence_after_sync();
            uint32_t v[4][32];
#pragma unroll
            for (int i = 0; i < 4; ++i) tmem_load_32(t_lane + static_cast<uint32_t>(128 * side + 32 * i), v[i]);
            tmem_load_wait();
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(tfree_bar);
                else mbar_arrive_cluster(even_tfree);
            }
            if (alpha.first != 1.0f) {  // hardly ever: multiplied always, 1024^3 took 5.8 us, so 5.6
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[i][j] = __float_as_uint(__uint_as_float(v[i][j]) * alpha.first);
            }
            const int row = r0 + static_cast<int>(rank) * 128 + 32 * g + lane;  // of the row operand: a column of C
            if (row < p.rows) {
                const float add = p.bias != nullptr ? load_any(p.bias, p.bias_dtype, row) : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int col = c0 + 128 * side + 32 * i, left = p.cols - col;
                    if (left <= 0) break;
                    const int64_t to = col * p.c_c + row;
                    if (p.c_dtype == ST_F32) store_columns(static_cast<float *>(p.c) + to, p.c_c, v[i], left, alpha.second, add);
                    else if (p.c_dtype == ST_F16) store_columns(static_cast<__half *>(p.c) + to, p.c_c, v[i], left, alpha.second, add);
                    else store_columns(static_cast<__nv_bfloat16 *>(p.c) + to, p.c_c, v[i], left, alpha.second, add);
                }
            }
            __syncwarp();  // TMEM is read by whole warps
        }
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

// ---------------------------------------------------------------- host side
int make_map_4(CUtensorMap *map, const char *what, const void *base, int64_t k_bytes, int64_t rows, int64_t ld, int box_rows) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(k_bytes), static_cast<cuuint64_t>(rows)};
    const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld)};
    const cuuint32_t box[2] = {kBlockK, static_cast<cuuint32_t>(box_rows)};
    return make_tensor_map(map, what, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box);
}

template <int BN, bool WIDE>
int launch_instance(const CUtensorMap &mr, const CUtensorMap &mc, const Fp4Params &p, cudaStream_t stream) {
    using Cfg = Fp4Cfg<BN>;
    auto kern = gemm_fp4_kernel<BN, WIDE>;
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
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "gemm_fp4_kernel launch");
}

template <int BN>
int launch_tile(const CUtensorMap &mr, const CUtensorMap &mc, const Fp4Params &p, bool wide, cudaStream_t stream) {
    return wide ? launch_instance<BN, true>(mr, mc, p, stream) : launch_instance<BN, false>(mr, mc, p, stream);
}

// An operand's scales, [row / 128][block / 4] of 512 bytes, in boxes of a stage's of `tiles` times 128 rows.
int make_map_scales(CUtensorMap *map, const void *base, int64_t rows, int64_t quads, int atoms, int tiles) {
    const cuuint64_t dims[3] = {kAtomBytes / 4, static_cast<cuuint64_t>(quads), static_cast<cuuint64_t>(cdiv(rows, 128))};
    const cuuint64_t strides[2] = {kAtomBytes, static_cast<cuuint64_t>(quads) * kAtomBytes};
    const cuuint32_t box[3] = {kAtomBytes / 4, static_cast<cuuint32_t>(atoms), static_cast<cuuint32_t>(tiles)};
    return make_tensor_map(map, "scales of a 4-bit operand", CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, base, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_NONE);
}

template <bool WIDE>
int launch_pair(const CUtensorMap &mr, const CUtensorMap &mc, const CUtensorMap &mrs, const CUtensorMap &mcs, const Fp4Params &p,
                int sm_count, cudaStream_t stream) {
    auto kern = gemm_fp4_pair_kernel<WIDE>;
    static uint64_t attr_set = 0;  // one bit per device ordinal
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Fp4PairCfg::kSmemBytes));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    const int64_t tiles = static_cast<int64_t>(p.tiles_r) * p.tiles_c;
    const int64_t pairs = tiles < sm_count / 2 ? tiles : sm_count / 2;
    ST_CUDA_TRY(launch_kernel(kern, static_cast<unsigned>(2 * pairs), Fp4PairCfg::kThreads, Fp4PairCfg::kSmemBytes, stream, mr, mc, mrs,
                              mcs, p));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "gemm_fp4_pair_kernel launch");
}

// TMA reads an operand in place if its rows lie along K on 16-byte boundaries
// and do not overlap; any other is copied first.
struct Access {
    bool copy;
    int64_t ld;  // bytes between rows
};

Access access_of(const Fp4Operand &o) {
    const bool fits = reinterpret_cast<uintptr_t>(o.data) % 16 == 0 && (o.s_k == 1 || o.k == 1) &&
                      (o.rows == 1 || (o.s_row >= o.k && o.s_row % 16 == 0 && o.s_row < (int64_t(1) << 40)));
    return {!fits, fits && o.rows > 1 ? o.s_row : (o.k + 15) / 16 * 16};
}

int64_t copy_bytes(const Fp4Operand &o, const Access &a) { return a.copy ? (o.rows * a.ld + 255) / 256 * 256 : 0; }

// Kernel, tile and split of a product: the least estimated time.  The figures
// are microseconds fitted to B200 timings of 1 x 1024 x 1024 to 4096 x 4096 x
// 1024 and 1 x 4096 x 16384 (within 15 %; 1 x 8192 x 8192 estimated 8.3 on 16
// columns and four parts, measured 8.4; 1024 x 512 x 8192 10.9 on 64 columns
// and four parts, 13.6 by pairs, measured 12.4 and 13.5).
struct Fp4Plan {
    bool pair = false, swap = false;  // swap: B is the row operand
    int bn = 64, split = 1;
    double us = 1e300;
};

Fp4Plan plan_fp4(int64_t m, int64_t n, int64_t k_blocks, int sm_count) {
    Fp4Plan best;
    {
        const int64_t waves = cdiv(cdiv(n, 256) * cdiv(m, 256), sm_count / 2);
        best.pair = best.swap = true;
        best.us = 3.7 + static_cast<double>(waves) * (0.3 * static_cast<double>(k_blocks) + 0.3);
    }
    struct Shape {
        int bn;
        double ends, block, two, join[4];  // a block of K alone on an SM, and beside another CTA; extra for 1 to 8 parts
    };
    const Shape shapes[] = {{16, 3.9, 0.30, 0.42, {0, 0.8, 1.0, 1.6}},
                            {32, 4.2, 0.33, 0.45, {0, 0.8, 1.2, 2.0}},
                            {64, 4.8, 0.31, 0.36, {0, 2.0, 3.2, 5.0}}};
    for (int swap = 0; swap < 2; ++swap) {
        const int64_t rows = swap ? n : m, cols = swap ? m : n;
        for (const Shape &s : shapes) {
            if (s.bn < 64 && cols > s.bn) continue;  // a column tile's scales begin with 64 or 128 of them
            const int64_t tiles = cdiv(rows, kTileRows) * cdiv(cols, s.bn);
            for (int parts = 0; parts <= 3 && (1 << parts) <= k_blocks; ++parts) {
                const int64_t ctas = tiles << parts, rounds = cdiv(ctas, 2 * static_cast<int64_t>(sm_count));
                if (rounds > 1 && parts > 0) break;
                const double block = ctas > sm_count ? s.two : s.block;
                const double us = static_cast<double>(rounds) * (s.ends + s.join[parts] + block * static_cast<double>(cdiv(k_blocks, int64_t(1) << parts)));
                if (us < best.us) best = Fp4Plan{false, swap != 0, s.bn, 1 << parts, us};
            }
        }
    }
    return best;
}

}  // namespace

int64_t gemm_fp4_workspace_bytes(const Fp4Operand &a, const Fp4Operand &b) {
    if (a.rows == 0 || b.rows == 0 || a.k == 0) return 0;
    return copy_bytes(a, access_of(a)) + copy_bytes(b, access_of(b));
}

int launch_gemm_fp4(const GemmFp4Args &g, void *workspace, int sm_count, int *dev_err, uint64_t timeout_ns,
                    cudaStream_t stream) {
    const int64_t m = g.a.rows, n = g.b.rows, k = g.a.k;
    if (m == 0 || n == 0) return ST_OK;
    if (k == 0) return launch_fill_bias(g.c, g.ldc, g.c_dtype, g.bias, g.bias_dtype, m, n, sm_count, stream);
    Fp4Operand op[2] = {g.a, g.b};
    Access acc[2] = {access_of(g.a), access_of(g.b)};
    uint8_t *ws = static_cast<uint8_t *>(workspace);
    for (int i = 0; i < 2; ++i) {
        if (!acc[i].copy) continue;
        ST_TRY(launch_repack_8(op[i].data, op[i].s_row, op[i].s_k, op[i].rows, op[i].k, ws, acc[i].ld, sm_count, stream));
        op[i].data = ws;
        ws += copy_bytes(op[i], acc[i]);
    }
    const int64_t k_blocks = cdiv(k, kBlockK);
    const Fp4Plan plan = plan_fp4(m, n, k_blocks, sm_count);
    const bool swap = plan.swap;
    const int ri = swap ? 1 : 0, ci = swap ? 0 : 1;
    const Fp4Operand &r = op[ri], &c = op[ci];
    Fp4Params p{};
    p.rows = static_cast<int>(r.rows);
    p.cols = static_cast<int>(c.rows);
    p.k_blocks = static_cast<int>(k_blocks);
    p.k_chunks = static_cast<int>(cdiv(k, 32));
    p.quads = static_cast<int>(cdiv(cdiv(k, g.wide ? 16 : 8), 4));
    p.tiles_r = static_cast<int>(cdiv(r.rows, plan.pair ? Fp4PairCfg::kRows : kTileRows));
    p.tiles_c = static_cast<int>(cdiv(c.rows, plan.pair ? Fp4PairCfg::kCols : plan.bn));
    p.split = plan.split;
    if (static_cast<int64_t>(p.tiles_r) * p.tiles_c * p.split > INT32_MAX)
        return fail(ST_ERR_UNSUPPORTED, "matmul_fp4: too many output tiles");
    p.rs = static_cast<const uint8_t *>(r.scale);
    p.cs = static_cast<const uint8_t *>(c.scale);
    p.ta = g.a.tensor_scale;
    p.tb = g.b.tensor_scale;
    p.c = g.c;
    p.c_r = swap ? 1 : g.ldc;
    p.c_c = swap ? g.ldc : 1;
    p.c_dtype = g.c_dtype;
    p.bias = g.bias;
    p.bias_dtype = g.bias_dtype;
    p.bias_on_rows = swap;
    for (uint32_t i = 0; i < 2; ++i)
        p.idesc[i] = plan.pair ? mma_idesc_fp4(g.wide, 2 * i, Fp4PairCfg::kRows, Fp4PairCfg::kCols)
                               : mma_idesc_fp4(g.wide, 2 * i, kTileRows, static_cast<uint32_t>(plan.bn));
    p.err = dev_err;
    p.timeout_ns = timeout_ns;
    CUtensorMap mr, mc;
    ST_TRY(make_map_4(&mr, "a 4-bit operand", r.data, k, r.rows, acc[ri].ld, kTileRows));
    ST_TRY(make_map_4(&mc, "a 4-bit operand", c.data, k, c.rows, acc[ci].ld, plan.pair ? 128 : plan.bn));
    if (plan.pair) {
        CUtensorMap mrs, mcs;
        const int atoms = g.wide ? 2 : 4;
        ST_TRY(make_map_scales(&mrs, r.scale, r.rows, p.quads, atoms, 1));
        ST_TRY(make_map_scales(&mcs, c.scale, c.rows, p.quads, atoms, 2));
        return g.wide ? launch_pair<true>(mr, mc, mrs, mcs, p, sm_count, stream)
                      : launch_pair<false>(mr, mc, mrs, mcs, p, sm_count, stream);
    }
    switch (plan.bn) {
    case 16: return launch_tile<16>(mr, mc, p, g.wide, stream);
    case 32: return launch_tile<32>(mr, mc, p, g.wide, stream);
    default: return launch_tile<64>(mr, mc, p, g.wide, stream);
    }
}

}  // namespace st
