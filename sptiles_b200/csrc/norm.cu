// norm.cu -- the norms after and before a block, fused with the block's gate
// and residual scale, forward and backward.
//
//   u  = x * rsqrt(mean(x^2) + eps) * (post + offset)      (u = x without post)
//   r' = r + alpha * gate * u
//   h  = r' * rsqrt(mean(r'^2) + eps) * (pre + offset)     (as 8-bit blocks of 128 if asked)
//
// One pass: a row of x and r is read once into registers, both means are
// reduced over the row's warps, r' and h are written once.  h comes from r'
// before its rounding to the stream's type.
//
// The way back takes r' and x, not the forward call's statistics: their sums
// come with the same read.  With t = dh * (pre + offset), R = r' * inv_r:
//
//   dpre  = sum_rows dh * R
//   dr    = dr' + inv_r * (t - R * mean(t * R))
//   du    = alpha * gate * dr,  dgate = alpha * dr * u (summed over what the gate was broadcast over)
//   dx    = the same with x, post and du in the place of r', pre and dh;  dpost likewise
//
// The sums over rows are kept in registers by a fixed set of row groups, each
// taking every G-th row, written once to a workspace and added in a fixed
// order by a second launch: no atomics, the same bits on every run.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "common.h"
#include "fp8.cuh"
#include "sm100.cuh"

namespace st {
namespace {

constexpr int kChunk = 256;     // elements of a row that a warp takes at a time, 8 a lane
constexpr int kRowsPerCta = 4;  // rows (warps) of a CTA when a warp covers a row
constexpr int kMaxThreads = 512;  // 128 registers a thread
constexpr int64_t kMaxCols = 4 * kMaxThreads * 8;

// Where a lane's 8 elements of a chunk lie.  VEC: next to each other;
// otherwise 32 apart, so that a warp's scalar loads are contiguous.
template <bool VEC>
__device__ __forceinline__ int element(int base, int lane, int j) {
    return VEC ? base + lane * 8 + j : base + lane + 32 * j;
}

// 8 elements as stored.
template <typename T>
struct Raw8 {
    uint4 w[sizeof(T) / 2];
    __device__ __forceinline__ float operator[](int j) const { return to_float(reinterpret_cast<const T *>(w)[j]); }
};

template <typename T, bool VEC>
__device__ __forceinline__ Raw8<T> load_raw(const NormView &view, int64_t r, int base, int lane, int cols) {
    Raw8<T> out;
    const T *row = static_cast<const T *>(view.p) + r * view.ld;
    if (VEC && base + lane * 8 + 8 <= cols) {
        const uint4 *src = reinterpret_cast<const uint4 *>(row + base + lane * 8);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) out.w[i] = src[i];
    } else if (!VEC && base + kChunk <= cols) {
        T *e = reinterpret_cast<T *>(out.w);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] = row[base + lane + 32 * j];
    } else {
        T *e = reinterpret_cast<T *>(out.w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = element<VEC>(base, lane, j);
            if (c < cols) e[j] = row[c];
            else from_float(0.0f, e[j]);
        }
    }
    return out;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T *row, int base, int lane, int cols, float (&f)[8]) {
    if (VEC && base + lane * 8 + 8 <= cols) {
        uint4 w[sizeof(T) / 2];
        const uint4 *src = reinterpret_cast<const uint4 *>(row + base + lane * 8);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = src[i];
        const T *e = reinterpret_cast<const T *>(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = to_float(e[j]);
    } else if (!VEC && base + kChunk <= cols) {  // the whole warp is inside: no checks
        row += base + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = to_float(row[32 * j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = element<VEC>(base, lane, j);
            f[j] = c < cols ? to_float(row[c]) : 0.0f;
        }
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T *row, int base, int lane, int cols, const float (&f)[8]) {
    if (VEC && base + lane * 8 + 8 <= cols) {
        uint4 w[sizeof(T) / 2];
        T *e = reinterpret_cast<T *>(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) from_float(f[j], e[j]);
        uint4 *dst = reinterpret_cast<uint4 *>(row + base + lane * 8);
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) dst[i] = w[i];
    } else if (!VEC && base + kChunk <= cols) {
        row += base + lane;
#pragma unroll
        for (int j = 0; j < 8; ++j) from_float(f[j], row[32 * j]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = element<VEC>(base, lane, j);
            if (c < cols) from_float(f[j], row[c]);
        }
    }
}

// A weight or gate of type T or fp32.
template <typename T, bool VEC>
__device__ __forceinline__ void load8_of(const NormView &v, int64_t row, int base, int lane, int cols,
                                         float (&f)[8]) {
    if (v.dtype == ST_F32) load8<float, VEC>(static_cast<const float *>(v.p) + row * v.ld, base, lane, cols, f);
    else load8<T, VEC>(static_cast<const T *>(v.p) + row * v.ld, base, lane, cols, f);
}

template <typename T>
__device__ __forceinline__ float load1_of(const NormView &v, int64_t row) {
    if (v.dtype == ST_F32) return static_cast<const float *>(v.p)[row * v.ld];
    return to_float(static_cast<const T *>(v.p)[row * v.ld]);
}

// Sums of N values over the warps of a row.  `slot` alternates between two
// buffers, so that one barrier a call is enough.
template <int N>
__device__ __forceinline__ void row_sum(float (&v)[N], int warps, int warp, int lane, float *slots, int &slot) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (warps == 1) return;
    float *s = slots + slot * 3 * 32;
    slot ^= 1;
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) s[i * 32 + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = lane < warps ? s[i * 32 + lane] : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
}

// One row: the warps of the CTA (warps > 1), or one warp of it.
struct RowGroup {
    int warps, warp, lane;
    int64_t first, step;
    __device__ __forceinline__ RowGroup(int warps_) : warps(warps_), lane(threadIdx.x & 31) {
        const int w = threadIdx.x >> 5;
        const int per_cta = warps == 1 ? static_cast<int>(blockDim.x >> 5) : 1;
        warp = warps == 1 ? 0 : w;
        first = static_cast<int64_t>(blockIdx.x) * per_cta + (warps == 1 ? w : 0);
        step = static_cast<int64_t>(gridDim.x) * per_cta;
    }
    __device__ __forceinline__ int base(int v) const { return (v * warps + warp) * kChunk; }
};

// 8 elements of a row's normed copy, in the branch's type or as 8-bit blocks.
template <typename TX, bool VEC>
__device__ __forceinline__ void store_normed(const NormArgs &p, int64_t row, int base, int lane, int cols, const float (&h)[8]) {
    if (!p.h_fp8) {
        store8<TX, VEC>(static_cast<TX *>(p.h.p) + row * p.h.ld, base, lane, cols, h);
        return;
    }
    // a chunk is two blocks of 128: VEC, 16 lanes each; otherwise the lanes' first and last four elements
    const float limit = p.h_e5m2 ? 57344.0f : 448.0f;
    float m[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 8; j += 2) m[VEC ? 0 : j / 4] = max_abs(m[VEC ? 0 : j / 4], h[j], h[j + 1]);
    float inverse[2];
#pragma unroll
    for (int b = 0; b < (VEC ? 1 : 2); ++b) {
#pragma unroll
        for (int o = VEC ? 8 : 16; o > 0; o >>= 1) m[b] = max_abs(m[b], __shfl_xor_sync(0xffffffffu, m[b], o));
        const float scale = fp8_scale(m[b], limit);
        inverse[b] = __frcp_rn(scale);
        const int block = base / 128 + (VEC ? lane / 16 : b);
        if ((VEC ? lane % 16 : lane) == 0 && block * 128 < cols) p.h_scale[row * p.hs0 + block * p.hs1] = scale;
    }
    if constexpr (VEC) inverse[1] = inverse[0];
    uint32_t q[2];
#pragma unroll
    for (int b = 0; b < 2; ++b)
        q[b] = to_fp8x4(__fmul_rn(h[4 * b], inverse[b]), __fmul_rn(h[4 * b + 1], inverse[b]),
                        __fmul_rn(h[4 * b + 2], inverse[b]), __fmul_rn(h[4 * b + 3], inverse[b]), p.h_e5m2);
    uint8_t *to = static_cast<uint8_t *>(p.h.p) + row * p.h.ld;
    if (VEC && base + lane * 8 + 8 <= cols) {
        *reinterpret_cast<uint2 *>(to + base + lane * 8) = make_uint2(q[0], q[1]);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int c = element<VEC>(base, lane, j);
            if (c < cols) to[c] = static_cast<uint8_t>(q[j / 4] >> (8 * (j % 4)));
        }
    }
}

// Few rows, short ones, and any alignment: a CTA or a warp for each row.
// AHEAD: all of a row's reads, the weights among them, are under way before
// the first sum, for few rows (1 x 4096 in 3.6 us, latency alone); many rows
// would rather have the registers (unaligned 1025 x 2049 with a full gate in
// 14.1 us a call; inputs not in L2: 16.5, and 19.6 at 128 registers a thread).
template <typename TX, typename TR, int VPT, bool VEC, bool AHEAD>
__global__ void __launch_bounds__(VPT == 1 && !AHEAD ? 2 * kMaxThreads : kMaxThreads) residual_norm_kernel(const NormArgs p, int warps) {
    pdl_wait();
    __shared__ float slots[2 * 3 * 32];
    const RowGroup g(warps);
    const int cols = static_cast<int>(p.cols);
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    const bool has_x = p.x.p != nullptr, has_post = p.post.p != nullptr, has_pre = p.pre.p != nullptr;
    const bool wide_gate = p.gate_mode == kGateChannel || p.gate_mode == kGateFull;
    int slot = 0;
    for (int64_t row = g.first; row < p.rows; row += g.step) {
        const int64_t gate_row = p.gate_mode == kGateFull ? row : 0;
        float r[VPT][8], x[VPT][8], post[VPT][8], gate[VPT][8], pre[VPT][8];
        float token = p.alpha;
        if (p.gate_mode == kGateToken) token *= load1_of<TX>(p.gate, row);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            if (has_x) load8<TX, VEC>(static_cast<const TX *>(p.x.p) + row * p.x.ld, g.base(v), g.lane, cols, x[v]);
            load8<TR, VEC>(static_cast<const TR *>(p.r.p) + row * p.r.ld, g.base(v), g.lane, cols, r[v]);
            if (AHEAD && has_post) load8_of<TX, VEC>(p.post, 0, g.base(v), g.lane, cols, post[v]);
            if (AHEAD && wide_gate) load8_of<TX, VEC>(p.gate, gate_row, g.base(v), g.lane, cols, gate[v]);
            if (AHEAD && has_pre) load8_of<TX, VEC>(p.pre, 0, g.base(v), g.lane, cols, pre[v]);
        }
        if (has_x) {
            if (has_post) {
                float s[1] = {0.0f};
#pragma unroll
                for (int v = 0; v < VPT; ++v)
#pragma unroll
                    for (int j = 0; j < 8; ++j) s[0] += x[v][j] * x[v][j];
                row_sum(s, g.warps, g.warp, g.lane, slots, slot);
                const float inv = rsqrtf(s[0] * inv_cols + p.eps);
#pragma unroll
                for (int v = 0; v < VPT; ++v) {
                    if (!AHEAD) load8_of<TX, VEC>(p.post, 0, g.base(v), g.lane, cols, post[v]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[v][j] *= inv * (post[v][j] + p.offset);
                }
            }
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                if (wide_gate) {
                    if (!AHEAD) load8_of<TX, VEC>(p.gate, gate_row, g.base(v), g.lane, cols, gate[v]);
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[v][j] *= gate[v][j];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) r[v][j] += token * x[v][j];
            }
        }
        if (p.r_out.p != nullptr) {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
                store8<TR, VEC>(static_cast<TR *>(p.r_out.p) + row * p.r_out.ld, g.base(v), g.lane, cols, r[v]);
        }
        if (!has_pre) continue;
        float s[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int j = 0; j < 8; ++j) s[0] += r[v][j] * r[v][j];
        row_sum(s, g.warps, g.warp, g.lane, slots, slot);
        const float inv = rsqrtf(s[0] * inv_cols + p.eps);
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            if (!AHEAD) load8_of<TX, VEC>(p.pre, 0, g.base(v), g.lane, cols, pre[v]);
#pragma unroll
            for (int j = 0; j < 8; ++j) r[v][j] *= inv * (pre[v][j] + p.offset);
            store_normed<TX, VEC>(p, row, g.base(v), g.lane, cols, r[v]);
        }
    }
    pdl_trigger();
}

// ---------------------------------------------------------------- many rows on 16-byte boundaries
// Persistent CTAs, each taking every G-th row: rows of x and r arrive by bulk
// copies in a ring of shared memory, S rows ahead, so that what is in flight
// does not depend on registers or on where the row before stands between its
// two sums; the weights stay in registers over the rows, folded into one
// factor per element and norm.  Bound by DRAM, less what a row's two sums
// keep waiting: 16384 x 4096 bf16 to 8-bit blocks in 83 to 87 us, 72.0 at
// the copy rate.
constexpr int kMaxStages = 8;

struct RowRing {
    uint32_t bar0;
    uint8_t *data;
    int stages, stage_bytes;
    volatile int *abort_flag;
    int *err;
    uint64_t limit_ns;
    __device__ __forceinline__ void init() const {
        if (threadIdx.x == 0) {
            for (int s = 0; s < stages; ++s) mbar_init(bar0 + 8u * s, 1);
            *abort_flag = 0;
            fence_barrier_init();
        }
        __syncthreads();
    }
    __device__ __forceinline__ uint8_t *stage(int s) const { return data + s * stage_bytes; }
    // One thread: begin the copies of stage s (`bytes` in all).
    __device__ __forceinline__ void expect(int s, uint32_t bytes) const { mbar_arrive_expect_tx(bar0 + 8u * s, bytes); }
    __device__ __forceinline__ void copy(int s, int at, const void *src, uint32_t bytes) const {
        bulk_load(smem_addr(data) + static_cast<uint32_t>(s * stage_bytes + at), src, bytes, bar0 + 8u * s);
    }
    // Thread 0: stages may be filled again, unless a wait ran out.
    __device__ __forceinline__ bool open() const { return *abort_flag == 0; }
    // Thread 0, at the end: after a wait that ran out, what is on its way is
    // waited for.  A stage's current phase is not known then: one of the two
    // waits returns at once, the other with the copies or, where none is under
    // way, at its share of the limit.
    __device__ __forceinline__ void drain() const {
        if (open()) return;
        const volatile int never = 0;
        for (int q = 0; q < 2 * stages; ++q) (void)mbar_wait(bar0 + 8u * (q >> 1), q & 1u, &never, limit_ns / kMaxStages);
    }
    // Every thread: a wait that ran out is recorded and lets the CTA run on
    // (all later waits return at once), so that no barrier is missed.
    __device__ __forceinline__ void wait(int s, uint32_t parity) const {
        if (mbar_wait(bar0 + 8u * s, parity, abort_flag, limit_ns)) return;
        if (*abort_flag != 0) return;
        atomicExch(err, kDevAbortNorm);
        *abort_flag = 1;
    }
};

// A ring whose first row comes and whose second never does (st_check_device_wait).
__device__ float4 g_checked_row[8];

__global__ void __launch_bounds__(64) norm_wait_check_kernel(uint64_t limit_ns, int *err) {
    __shared__ __align__(128) uint8_t rows[2 * sizeof(g_checked_row)];
    __shared__ uint64_t bars[2];
    __shared__ int aborted;
    constexpr uint32_t kBytes = sizeof(g_checked_row);
    const RowRing ring{smem_addr(bars), rows, 2, static_cast<int>(kBytes), &aborted, err, limit_ns};
    ring.init();
    if (threadIdx.x == 0) {
        ring.expect(0, kBytes);
        ring.copy(0, 0, g_checked_row, kBytes);
        ring.expect(1, kBytes);
    }
    ring.wait(0, 0);
    ring.wait(1, 0);
    __syncthreads();
    if (threadIdx.x == 0) ring.drain();
}

template <typename T>
__device__ __forceinline__ void read8(const uint8_t *row, int col, uint64_t (&f)[4]) {
    uint4 w[sizeof(T) / 2];
    const uint4 *src = reinterpret_cast<const uint4 *>(row + col * static_cast<int>(sizeof(T)));
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) w[i] = src[i];
    unpack8(w, f, T{});
}

template <typename T>
__device__ __forceinline__ void write8(T *dst, const uint64_t (&f)[4]) {
    uint4 w[sizeof(T) / 2];
    pack8(f, w, T{});
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) reinterpret_cast<uint4 *>(dst)[i] = w[i];
}

__device__ __forceinline__ uint64_t twice(float v) { return pack2(v, v); }

// Sums of N values over the warps of a CTA; every thread adds the warps'
// parts itself.  MOST: the largest N of the kernel's calls, whose two buffers
// `slots` holds.
template <int MOST, int N>
__device__ __forceinline__ void cta_sum(float (&v)[N], int warps, int warp, int lane, float4 *slots, int &slot) {
    float *mine = reinterpret_cast<float *>(slots + slot * MOST * 4);
    slot ^= 1;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) mine[i * 16 + warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
        v[i] = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (4 * q >= warps) break;
            const float4 s = reinterpret_cast<const float4 *>(mine)[i * 4 + q];  // slots past the last warp stay 0
            v[i] += (s.x + s.y) + (s.z + s.w);
        }
    }
}

// What a ring kernel's call has: every tensor, with no gate of a row's own or
// with a token's or an element's, known to the compiler; any other set is
// looked up in each row, which took the backward kernel a third of its issue
// slots (the kernel alone, 8192 x 4096 bf16 94.6 us, 72.0 known; a token's gate
// 98.6 and 77.6).
enum class Parts { kSome, kPlain, kToken, kFull };
inline Parts whole(int gate_mode) {
    return gate_mode == kGateToken ? Parts::kToken : gate_mode == kGateFull ? Parts::kFull : Parts::kPlain;
}

constexpr int kRowVecs = 4;  // chunks of 8 elements a thread: its share of the sums' and scales' cost stays small

// x is read twice from its stage instead of being kept: at 128 registers with
// both factors and r in them, 16 warps of an SM are at work.
template <typename TX, typename TR, Parts PARTS>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_rows_kernel(const NormArgs p, int warps, int stages) {
    constexpr int VPT = kRowVecs;
    constexpr bool ALL = PARTS != Parts::kSome;
    extern __shared__ __align__(128) uint8_t ring_smem[];
    __shared__ float4 slots[2 * 4];
    __shared__ uint64_t bars[kMaxStages];
    __shared__ int aborted;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t first = blockIdx.x, step = gridDim.x;
    const int cols = static_cast<int>(p.cols);
    const int x_bytes = cols * static_cast<int>(sizeof(TX)), r_bytes = cols * static_cast<int>(sizeof(TR));
    const bool token_gate = PARTS == Parts::kToken || (!ALL && p.gate_mode == kGateToken);
    const bool full_gate = PARTS == Parts::kFull || (!ALL && p.gate_mode == kGateFull);
    const int gate_size = p.gate.dtype == ST_F32 ? 4 : static_cast<int>(sizeof(TX)), gate_bytes = full_gate ? cols * gate_size : 0;
    const int r_at = (x_bytes + 127) / 128 * 128, gate_at = r_at + (r_bytes + 127) / 128 * 128;
    const RowRing ring{smem_addr(bars), ring_smem, stages, gate_at + (gate_bytes + 127) / 128 * 128, &aborted, p.err, p.limit_ns};
    if (threadIdx.x < 32) reinterpret_cast<float *>(slots)[threadIdx.x] = 0.0f;
    ring.init();
    pdl_wait();
    auto fetch = [&](int s, int64_t row) {
        ring.expect(s, static_cast<uint32_t>(x_bytes + r_bytes + gate_bytes));
        ring.copy(s, 0, static_cast<const TX *>(p.x.p) + row * p.x.ld, static_cast<uint32_t>(x_bytes));
        ring.copy(s, r_at, static_cast<const TR *>(p.r.p) + row * p.r.ld, static_cast<uint32_t>(r_bytes));
        if (full_gate)
            ring.copy(s, gate_at, static_cast<const uint8_t *>(p.gate.p) + row * p.gate.ld * gate_size, static_cast<uint32_t>(gate_bytes));
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; ++s)
            if (first + s * step < p.rows) fetch(s, first + s * step);

    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    const bool has_post = ALL || p.post.p != nullptr, has_pre = ALL || p.pre.p != nullptr;
    // branch factor alpha * gate * (post + offset), norm factor pre + offset
    uint64_t c1[VPT][4], c2[VPT][4];
    int col[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int base = (v * warps + warp) * kChunk;
        col[v] = base + lane * 8;
        float f[8], w[8] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = p.alpha;
        if (has_post) {
            load8_of<TX, true>(p.post, 0, base, lane, cols, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= w[j] + p.offset;
        }
        if (p.gate_mode == kGateChannel) {
            load8_of<TX, true>(p.gate, 0, base, lane, cols, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) c1[v][j] = pack2(f[2 * j], f[2 * j + 1]);
        if (has_pre) load8_of<TX, true>(p.pre, 0, base, lane, cols, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) c2[v][j] = pack2(w[2 * j] + p.offset, w[2 * j + 1] + p.offset);
    }

    int slot = 0, s = 0;
    uint32_t ph = 0;
    for (int64_t row = first; row < p.rows; row += step) {
        float token = 1.0f;
        if (token_gate) token = load1_of<TX>(p.gate, row);
        ring.wait(s, ph);
        const uint8_t *stage = ring.stage(s);
        float inv = token;
        if (has_post) {
            uint64_t a = 0;
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                if (col[v] >= cols) continue;
                uint64_t x[4];
                read8<TX>(stage, col[v], x);
#pragma unroll
                for (int j = 0; j < 4; ++j) a = fma2(x[j], x[j], a);
            }
            float sum[1] = {lo2(a) + hi2(a)};
            cta_sum<1>(sum, warps, warp, lane, slots, slot);
            inv = token * rsqrtf(sum[0] * inv_cols + p.eps);
        }
        const uint64_t inv2 = twice(inv);
        uint64_t a = 0, r[VPT][4];
        TR *to = static_cast<TR *>(p.r_out.p) + row * p.r_out.ld;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) r[v][j] = 0;
            if (col[v] >= cols) continue;
            uint64_t x[4];
            read8<TX>(stage, col[v], x);
            read8<TR>(stage + r_at, col[v], r[v]);
            if (full_gate) {
                uint64_t gate[4];
                if (gate_size == 4) read8<float>(stage + gate_at, col[v], gate);
                else read8<TX>(stage + gate_at, col[v], gate);
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = mul2(x[j], gate[j]);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                r[v][j] = fma2(mul2(x[j], c1[v][j]), inv2, r[v][j]);
                a = fma2(r[v][j], r[v][j], a);
            }
            write8<TR>(to + col[v], r[v]);
        }
        float sum[1] = {lo2(a) + hi2(a)};
        cta_sum<1>(sum, warps, warp, lane, slots, slot);
        // every thread has read the stage: the next row that it is for may come in
        if (threadIdx.x == 0 && row + stages * step < p.rows && ring.open()) fetch(s, row + stages * step);
        if (has_pre) {
            const uint64_t inv_r = twice(rsqrtf(sum[0] * inv_cols + p.eps));
            float top[VPT];
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                top[v] = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    r[v][j] = mul2(mul2(r[v][j], c2[v][j]), inv_r);
                    top[v] = max_abs(top[v], lo2(r[v][j]), hi2(r[v][j]));
                }
                if (!p.h_fp8 && col[v] < cols) write8<TX>(static_cast<TX *>(p.h.p) + row * p.h.ld + col[v], r[v]);
            }
            if (p.h_fp8) {  // 16 lanes hold a block of 128
                uint8_t *h = static_cast<uint8_t *>(p.h.p) + row * p.h.ld;
                const float scale = fp8_scale(max_of_four(top, lane), p.h_e5m2 ? 57344.0f : 448.0f);
                const float inverse = __frcp_rn(scale);
                const int mine = (lane >> 2) & 3;
                const int block = (mine * warps + warp) * 2 + (lane >> 4);
                if ((lane & 3) == 0 && block * 128 < cols) p.h_scale[row * p.hs0 + block * p.hs1] = scale;
#pragma unroll
                for (int v = 0; v < VPT; ++v) {
                    const float k = __shfl_sync(0xffffffffu, inverse, (lane & 16) | (v * 4));
                    if (col[v] < cols)
                        *reinterpret_cast<uint2 *>(h + col[v]) = p.h_e5m2 ? to_fp8x8<true>(r[v], k) : to_fp8x8<false>(r[v], k);
                }
            }
        }
        if (++s == stages) {
            s = 0;
            ph ^= 1u;
        }
    }
    if (threadIdx.x == 0) ring.drain();
    pdl_trigger();
}

// The sums over a group's rows, in shared memory: thread t's 8 elements of
// (plane, v) are two float4 at [plane][v][half][t], its own and free of bank
// conflicts.  The traffic is 8 bytes an element and plane beside the 12 of a
// 16-bit row's six streams, and shared memory moves five times what HBM
// does; in registers the sums would halve the rows in flight.
template <int VPT>
struct Sums {
    float4 *mine;
    __device__ __forceinline__ Sums(float4 *smem) : mine(smem + threadIdx.x) {}
    __device__ __forceinline__ float4 &at(int plane, int v, int half) {
        return mine[((plane * VPT + v) * 2 + half) * blockDim.x];
    }
    __device__ __forceinline__ void add(int plane, int v, const float (&f)[8]) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float4 &a = at(plane, v, h);
            float4 s = a;
            s.x += f[4 * h];
            s.y += f[4 * h + 1];
            s.z += f[4 * h + 2];
            s.w += f[4 * h + 3];
            a = s;
        }
    }
};

// planes: which sums are kept, and in what order (-1: not kept).
struct Planes {
    int pre, post, gate, count;
};

// out: [planes.count][groups][cols], one row a group.
template <typename TX, typename TR, int VPT, bool VEC>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_backward_kernel(const NormBackwardArgs p, int warps,
                                                                             const Planes planes, float *out) {
    extern __shared__ float4 sums_smem[];
    __shared__ float slots[2 * 3 * 32];
    const RowGroup g(warps);
    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    const bool has_x = p.x.p != nullptr, has_post = p.post.p != nullptr, has_pre = p.pre.p != nullptr;
    const int cols = static_cast<int>(p.cols);
    int slot = 0;
    Sums<VPT> sums(sums_smem);
    for (int i = 0; i < planes.count; ++i)
#pragma unroll
        for (int v = 0; v < VPT; ++v)
#pragma unroll
            for (int h = 0; h < 2; ++h) sums.at(i, v, h) = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    pdl_wait();

    for (int64_t row = g.first; row < p.rows; row += g.step) {
        Raw8<TX> x[VPT];
        float d[VPT][8];  // dr', then dr, then du
        if (has_x) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) x[v] = load_raw<TX, VEC>(p.x, row, g.base(v), g.lane, cols);
        }
        Raw8<TR> dres[VPT];
        if (p.d_residual.p != nullptr) {
#pragma unroll
            for (int v = 0; v < VPT; ++v) dres[v] = load_raw<TR, VEC>(p.d_residual, row, g.base(v), g.lane, cols);
        }
        float s[3] = {0.0f, 0.0f, 0.0f};
        if (has_x && has_post) {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) s[2] += x[v][j] * x[v][j];
        }
        float inv_x = 1.0f;
        if (has_pre) {
            Raw8<TR> r[VPT];
            Raw8<TX> dh[VPT];
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                r[v] = load_raw<TR, VEC>(p.r, row, g.base(v), g.lane, cols);
                dh[v] = load_raw<TX, VEC>(p.d_normed, row, g.base(v), g.lane, cols);
            }
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                float w[8];
                load8_of<TX, VEC>(p.pre, 0, g.base(v), g.lane, cols, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float rj = r[v][j];
                    s[0] += rj * rj;
                    s[1] += rj * (dh[v][j] * (w[j] + p.offset));
                }
            }
            row_sum(s, g.warps, g.warp, g.lane, slots, slot);
            const float inv = rsqrtf(s[0] * inv_cols + p.eps);
            const float mean = inv * s[1] * inv_cols;  // of t * R
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                float w[8], dw[8];
                load8_of<TX, VEC>(p.pre, 0, g.base(v), g.lane, cols, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float hat = r[v][j] * inv, dhj = dh[v][j];
                    dw[j] = dhj * hat;
                    d[v][j] = inv * (dhj * (w[j] + p.offset) - hat * mean);
                }
                if (planes.pre >= 0) sums.add(planes.pre, v, dw);
            }
        } else {
            if (has_x && has_post) row_sum(s, g.warps, g.warp, g.lane, slots, slot);
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) d[v][j] = 0.0f;
        }
        if (has_post) inv_x = rsqrtf(s[2] * inv_cols + p.eps);
        if (p.d_residual.p != nullptr) {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
#pragma unroll
                for (int j = 0; j < 8; ++j) d[v][j] += dres[v][j];
        }
        if (p.dr.p != nullptr) {
#pragma unroll
            for (int v = 0; v < VPT; ++v)
                store8<TR, VEC>(static_cast<TR *>(p.dr.p) + row * p.dr.ld, g.base(v), g.lane, cols, d[v]);
        }
        if (!has_x) continue;

        float token = p.alpha;
        if (p.gate_mode == kGateToken) token *= load1_of<TX>(p.gate, row);
        // with X = x * inv_x, t = du * (post + offset): sums of t * X and of dgate
        float e[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            float w[8], gt[8], dw[8], dg[8];
            if (has_post) {
                load8_of<TX, VEC>(p.post, 0, g.base(v), g.lane, cols, w);
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] += p.offset;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = 1.0f;
            }
            if (p.gate_mode == kGateChannel || p.gate_mode == kGateFull) {
                load8_of<TX, VEC>(p.gate, p.gate_mode == kGateFull ? row : 0, g.base(v), g.lane, cols, gt);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) gt[j] = 1.0f;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float hat = x[v][j] * inv_x;
                dg[j] = p.alpha * d[v][j] * (hat * w[j]);
                d[v][j] *= token * gt[j];
                dw[j] = d[v][j] * hat;
                e[0] += dw[j] * w[j];
                e[1] += dg[j];
            }
            if (planes.post >= 0) sums.add(planes.post, v, dw);
            if (planes.gate >= 0) sums.add(planes.gate, v, dg);
            if (p.gate_mode == kGateFull) {
                if (p.dgate.dtype == ST_F32)
                    store8<float, VEC>(static_cast<float *>(p.dgate.p) + row * p.dgate.ld, g.base(v), g.lane, cols, dg);
                else
                    store8<TX, VEC>(static_cast<TX *>(p.dgate.p) + row * p.dgate.ld, g.base(v), g.lane, cols, dg);
            }
        }
        if (has_post || p.gate_mode == kGateToken) row_sum(e, g.warps, g.warp, g.lane, slots, slot);
        if (p.gate_mode == kGateToken && g.warp == 0 && g.lane == 0)
            static_cast<float *>(p.dgate.p)[row * p.dgate.ld] = e[1];
        const float mean = e[0] * inv_cols;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            if (has_post) {
                float w[8];
                load8_of<TX, VEC>(p.post, 0, g.base(v), g.lane, cols, w);
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    d[v][j] = inv_x * (d[v][j] * (w[j] + p.offset) - x[v][j] * inv_x * mean);
            }
            store8<TX, VEC>(static_cast<TX *>(p.dx.p) + row * p.dx.ld, g.base(v), g.lane, cols, d[v]);
        }
    }

    for (int i = 0; i < planes.count; ++i) {
        float *to = out + (i * g.step + g.first) * p.cols;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
            const float4 a = sums.at(i, v, 0), b = sums.at(i, v, 1);
            const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            store8<float, VEC>(to, g.base(v), g.lane, cols, f);
        }
    }
    pdl_trigger();
}

// Backward for many rows on 16-byte boundaries, as residual_norm_rows_kernel:
// a ring of rows of x, dh, r and dr', the factors and the sums over rows in
// registers.  With X = x * inv_x and c1 = alpha * gate * (post + offset) (the
// gate only where it is a channel's; a token's or element's is g), one sum
// over rows S = sum dr * X * g serves dpost = alpha * gate * S and a channel's
// dgate = alpha * (post + offset) * S, and one over the row, sum dr * X * c1
// (times an element's g), the mean in dx and a token's dgate.  Bound by DRAM
// and by issue slots (8192 x 4096 bf16 with its column sums in 80 to 81 us, 61.5
// at the copy rate; 64 registers a thread and twice the warps spilled: 113
// against 95 then).
constexpr int kBackVecs = 2;

template <typename TX, typename TR, Parts PARTS>
__global__ void __launch_bounds__(kMaxThreads) residual_norm_backward_rows_kernel(const NormBackwardArgs p, int warps,
                                                                                  const Planes planes, float *out,
                                                                                  int stages) {
    constexpr int VPT = kBackVecs;
    constexpr bool ALL = PARTS != Parts::kSome, PLAIN = PARTS == Parts::kPlain;
    extern __shared__ __align__(128) uint8_t ring_smem[];
    __shared__ float4 slots[2 * 3 * 4];
    __shared__ uint64_t bars[kMaxStages];
    __shared__ int aborted;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t first = blockIdx.x, step = gridDim.x;
    const int cols = static_cast<int>(p.cols);
    const bool has_x = ALL || p.x.p != nullptr, has_post = ALL || p.post.p != nullptr, has_pre = ALL || p.pre.p != nullptr;
    const bool has_dr = ALL || p.d_residual.p != nullptr;
    const bool token = PARTS == Parts::kToken || (!ALL && p.gate_mode == kGateToken);
    const bool full = PARTS == Parts::kFull || (!ALL && p.gate_mode == kGateFull);
    const uint32_t x_bytes = static_cast<uint32_t>(cols) * sizeof(TX), r_bytes = static_cast<uint32_t>(cols) * sizeof(TR);
    const int x_room = (x_bytes + 127) / 128 * 128, r_room = (r_bytes + 127) / 128 * 128;
    const int dh_at = has_x ? x_room : 0, r_at = dh_at + (has_pre ? x_room : 0), dr_at = r_at + (has_pre ? r_room : 0);
    const int gate_size = p.gate.dtype == ST_F32 ? 4 : static_cast<int>(sizeof(TX)), gate_at = dr_at + (has_dr ? r_room : 0);
    const uint32_t gate_bytes = full ? static_cast<uint32_t>(cols * gate_size) : 0;
    const RowRing ring{smem_addr(bars), ring_smem, stages, gate_at + static_cast<int>((gate_bytes + 127) / 128 * 128), &aborted, p.err, p.limit_ns};
    if (threadIdx.x < 32)
        for (int i = 0; i < 3; ++i) reinterpret_cast<float *>(slots)[threadIdx.x + 32 * i] = 0.0f;
    ring.init();
    pdl_wait();
    auto fetch = [&](int s, int64_t row) {
        ring.expect(s, (has_x ? x_bytes : 0) + (has_pre ? x_bytes + r_bytes : 0) + (has_dr ? r_bytes : 0) + gate_bytes);
        if (full)
            ring.copy(s, gate_at, static_cast<const uint8_t *>(p.gate.p) + row * p.gate.ld * gate_size, gate_bytes);
        if (has_x) ring.copy(s, 0, static_cast<const TX *>(p.x.p) + row * p.x.ld, x_bytes);
        if (has_pre) {
            ring.copy(s, dh_at, static_cast<const TX *>(p.d_normed.p) + row * p.d_normed.ld, x_bytes);
            ring.copy(s, r_at, static_cast<const TR *>(p.r.p) + row * p.r.ld, r_bytes);
        }
        if (has_dr) ring.copy(s, dr_at, static_cast<const TR *>(p.d_residual.p) + row * p.d_residual.ld, r_bytes);
    };
    if (threadIdx.x == 0)
        for (int s = 0; s < stages; ++s)
            if (first + s * step < p.rows) fetch(s, first + s * step);

    const float inv_cols = 1.0f / static_cast<float>(p.cols);
    uint64_t c1[VPT][4], c2[VPT][4], spre[VPT][4], spost[VPT][4];
    int col[VPT];
#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        const int base = (v * warps + warp) * kChunk;
        col[v] = base + lane * 8;
        float f[8], w[8] = {};
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = p.alpha;
        if (has_post) {
            load8_of<TX, true>(p.post, 0, base, lane, cols, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= w[j] + p.offset;
        }
        if (p.gate_mode == kGateChannel) {
            load8_of<TX, true>(p.gate, 0, base, lane, cols, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= w[j];
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) c1[v][j] = pack2(f[2 * j], f[2 * j + 1]);
        if (has_pre) load8_of<TX, true>(p.pre, 0, base, lane, cols, w);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            c2[v][j] = pack2(w[2 * j] + p.offset, w[2 * j + 1] + p.offset);
            spre[v][j] = spost[v][j] = 0;
        }
    }

    int slot = 0, s = 0;
    uint32_t ph = 0;
    for (int64_t row = first; row < p.rows; row += step) {
        float g = 1.0f;
        if (token) g = load1_of<TX>(p.gate, row);
        ring.wait(s, ph);
        const uint8_t *stage = ring.stage(s);
        float sum[3] = {0.0f, 0.0f, 0.0f};  // of r^2, r t and x^2
        if (has_pre || has_post) {
            uint64_t a[3] = {0, 0, 0};
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                if (col[v] >= cols) continue;
                if (has_pre) {
                    uint64_t r[4], dh[4];
                    read8<TR>(stage + r_at, col[v], r);
                    read8<TX>(stage + dh_at, col[v], dh);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        a[0] = fma2(r[j], r[j], a[0]);
                        a[1] = fma2(r[j], mul2(dh[j], c2[v][j]), a[1]);
                    }
                }
                if (has_post) {
                    uint64_t x[4];
                    read8<TX>(stage, col[v], x);
#pragma unroll
                    for (int j = 0; j < 4; ++j) a[2] = fma2(x[j], x[j], a[2]);
                }
            }
#pragma unroll
            for (int i = 0; i < 3; ++i) sum[i] = lo2(a[i]) + hi2(a[i]);
            cta_sum<3>(sum, warps, warp, lane, slots, slot);
        }
        const float inv_r = rsqrtf(sum[0] * inv_cols + p.eps);
        const float inv_x = has_post ? rsqrtf(sum[2] * inv_cols + p.eps) : 1.0f;
        const uint64_t inv_r2 = twice(inv_r), inv_x2 = twice(inv_x), less = twice(-inv_r * sum[1] * inv_cols);
        uint64_t d[VPT][4], hat[VPT][4], e = 0;
#pragma unroll
        for (int v = 0; v < VPT; ++v) {
#pragma unroll
            for (int j = 0; j < 4; ++j) d[v][j] = hat[v][j] = 0;
            if (col[v] >= cols) continue;
            if (has_dr) read8<TR>(stage + dr_at, col[v], d[v]);
            if (has_pre) {
                uint64_t r[4], dh[4];
                read8<TR>(stage + r_at, col[v], r);
                read8<TX>(stage + dh_at, col[v], dh);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint64_t R = mul2(r[j], inv_r2);
                    spre[v][j] = fma2(dh[j], R, spre[v][j]);
                    d[v][j] = fma2(inv_r2, fma2(R, less, mul2(dh[j], c2[v][j])), d[v][j]);
                }
            }
            if (ALL || p.dr.p != nullptr) write8<TR>(static_cast<TR *>(p.dr.p) + row * p.dr.ld + col[v], d[v]);
            if (!has_x) continue;
            read8<TX>(stage, col[v], hat[v]);
            uint64_t gate[4] = {twice(g), twice(g), twice(g), twice(g)}, q[4];
            if (full) {
                if (gate_size == 4) read8<float>(stage + gate_at, col[v], gate);
                else read8<TX>(stage + gate_at, col[v], gate);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                hat[v][j] = mul2(hat[v][j], inv_x2);
                q[j] = mul2(d[v][j], hat[v][j]);
                spost[v][j] = PLAIN ? add2(q[j], spost[v][j]) : fma2(q[j], gate[j], spost[v][j]);
                q[j] = mul2(q[j], c1[v][j]);
                e = full ? fma2(q[j], gate[j], e) : add2(q[j], e);
                d[v][j] = mul2(d[v][j], c1[v][j]);
                if (!PLAIN) d[v][j] = mul2(d[v][j], gate[j]);
            }
            if (full) {
                if (p.dgate.dtype == ST_F32) write8<float>(static_cast<float *>(p.dgate.p) + row * p.dgate.ld + col[v], q);
                else write8<TX>(static_cast<TX *>(p.dgate.p) + row * p.dgate.ld + col[v], q);
            }
        }
        float es[1] = {lo2(e) + hi2(e)};
        cta_sum<3>(es, warps, warp, lane, slots, slot);
        // every thread has read the stage: the next row that it is for may come in
        if (threadIdx.x == 0 && row + stages * step < p.rows && ring.open()) fetch(s, row + stages * step);
        if (has_x) {
            if (token && threadIdx.x == 0) static_cast<float *>(p.dgate.p)[row * p.dgate.ld] = es[0];
            const uint64_t minus = twice(has_post ? (PLAIN ? -es[0] : -g * es[0]) * inv_cols : 0.0f);
#pragma unroll
            for (int v = 0; v < VPT; ++v) {
                if (col[v] >= cols) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) d[v][j] = mul2(inv_x2, fma2(hat[v][j], minus, d[v][j]));
                write8<TX>(static_cast<TX *>(p.dx.p) + row * p.dx.ld + col[v], d[v]);
            }
        }
        if (++s == stages) {
            s = 0;
            ph ^= 1u;
        }
    }

#pragma unroll
    for (int v = 0; v < VPT; ++v) {
        if (col[v] >= cols) continue;
        if (ALL || planes.pre >= 0) write8<float>(out + (planes.pre * step + first) * p.cols + col[v], spre[v]);
        if (ALL || planes.post >= 0) write8<float>(out + (planes.post * step + first) * p.cols + col[v], spost[v]);
    }
    if (threadIdx.x == 0) ring.drain();
    pdl_trigger();
}

// One sum over rows: out[c] = scale * (factor[c] + offset) * sum over groups
// of sums[plane][g][c] (without a factor, scale * the sum).
struct ColumnSum {
    float *out = nullptr;
    int plane = 0;
    float scale = 1.0f, offset = 0.0f;
    NormView factor;
};
struct ColumnSums {
    ColumnSum sum[3];
    int count = 0;
};

// In a fixed order: 1024 / W threads a column, each every (1024 / W)th group,
// then a sum over them.  W columns a CTA: 32 (two planes of 296 groups of 4096
// columns in 7.9 us), or 8, a sector, where that would leave half of the SMs
// idle: narrow rows have many groups (bf16 backward of 65536 x 256 in 55.8 us
// with 32, 52.8 with 8; 32768 x 512 on an f32 stream in 65.0 and 62.1; but 16384
// x 2048 in 72.3 and 73.5).  blockIdx.y picks the plane, read once for all its sums.
template <typename T, int W>
__global__ void __launch_bounds__(1024) column_sums_kernel(const float *sums, int groups, int cols, const ColumnSums todo) {
    pdl_wait();
    constexpr int kRows = 1024 / W;
    __shared__ float part[kRows][W + 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int at = static_cast<int>(threadIdx.x) % W, first = static_cast<int>(threadIdx.x) / W;
    const int c = static_cast<int>(blockIdx.x) * W + at;
    const float *src = sums + static_cast<int64_t>(blockIdx.y) * groups * cols + c;
    float s = 0.0f;
    if (c < cols) {
        int i = first;
        for (; i + 3 * kRows < groups; i += 4 * kRows) {  // four loads in flight
            const float v0 = src[static_cast<int64_t>(i) * cols], v1 = src[static_cast<int64_t>(i + kRows) * cols];
            const float v2 = src[static_cast<int64_t>(i + 2 * kRows) * cols], v3 = src[static_cast<int64_t>(i + 3 * kRows) * cols];
            s += (v0 + v1) + (v2 + v3);
        }
        for (; i < groups; i += kRows) s += src[static_cast<int64_t>(i) * cols];
    }
    part[first][at] = s;
    __syncthreads();
    if (warp < W) {
        s = 0.0f;
#pragma unroll
        for (int k = 0; k < kRows; k += 32) s += part[k + lane][warp];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    }
    const int mine = static_cast<int>(blockIdx.x) * W + warp;
    if (lane == 0 && warp < W && mine < cols) {
        for (int i = 0; i < todo.count; ++i) {
            const ColumnSum &o = todo.sum[i];
            if (o.plane != static_cast<int>(blockIdx.y)) continue;
            float v = s * o.scale;
            if (o.factor.p != nullptr)
                v *= (o.factor.dtype == ST_F32 ? static_cast<const float *>(o.factor.p)[mine]
                                               : to_float(static_cast<const T *>(o.factor.p)[mine])) +
                     o.offset;
            o.out[mine] = v;
        }
    }
    pdl_trigger();
}

// Row groups of the backward kernels: each leaves one row of partial sums.
// As many as CTAs of the ring kernel are at work, 16 warps an SM, and no
// fewer than two an SM.
constexpr int64_t kGroupSms = 148;

int64_t backward_groups(int64_t rows, int64_t cols) {
    const int64_t warps = cdiv(cols, kBackVecs * kChunk);
    const int64_t per_sm = warps >= 8 ? 2 : 16 / warps;
    return rows < kGroupSms * per_sm ? rows : kGroupSms * per_sm;
}

bool aligned_rows(const NormView &v, int64_t rows, size_t size, size_t to) {
    if (v.p == nullptr) return true;
    return reinterpret_cast<uintptr_t>(v.p) % to == 0 && (rows == 1 || v.ld * static_cast<int64_t>(size) % to == 0);
}

struct Shape {
    int vpt, warps, ctas, threads;
};

// `rows` rows of `cols` on up to `most` row groups; a chunk a thread up to `one_chunk` of them.
Shape shape_of(int64_t rows, int64_t cols, int64_t most, int one_chunk) {
    Shape s;
    const int64_t chunks = cdiv(cols, kChunk);
    if (chunks <= 2) {
        s.vpt = static_cast<int>(chunks);
    } else {
        s.vpt = chunks <= one_chunk ? 1 : chunks <= 32 ? 2 : 4;
    }
    s.warps = static_cast<int>(cdiv(chunks, s.vpt));
    const int64_t groups = rows < most ? rows : most;
    if (s.warps == 1) {
        s.threads = 32 * kRowsPerCta;
        s.ctas = static_cast<int>(cdiv(groups, kRowsPerCta));
    } else {
        s.threads = 32 * s.warps;
        s.ctas = static_cast<int>(groups);
    }
    return s;
}

template <typename TX, typename TR, int VPT, bool AHEAD>
int forward_vpt(const NormArgs &p, const Shape &s, bool vec, cudaStream_t stream) {
    if (vec)
        ST_CUDA_TRY(launch_kernel(residual_norm_kernel<TX, TR, VPT, true, AHEAD>, s.ctas, s.threads, 0, stream, p, s.warps));
    else
        ST_CUDA_TRY(launch_kernel(residual_norm_kernel<TX, TR, VPT, false, AHEAD>, s.ctas, s.threads, 0, stream, p, s.warps));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "residual_norm_kernel");
}

// Rows in flight of the ring kernels: as many stages of a row's bytes as fit beside the other CTAs of an SM.
template <typename Kern, typename... Args>
int launch_rows(Kern kern, uint64_t &attr_set, int threads, int stage_bytes, int64_t rows, int sm_count, cudaStream_t stream,
                int *groups, Args... args) {
    constexpr int kMostSmem = 200 * 1024;
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    int per_sm = kMaxThreads / threads;  // at 128 registers a thread
    while (per_sm > 1 && kMostSmem / per_sm / stage_bytes < 2) --per_sm;  // one row a CTA leaves nothing in flight: backward 8192 x 4096 f32 211 us, 183 so
    int stages = kMostSmem / per_sm / stage_bytes;
    stages = stages > kMaxStages ? kMaxStages : stages;
    const int64_t ctas = rows < sm_count * per_sm ? rows : sm_count * per_sm;
    if (groups != nullptr) *groups = static_cast<int>(ctas);
    ST_CUDA_TRY(launch_kernel(kern, static_cast<unsigned>(ctas), threads, static_cast<size_t>(stages) * stage_bytes, stream,
                              args..., stages));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "norm rows kernel");
}

int row_bytes(int64_t cols, size_t size) { return static_cast<int>((cols * size + 127) / 128 * 128); }

// Bytes of a row of the gate, where it has one of its own.
int gate_row_bytes(const NormView &gate, int mode, int64_t cols, size_t size) {
    return mode == kGateFull ? row_bytes(cols, gate.dtype == ST_F32 ? sizeof(float) : size) : 0;
}

template <typename TX, typename TR, Parts PARTS>
int forward_rows(const NormArgs &p, int sm_count, cudaStream_t stream) {
    static uint64_t attr_set = 0;  // one bit per device ordinal
    const int warps = static_cast<int>(cdiv(p.cols, kRowVecs * kChunk));
    return launch_rows(residual_norm_rows_kernel<TX, TR, PARTS>, attr_set, 32 * warps,
                       row_bytes(p.cols, sizeof(TX)) + row_bytes(p.cols, sizeof(TR)) +
                           gate_row_bytes(p.gate, p.gate_mode, p.cols, sizeof(TX)),
                       p.rows, sm_count, stream, nullptr, p,
                       warps);
}

template <typename TX, typename TR>
int forward_typed(const NormArgs &p, int sm_count, cudaStream_t stream) {
    auto side = [](const NormView &v) { return v.dtype == ST_F32 ? sizeof(float) : sizeof(TX); };
    const bool vec = aligned_rows(p.x, p.rows, sizeof(TX), 16) && aligned_rows(p.r, p.rows, sizeof(TR), 16) &&
                     aligned_rows(p.r_out, p.rows, sizeof(TR), 16) &&
                     (p.h_fp8 ? aligned_rows(p.h, p.rows, 1, 8) : aligned_rows(p.h, p.rows, sizeof(TX), 16)) &&
                     aligned_rows(p.post, 1, side(p.post), 16) && aligned_rows(p.pre, 1, side(p.pre), 16) &&
                     (p.gate_mode == kGateToken ||
                      aligned_rows(p.gate, p.gate_mode == kGateFull ? p.rows : 1, side(p.gate), 16));
    // one chunk a thread for few rows, whose latency counts, and for unaligned ones, whose single elements leave little in
    // flight otherwise: up to 4096 columns, 8192 of 16 bits (16001 x 4097 bf16 on an f32 stream, to 8 bits, 632 us with two,
    // 493 with one; 4000 x 8191 f32 137 and 163)
    const Shape s = shape_of(p.rows, p.cols, int64_t(1) << 30, p.rows < sm_count ? 16 : vec ? 0 : sizeof(TX) == 2 ? 32 : 16);
    if (vec && p.x.p != nullptr && p.r_out.p != nullptr && p.cols % 8 == 0 && p.cols > 2 * kChunk && p.rows >= 2 * sm_count)
        switch (p.post.p != nullptr && p.pre.p != nullptr ? whole(p.gate_mode) : Parts::kSome) {
        case Parts::kSome: return forward_rows<TX, TR, Parts::kSome>(p, sm_count, stream);
        case Parts::kPlain: return forward_rows<TX, TR, Parts::kPlain>(p, sm_count, stream);
        case Parts::kToken: return forward_rows<TX, TR, Parts::kToken>(p, sm_count, stream);
        case Parts::kFull: return forward_rows<TX, TR, Parts::kFull>(p, sm_count, stream);
        }
    if (s.vpt == 1)
        return p.rows < sm_count ? forward_vpt<TX, TR, 1, true>(p, s, vec, stream)
                                 : forward_vpt<TX, TR, 1, false>(p, s, vec, stream);
    if (s.vpt == 2) return forward_vpt<TX, TR, 2, false>(p, s, vec, stream);
    return forward_vpt<TX, TR, 4, false>(p, s, vec, stream);
}

template <typename TX, typename TR, int VPT, bool VEC>
int backward_launch(const NormBackwardArgs &p, const Shape &s, const Planes &planes, float *sums, cudaStream_t stream) {
    auto kern = residual_norm_backward_kernel<TX, TR, VPT, VEC>;
    static uint64_t attr_set = 0;  // one bit per device ordinal
    int dev = 0;
    ST_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !(attr_set & (1ull << dev))) {
        ST_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         3 * VPT * 8 * kMaxThreads * static_cast<int>(sizeof(float))));
        if (dev >= 0 && dev < 64) attr_set |= 1ull << dev;
    }
    const size_t smem = static_cast<size_t>(planes.count) * VPT * 8 * s.threads * sizeof(float);
    ST_CUDA_TRY(launch_kernel(kern, s.ctas, s.threads, smem, stream, p, s.warps, planes, sums));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "residual_norm_backward_kernel");
}

template <typename TX, typename TR, int VPT>
int backward_vpt(const NormBackwardArgs &p, const Shape &s, bool vec, const Planes &planes, float *sums,
                 cudaStream_t stream) {
    return vec ? backward_launch<TX, TR, VPT, true>(p, s, planes, sums, stream)
               : backward_launch<TX, TR, VPT, false>(p, s, planes, sums, stream);
}

template <typename T>
int finish_sums(const ColumnSums &todo, const float *sums, int planes, int64_t groups, int64_t cols, cudaStream_t stream) {
    if (todo.count == 0) return ST_OK;
    const bool narrow = cdiv(cols, 32) * planes < kGroupSms / 2 && groups > 32;
    ST_CUDA_TRY(launch_kernel(narrow ? column_sums_kernel<T, 8> : column_sums_kernel<T, 32>,
                              dim3(static_cast<unsigned>(cdiv(cols, narrow ? 8 : 32)), static_cast<unsigned>(planes)), 1024, 0,
                              stream, sums, static_cast<int>(groups), static_cast<int>(cols), todo));
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "column_sums_kernel");
}

template <typename TX, typename TR, Parts PARTS>
int backward_rows(const NormBackwardArgs &p, const Planes &planes, float *sums, cudaStream_t stream, int *groups) {
    static uint64_t attr_set = 0;  // one bit per device ordinal
    const int warps = static_cast<int>(cdiv(p.cols, kBackVecs * kChunk));
    const int stage = (p.x.p != nullptr ? row_bytes(p.cols, sizeof(TX)) : 0) +
                      (p.pre.p != nullptr ? row_bytes(p.cols, sizeof(TX)) + row_bytes(p.cols, sizeof(TR)) : 0) +
                      (p.d_residual.p != nullptr ? row_bytes(p.cols, sizeof(TR)) : 0) +
                      gate_row_bytes(p.gate, p.gate_mode, p.cols, sizeof(TX));
    return launch_rows(residual_norm_backward_rows_kernel<TX, TR, PARTS>, attr_set, 32 * warps, stage, p.rows,
                       static_cast<int>(kGroupSms), stream, groups, p, warps, planes, sums);
}

template <typename TX, typename TR>
int backward_typed(const NormBackwardArgs &p, float *sums, cudaStream_t stream) {
    auto side = [](const NormView &v) { return v.dtype == ST_F32 ? sizeof(float) : sizeof(TX); };
    const bool vec =
        aligned_rows(p.d_residual, p.rows, sizeof(TR), 16) && aligned_rows(p.d_normed, p.rows, sizeof(TX), 16) &&
        aligned_rows(p.x, p.rows, sizeof(TX), 16) && aligned_rows(p.r, p.rows, sizeof(TR), 16) &&
        aligned_rows(p.dx, p.rows, sizeof(TX), 16) && aligned_rows(p.dr, p.rows, sizeof(TR), 16) &&
        aligned_rows(p.post, 1, side(p.post), 16) && aligned_rows(p.pre, 1, side(p.pre), 16) &&
        (p.gate_mode == kGateToken || p.gate_mode == kGateNone ||
         aligned_rows(p.gate, p.gate_mode == kGateFull ? p.rows : 1, side(p.gate), 16)) &&
        (p.gate_mode != kGateFull || aligned_rows(p.dgate, p.rows, side(p.dgate), 16)) && p.cols % 4 == 0;
    Planes planes{-1, -1, -1, 0};
    ColumnSums todo;
    const bool channel = p.gate_mode == kGateChannel;
    if (vec && p.cols % 8 == 0 && p.cols <= kBackVecs * 8 * kMaxThreads && p.rows >= 2 * kGroupSms) {
        if (p.dpre != nullptr) {
            planes.pre = planes.count++;
            todo.sum[todo.count++] = {p.dpre, planes.pre, 1.0f, 0.0f, NormView{}};
        }
        if (p.dpost != nullptr || channel) planes.post = planes.count++;
        if (p.dpost != nullptr) todo.sum[todo.count++] = {p.dpost, planes.post, p.alpha, 0.0f, channel ? p.gate : NormView{}};
        if (channel) todo.sum[todo.count++] = {static_cast<float *>(p.dgate.p), planes.post, p.alpha, p.offset, p.post};
        const bool all = p.x.p != nullptr && p.post.p != nullptr && p.pre.p != nullptr && p.d_residual.p != nullptr &&
                         p.dr.p != nullptr && planes.pre >= 0 && planes.post >= 0;
        int groups = 0;
        switch (all ? whole(p.gate_mode) : Parts::kSome) {
        case Parts::kSome: ST_TRY((backward_rows<TX, TR, Parts::kSome>(p, planes, sums, stream, &groups))); break;
        case Parts::kPlain: ST_TRY((backward_rows<TX, TR, Parts::kPlain>(p, planes, sums, stream, &groups))); break;
        case Parts::kToken: ST_TRY((backward_rows<TX, TR, Parts::kToken>(p, planes, sums, stream, &groups))); break;
        case Parts::kFull: ST_TRY((backward_rows<TX, TR, Parts::kFull>(p, planes, sums, stream, &groups))); break;
        }
        return finish_sums<TX>(todo, sums, planes.count, groups, p.cols, stream);
    }
    const Shape s = shape_of(p.rows, p.cols, backward_groups(p.rows, p.cols), 0);
    const int64_t groups = s.warps == 1 ? static_cast<int64_t>(s.ctas) * kRowsPerCta : s.ctas;
    auto keep = [&](int &plane, float *to) {
        if (to == nullptr) return;
        plane = planes.count++;
        todo.sum[todo.count++] = {to, plane, 1.0f, 0.0f, NormView{}};
    };
    keep(planes.pre, p.dpre);
    keep(planes.post, p.dpost);
    if (channel) keep(planes.gate, static_cast<float *>(p.dgate.p));
    if (s.vpt == 1) ST_TRY((backward_vpt<TX, TR, 1>(p, s, vec, planes, sums, stream)));
    else if (s.vpt == 2) ST_TRY((backward_vpt<TX, TR, 2>(p, s, vec, planes, sums, stream)));
    else ST_TRY((backward_vpt<TX, TR, 4>(p, s, vec, planes, sums, stream)));
    return finish_sums<TX>(todo, sums, planes.count, groups, p.cols, stream);
}

}  // namespace

int launch_norm_wait_check(uint64_t limit_ns, int *dev_err, cudaStream_t stream) {
    norm_wait_check_kernel<<<1, 64, 0, stream>>>(limit_ns, dev_err);
    note_launch();
    const cudaError_t e = cudaPeekAtLastError();
    return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "norm_wait_check_kernel launch");
}

int launch_residual_norm(const NormArgs &args, int sm_count, int *dev_err, uint64_t timeout_ns, cudaStream_t stream) {
    NormArgs p = args;
    p.err = dev_err;
    p.limit_ns = timeout_ns;
    if (p.rows == 0) return ST_OK;
    if (p.cols > kMaxCols) return fail(ST_ERR_UNSUPPORTED, "residual_norm: at most 16384 columns");
    const bool wide = p.stream == ST_F32;
    if (p.branch == ST_F32) return forward_typed<float, float>(p, sm_count, stream);
    if (p.branch == ST_F16)
        return wide ? forward_typed<__half, float>(p, sm_count, stream) : forward_typed<__half, __half>(p, sm_count, stream);
    return wide ? forward_typed<__nv_bfloat16, float>(p, sm_count, stream)
                : forward_typed<__nv_bfloat16, __nv_bfloat16>(p, sm_count, stream);
}

int64_t residual_norm_backward_workspace(int64_t rows, int64_t cols) {
    // a CTA of single-warp rows may hold up to three groups without a row
    const int64_t groups = cdiv(backward_groups(rows, cols), kRowsPerCta) * kRowsPerCta;
    return 3 * groups * cols * static_cast<int64_t>(sizeof(float));
}

int launch_residual_norm_backward(const NormBackwardArgs &args, void *workspace, int *dev_err, uint64_t timeout_ns,
                                  cudaStream_t stream) {
    NormBackwardArgs p = args;
    p.err = dev_err;
    p.limit_ns = timeout_ns;
    if (p.cols > kMaxCols) return fail(ST_ERR_UNSUPPORTED, "residual_norm_backward: at most 16384 columns");
    float *sums = static_cast<float *>(workspace);
    if (p.rows == 0) {  // the sums over no rows
        float *dgate = p.gate_mode == kGateChannel ? static_cast<float *>(p.dgate.p) : nullptr;
        for (float *out : {p.dpre, p.dpost, dgate})
            if (out != nullptr) ST_CUDA_TRY(cudaMemsetAsync(out, 0, p.cols * sizeof(float), stream));
        return ST_OK;
    }
    const bool wide = p.stream == ST_F32;
    if (p.branch == ST_F32) return backward_typed<float, float>(p, sums, stream);
    if (p.branch == ST_F16)
        return wide ? backward_typed<__half, float>(p, sums, stream) : backward_typed<__half, __half>(p, sums, stream);
    return wide ? backward_typed<__nv_bfloat16, float>(p, sums, stream)
                : backward_typed<__nv_bfloat16, __nv_bfloat16>(p, sums, stream);
}

}  // namespace st
