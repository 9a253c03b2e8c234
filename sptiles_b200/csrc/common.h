// common.h -- shared host-side declarations of the runtime: status helpers,
// the kernel launchers each .cu file provides, and tensor-view utilities.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>
#include <string>
#include <utility>

#include "../../include/sptiles_b200.h"

namespace st {

// Record `msg` as the calling thread's last error and return `code`.
int fail(int code, const std::string &msg);
// Map a CUDA error to ST_ERR_CUDA / ST_ERR_OUT_OF_MEMORY with a message.
int cuda_fail(cudaError_t e, const char *what);

#define ST_CUDA_TRY(expr)                                        \
    do {                                                         \
        cudaError_t st_e_ = (expr);                              \
        if (st_e_ != cudaSuccess) return ::st::cuda_fail(st_e_, #expr); \
    } while (0)

#define ST_TRY(expr)                 \
    do {                             \
        int st_rc_ = (expr);         \
        if (st_rc_ != ST_OK) return st_rc_; \
    } while (0)

inline int64_t cdiv(int64_t a, int64_t b) { return (a + b - 1) / b; }

// ---- programmatic dependent launch
// Every kernel of this library is launched with programmatic stream
// serialisation (launch_kernel) and waits (pdl_wait) until the previous
// kernel on the stream has completed and its memory is visible before it
// touches global memory; only code before that -- barrier set-up, TMEM
// allocation, tensor-map prefetch -- overlaps the predecessor.  pdl_trigger
// lets the next kernel start launching: the GEMMs do it at once (one CTA per
// SM, so a successor's CTAs only take SMs this grid has left), the streaming
// kernels after their loop (their successors' CTAs would otherwise sit
// resident beside them).  SPTILES_B200_PDL=0 launches without the attribute.
#ifdef __CUDACC__
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void pdl_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_begin() {
    pdl_trigger();
    pdl_wait();
}
#endif

bool pdl_enabled();

template <typename... KArgs, typename... Args>
inline cudaError_t launch_kernel(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                 Args &&...args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = pdl_enabled() ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}

// Process-wide count of kernel launches issued by this library.
void note_launch(uint64_t n = 1);

inline size_t dtype_size(int dtype) {
    switch (dtype) {
    case ST_F32: return 4;
    case ST_F16: return 2;
    case ST_BF16: return 2;
    case ST_I32: return 4;
    default: return 0;
    }
}

// Error word each kernel with bounded waits may set (one int per device).
// Codes written by kernels:
constexpr int kDevAbortGemmProducer = 0x101;
constexpr int kDevAbortGemmMma = 0x102;
constexpr int kDevAbortGemmEpilogue = 0x103;
constexpr int kDevAbortGemmStreamK = 0x104;  // a split tile's partial never arrived
constexpr int kDevAbortNorm = 0x201;  // a row's copies never arrived
constexpr int kDevAbortWaitCheckBarrier = 0x1f0;  // st_check_device_wait: mbarrier wait ran out
constexpr int kDevAbortWaitCheckFlag = 0x1f1;     // st_check_device_wait: flag poll ran out

// One warp waits (bounded by limit_ns) on an mbarrier nothing arrives on
// (kind 0) or a flag nothing sets (kind 1), then records its abort code in
// dev_err and returns (diag.cu).
int launch_wait_check(int kind, uint64_t limit_ns, int *dev_err, cudaStream_t stream);
// The same for the norms' ring of rows (norm.cu) and a scaling warp of the
// 8-bit product, by rows or by columns (gemm_fp8.cu), with their own codes.
int launch_norm_wait_check(uint64_t limit_ns, int *dev_err, cudaStream_t stream);
int launch_fp8_wait_check(bool by_column, uint64_t limit_ns, int *dev_err, cudaStream_t stream);

// ---- launchers (implemented in vecadd.cu, gemm.cu, pack.cu) ----

// C[i] = A[i] + B[i] for i in [0, n), element strides sa, sb, sc.
int launch_vector_add_1d(const float *a, int64_t sa, const float *b, int64_t sb, float *c, int64_t sc, int64_t n,
                         int sm_count, cudaStream_t stream);
// C[r, q] = A[r, q] + B[r, q] for r < rows, q < cols with 2D element strides.
int launch_vector_add_2d(const float *a, const int64_t sa[2], const float *b, const int64_t sb[2], float *c,
                         const int64_t sc[2], int64_t rows, int64_t cols, int sm_count, cudaStream_t stream);

// C = fma(A, B, D) elementwise (f32), 2D strides; a rank-1 view is one row.
int launch_vector_fma(const float *a, const int64_t sa[2], const float *b, const int64_t sb[2], const float *d,
                      const int64_t sd[2], float *c, const int64_t sc[2], int64_t rows, int64_t cols, int sm_count,
                      cudaStream_t stream);
// C = A converted to C's dtype (ST_F32 / ST_F16 / ST_BF16), 2D strides.
int launch_cast(const void *a, int a_dtype, const int64_t sa[2], void *c, int c_dtype, const int64_t sc[2],
                int64_t rows, int64_t cols, int sm_count, cudaStream_t stream);

// Tensor-core GEMM plan.
struct GemmPlan {
    bool pair = false;  // CTA-pair kernel (cta_group::2): block_m 256, block_n 256
    int block_m = 128;
    int block_n = 256;
    int block_k = 64;  // elements per pipeline stage (128 bytes of K)
    int stages = 4;
    int ctas = 148;
    int tiles = 0;
};

// sk_mode: the stream-K mode to score a partial last wave with (-1: the
// environment's, else 1); force_pair: the CTA-pair plan whatever the scores
int plan_gemm(int in_dtype, int64_t m, int64_t n, int64_t k, int sm_count, GemmPlan *plan, int sk_mode = -1,
              bool force_pair = false);

// D = A' B'^T-style tensor-core GEMM on operands already laid out for TMA:
//   A: [M, K] row-major (K contiguous) of `ab_dtype` (ST_F16 / ST_BF16, or
//      ST_F32 meaning tf32 operands), row stride lda elements.
//   B: if b_k_major, [N, K] row-major (K contiguous), row stride ldb;
//      else [K, N] row-major (N contiguous), row stride ldb.
//   C: [M, N] with row stride ldc, element type c_dtype; bias[N] optional.
// Other GPUs' copies of C (CUDA IPC mappings over NVLink): the epilogue
// writes every finished chunk to each of them at the same offset as locally.
constexpr int kMaxPeers = 7;
struct PeerOutputs {
    void *base[kMaxPeers] = {};  // element (0, 0) of this call's C in each peer's copy
    int n = 0;
};

struct GemmArgs {
    PeerOutputs peers;
    int ab_dtype;
    const void *a;
    int64_t lda;
    const void *b;
    int64_t ldb;
    bool b_k_major;
    void *c;
    int64_t ldc;
    int c_dtype;
    const void *bias;
    int bias_dtype;
    int64_t m, n, k;
    // stream-K tail of the CTA-pair kernel (null: whole tiles only); sized by
    // stream_k_workspace_bytes, flags zero when idle
    float *sk_ws = nullptr;
    int *sk_flags = nullptr;
    // C already holds 0 + bias everywhere (the pack kernel preset it): an
    // L2-add stream-K launch then skips its own preset of the split tiles
    bool c_preset = false;
    // fold split tiles in a fixed order (ST_EXEC_DETERMINISTIC)
    bool deterministic = false;
    // the bytes from a row's end to the next 16-byte boundary are scratch of
    // this call's: a TMA store of C may write them
    bool c_padding = false;
    // ab_dtype ST_F32 with raw fp32 A [M, K] and B (K-major [N, K] or
    // N-contiguous [K, N]) and the true K: the CTA-pair kernel splits the
    // tiles into tf32 hi / lo itself (3xTF32); only when gemm_split_fp32_fits
    bool split_fp32 = false;
};
// Whether launch_gemm can take these fp32 operands raw (split_fp32): the
// plan picks the CTA-pair kernel and TMA can address A and B in place.
bool gemm_split_fp32_fits(const GemmArgs &args, int sm_count);
// Partial accumulators (one 256 x 256 fp32 tile per CTA pair) and arrival
// flags of the stream-K tail, for up to sm_count / 2 pairs.
size_t stream_k_workspace_bytes(int sm_count);
// True when launch_gemm folds split tiles through that workspace (an fp32 C
// of this GPU alone takes TMA reduce-adds instead and needs none).
bool gemm_uses_stream_k(const GemmArgs &args, int sm_count);
// How launch_gemm folds the tiles a stream-K schedule splits.
enum : int { kFoldNone = 0, kFoldExchange = 1, kFoldL2Add = 2 };
int stream_k_fold(const GemmArgs &args, int sm_count);
// For kFoldL2Add: 2 when split tiles fold ordered (needs the stream-K
// flags), 1 when C must hold 0 + bias first; 0 for other folds.
int stream_k_l2add_mode(const GemmArgs &args, int sm_count);
size_t stream_k_flag_offset(int sm_count);
int launch_gemm(const GemmArgs &args, int sm_count, int *dev_err, uint64_t timeout_ns, cudaStream_t stream);
// fp32 A and B used in place (TMA-addressable): the split into tf32 hi/lo
// happens in shared memory inside the kernel (args.ab_dtype must be ST_F32,
// args.k the true K).
int plan_gemm_x3(int64_t m, int64_t n, bool b_n_contiguous, int sm_count, GemmPlan *plan);
int launch_gemm_3xtf32(const GemmArgs &args, int sm_count, int *dev_err, uint64_t timeout_ns, cudaStream_t stream);

// 3xTF32 operand preparation.  x = hi + lo with hi, lo tf32-exact.
//   A [M, K] (strides sa0, sa1) -> Ap [M, 3*kp] = [hi | hi | lo], kp = round_up(K, 32)
//   B [K, N] (strides sb0, sb1) -> Bp [N, 3*kp] = [hi | lo | hi] (K contiguous)
// so that Ap @ Bp^T = hi*hi + hi*lo + lo*hi.
int64_t tf32_packed_k(int64_t k);
int launch_pack_a_tf32(const float *a, int64_t sa0, int64_t sa1, int64_t m, int64_t k, float *ap, int64_t kp,
                       cudaStream_t stream);
int launch_pack_b_tf32(const float *b, int64_t sb0, int64_t sb1, int64_t k, int64_t n, float *bp, int64_t kp,
                       cudaStream_t stream);
// CUDA places a kernel's code on the device at its first launch (lazy
// loading); these place the 3xTF32 path's packing and GEMM kernels on the
// current device now, for a caller that must make every device allocation
// of the library up front.
int preload_pack_tf32_kernels();
int preload_gemm_tf32_kernels();
// C[r, q] = 0 + bias[q] (or 0) for r < m, q < n, fp32, rows 16-byte aligned:
// the starting value of an L2-add stream-K launch (c == nullptr: nothing)
struct CPreset {
    float *c = nullptr;
    long long ldc = 0;
    const void *bias = nullptr;
    int bias_dtype = ST_F32;
    int m = 0, n = 0;
};
// both in one launch (B's transposing blocks first, then A's rows, whose
// blocks also write `preset`'s C when given)
int launch_pack_ab_tf32(const float *a, int64_t sa0, int64_t sa1, int64_t m, const float *b, int64_t sb0,
                        int64_t sb1, int64_t n, int64_t k, float *ap, float *bp, int64_t kp,
                        const CPreset *preset, cudaStream_t stream);
// Copy a 16-bit [rows, cols] matrix with arbitrary element strides into a
// dense row-major [rows, ld] buffer (ld >= cols, padding columns zeroed).
int launch_repack_16(const uint16_t *src, int64_t s0, int64_t s1, int64_t rows, int64_t cols, uint16_t *dst,
                     int64_t ld, cudaStream_t stream);

// ---- 8-bit operands with a scale per block of 128 along K (gemm_fp8.cu)
// One operand as [rows, k]: A's rows are M, B's rows are N.  Element (i, b)
// of `scale` belongs to rows [i << scale_shift, (i + 1) << scale_shift) and
// to K block b.
struct Fp8Operand {
    const void *data;
    int64_t rows, k;
    int64_t s_row, s_k;  // element strides
    uint32_t e5m2;       // 0: e4m3
    const void *scale;
    int64_t scale_row, scale_k;
    int scale_shift;  // 0 or 7
};

struct GemmFp8Args {
    Fp8Operand a, b;
    void *c;
    int64_t ldc;
    int c_dtype;
    const void *bias;
    int bias_dtype;
};

// Bytes of workspace for copies of the operands that TMA cannot address.
int64_t gemm_fp8_workspace_bytes(const Fp8Operand &a, const Fp8Operand &b);
int launch_gemm_fp8(const GemmFp8Args &args, void *workspace, int sm_count, int *dev_err, uint64_t timeout_ns,
                    cudaStream_t stream);

// q = fp8(a / scale) with one scale per block_rows x block_cols block (quantize.cu).
struct QuantizeArgs {
    const void *a;
    int a_dtype;
    int64_t sa0, sa1;
    void *q;
    bool e5m2;
    int64_t sq0, sq1;
    float *scale;
    int64_t ss0, ss1;
    int64_t rows, cols;
    int block_rows, block_cols;  // 1 x 128, 128 x 1 or 128 x 128
};
int launch_quantize_fp8(const QuantizeArgs &args, cudaStream_t stream);

// Dense copy of a strided byte matrix [rows, cols] into rows of `ld` bytes (a
// multiple of 16; the padding gets bytes of no meaning).
int launch_repack_8(const void *src, int64_t s0, int64_t s1, int64_t rows, int64_t cols, void *dst, int64_t ld,
                    int sm_count, cudaStream_t stream);
// C = bias (or 0) in every row: a product over nothing.
int launch_fill_bias(void *c, int64_t ldc, int c_dtype, const void *bias, int bias_dtype, int64_t m, int64_t n, int sm_count,
                     cudaStream_t stream);

// ---- 4-bit operands with a scale per block of 16 or 32 along K (quantize_fp4.cu, gemm_fp4.cu)
// Scales lie as [row / 128][block / 4][row % 32][row / 32 % 4][block % 4].
inline int64_t fp4_scale_bytes(int64_t rows, int64_t blocks) { return cdiv(rows, 128) * cdiv(blocks, 4) * 512; }

struct Quantize4Args {
    const void *a;
    int a_dtype;
    int64_t sa0, sa1;
    int64_t rows, cols;
    bool wide;  // blocks of 32 with e8m0 scales; else 16 with e4m3
    uint8_t *q;
    int64_t sq0;  // bytes; two codes a byte along a row
    uint8_t *scale;
    const float *maxima = nullptr;  // the tensor's known maximum; null: taken from a
    int n_maxima = 1;
    float *tensor_scale = nullptr;  // blocks of 16: where the tensor's scale goes
};
int64_t quantize_fp4_workspace_bytes();
int launch_quantize_fp4(const Quantize4Args &args, void *workspace, int sm_count, cudaStream_t stream);

struct Dequantize4Args {
    const uint8_t *q;
    int64_t sq0, sq1;
    int64_t rows, cols;
    bool wide;
    const uint8_t *scale;
    const float *tensor_scale;  // or null
    void *out;
    int out_dtype;
    int64_t so0, so1;
};
int launch_dequantize_fp4(const Dequantize4Args &args, int sm_count, cudaStream_t stream);

// One operand as [rows, k]: A's rows are M, B's rows are N; k in bytes (two elements each).
struct Fp4Operand {
    const void *data;
    int64_t rows, k;
    int64_t s_row, s_k;
    const void *scale;
    const float *tensor_scale;  // or null
};
struct GemmFp4Args {
    Fp4Operand a, b;
    bool wide;
    void *c;
    int64_t ldc;
    int c_dtype;
    const void *bias;
    int bias_dtype;
};
int64_t gemm_fp4_workspace_bytes(const Fp4Operand &a, const Fp4Operand &b);
int launch_gemm_fp4(const GemmFp4Args &args, void *workspace, int sm_count, int *dev_err, uint64_t timeout_ns,
                    cudaStream_t stream);

// ---- products by groups of rows (gemm_grouped.cu); group g is rows [ends[g - 1], ends[g])
constexpr int kGroupedMaxGroups = 1024;
struct GroupedArgs {
    bool weights;  // false: C [rows, n] = A [rows, k] @ B [groups, k, n];  true: C [groups, k, n] = A [rows, k]^T @ B [rows, n]
    int dtype;     // ST_F16 or ST_BF16
    int64_t groups, rows, k, n;
    const int *ends;
    const void *a;
    int64_t a_s0, a_s1;
    const void *b;
    int64_t b_g, b_s0, b_s1;
    void *c;
    int64_t c_g, ldc;
    int c_dtype;
    bool zero_rest;  // rows of no group become 0
};
int64_t gemm_grouped_workspace_bytes(const GroupedArgs &args);
int launch_gemm_grouped(const GroupedArgs &args, void *workspace, int sm_count, int *dev_err, uint64_t timeout_ns,
                        cudaStream_t stream);

// Norms around a block (norm.cu).  Strides in elements; unit column strides.
struct NormView {
    void *p = nullptr;
    int dtype = ST_F32;
    int64_t ld = 0;
};
enum : int { kGateNone = 0, kGateChannel = 1, kGateToken = 2, kGateFull = 3 };
struct NormArgs {
    int64_t rows, cols;
    float alpha, eps, offset;
    int branch, stream;  // types of x, h and their gradients, and of the residual stream, as the caller has checked them
    NormView x, r, r_out, h;
    NormView post, pre, gate;  // post, pre and a channel gate: one row; a token gate: ld per row
    int gate_mode = kGateNone;
    float *h_scale = nullptr;  // h is 8-bit: its scales per 1 x 128 block
    int64_t hs0 = 0, hs1 = 0;
    bool h_e5m2 = false, h_fp8 = false;
    int *err = nullptr;  // set by the launcher
    unsigned long long limit_ns = 0;
};
int launch_residual_norm(const NormArgs &args, int sm_count, int *dev_err, uint64_t timeout_ns, cudaStream_t stream);

struct NormBackwardArgs {
    int64_t rows, cols;
    float alpha, eps, offset;
    int branch, stream;  // as in NormArgs
    NormView d_residual, d_normed;  // p null: absent
    NormView x, r;                  // the branch and the updated stream
    NormView post, pre, gate;
    int gate_mode = kGateNone;
    NormView dx, dr, dgate;  // dgate: rows x cols (full) or float per row / column
    float *dpost = nullptr, *dpre = nullptr;
    int *err = nullptr;  // set by the launcher
    unsigned long long limit_ns = 0;
};
int64_t residual_norm_backward_workspace(int64_t rows, int64_t cols);
int launch_residual_norm_backward(const NormBackwardArgs &args, void *workspace, int *dev_err, uint64_t timeout_ns,
                                  cudaStream_t stream);

}  // namespace st
