// runtime.cu -- the host runtime behind the C ABI (include/sptiles_b200.h).
//
// It replaces the reference's Vulkan host (src/examples.cpp:133-448) and the
// Kompute runner (shaders/spirv_runtime.py:153-174): instead of building a
// pipeline from SPIR-V per call, a named cuda_tile entry is looked up in a
// registry of hand-written sm_100a kernels, its cutile_python_v1 bindings are
// turned back into tensor views, the cuda_tile grid is mapped onto the
// kernels' own launch shape, and the work is queued on a CUDA stream.
// Waits are bounded (an event poll with a deadline) where the reference
// waited on a fence forever (examples.cpp:439).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <chrono>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <initializer_list>
#include <string>
#include <thread>
#include <utility>
#include <vector>

#include "common.h"

namespace st {

static thread_local std::string g_last_error;
static std::atomic<uint64_t> g_launches{0};

void note_launch(uint64_t n) { g_launches.fetch_add(n, std::memory_order_relaxed); }

bool pdl_enabled() {
    static const bool on = [] {
        const char *v = std::getenv("SPTILES_B200_PDL");
        return !(v != nullptr && v[0] == '0');
    }();
    return on;
}

int fail(int code, const std::string &msg) {
    g_last_error = msg;
    return code;
}

int cuda_fail(cudaError_t e, const char *what) {
    const int code = (e == cudaErrorMemoryAllocation) ? ST_ERR_OUT_OF_MEMORY
                     : (e == cudaErrorNoDevice || e == cudaErrorInsufficientDriver) ? ST_ERR_NO_DEVICE
                                                                                     : ST_ERR_CUDA;
    return fail(code, std::string(what) + ": " + cudaGetErrorName(e) + " (" + cudaGetErrorString(e) + ")");
}

namespace {

constexpr uint32_t kDefaultTimeoutMs = 60000;
// bound for every on-device barrier wait of the tensor-core kernels
constexpr uint64_t kDeviceWaitLimitNs = 4ull * 1000 * 1000 * 1000;

// A device buffer the runtime owns and grows on demand (operand packing,
// staging of host-memory calls).  `ready` orders reuse across streams.
struct Workspace {
    void *ptr = nullptr;
    size_t bytes = 0;
    cudaEvent_t ready = nullptr;
};

struct DeviceState {
    int ordinal = 0;
    int sm_count = 0;
    cudaStream_t stream = nullptr;
    int *dev_err = nullptr;
    Workspace scratch;  // packed / repacked matmul operands
    Workspace stage;    // device copies of host-memory arguments
    Workspace sk;       // stream-K partials and flags of the CTA-pair GEMM (fixed size, flags zeroed)
    // host-memory calls: copies in and out run on their own streams so that
    // both PCIe directions overlap the kernels
    cudaStream_t copy_in = nullptr;
    cudaStream_t copy_out = nullptr;
    std::vector<cudaEvent_t> events;  // reusable ordering events
};

class DeviceGuard {
  public:
    explicit DeviceGuard(int dev) {
        cudaGetDevice(&prev_);
        cudaSetDevice(dev);
    }
    ~DeviceGuard() { cudaSetDevice(prev_); }

  private:
    int prev_ = 0;
};

}  // namespace
}  // namespace st

struct st_ctx {
    std::vector<st::DeviceState> devs;
};

namespace st {
namespace {

DeviceState *find_dev(st_ctx *ctx, int device) {
    if (!ctx || ctx->devs.empty()) return nullptr;
    if (device < 0) return &ctx->devs[0];
    for (auto &d : ctx->devs)
        if (d.ordinal == device) return &d;
    return nullptr;
}

int get_dev(st_ctx *ctx, int device, DeviceState **out) {
    if (!ctx) return fail(ST_ERR_INVALID_ARGUMENT, "null context");
    DeviceState *d = find_dev(ctx, device);
    if (!d) return fail(ST_ERR_INVALID_ARGUMENT, "device " + std::to_string(device) + " is not part of the context");
    *out = d;
    return ST_OK;
}

bool capturing(cudaStream_t stream) {
    cudaStreamCaptureStatus st = cudaStreamCaptureStatusNone;
    return cudaStreamIsCapturing(stream, &st) == cudaSuccess && st != cudaStreamCaptureStatusNone;
}

// Grow `ws` to at least `need` bytes for use on `stream`.  While `stream` is
// being captured into a CUDA graph the buffer must already be large enough
// (a warm-up call sizes it) and stream order alone sequences its users.
int ws_acquire(Workspace &ws, size_t need, cudaStream_t stream, void **out) {
    if (capturing(stream)) {
        if (need > ws.bytes)
            return fail(ST_ERR_UNSUPPORTED, "the workspace must be sized by an uncaptured call before graph capture");
        *out = ws.ptr;
        return ST_OK;
    }
    if (ws.ready == nullptr) ST_CUDA_TRY(cudaEventCreateWithFlags(&ws.ready, cudaEventDisableTiming));
    // a previous user on another stream must be done with the buffer
    ST_CUDA_TRY(cudaStreamWaitEvent(stream, ws.ready, 0));
    if (need > ws.bytes) {
        if (ws.ptr) {
            ST_CUDA_TRY(cudaStreamSynchronize(stream));
            ST_CUDA_TRY(cudaFree(ws.ptr));
            ws.ptr = nullptr;
            ws.bytes = 0;
        }
        const size_t rounded = (need + (size_t(2) << 20) - 1) & ~((size_t(2) << 20) - 1);
        ST_CUDA_TRY(cudaMalloc(&ws.ptr, rounded));
        ws.bytes = rounded;
    }
    *out = ws.ptr;
    return ST_OK;
}

int ws_release(Workspace &ws, cudaStream_t stream) {
    if (capturing(stream)) return ST_OK;
    ST_CUDA_TRY(cudaEventRecord(ws.ready, stream));
    return ST_OK;
}

void ws_free(Workspace &ws) {
    if (ws.ptr) cudaFree(ws.ptr);
    if (ws.ready) cudaEventDestroy(ws.ready);
    ws = Workspace{};
}

// The stream-K workspace: allocated with its flags zeroed by the first
// uncaptured matmul on the device (a capture before that runs whole tiles
// only), then ordered across streams like the other workspaces.
int sk_acquire(DeviceState *d, cudaStream_t stream, GemmArgs &g) {
    if (!d->sk.ptr) {
        if (capturing(stream)) return ST_OK;
        const size_t bytes = stream_k_workspace_bytes(d->sm_count);
        ST_CUDA_TRY(cudaMalloc(&d->sk.ptr, bytes));
        d->sk.bytes = bytes;
        ST_CUDA_TRY(cudaMemsetAsync(d->sk.ptr, 0, bytes, stream));
    }
    void *base = nullptr;
    ST_TRY(ws_acquire(d->sk, d->sk.bytes, stream, &base));
    g.sk_ws = static_cast<float *>(base);
    g.sk_flags = reinterpret_cast<int *>(static_cast<uint8_t *>(base) + stream_k_flag_offset(d->sm_count));
    return ST_OK;
}

// After an abort a split tile's flags may still be raised: clear them.
void sk_reset(DeviceState *d) {
    if (!d->sk.ptr) return;
    DeviceGuard guard(d->ordinal);
    const size_t off = stream_k_flag_offset(d->sm_count);
    cudaMemset(static_cast<uint8_t *>(d->sk.ptr) + off, 0, d->sk.bytes - off);
    cudaDeviceSynchronize();
}

// Bounded wait for `stream`, then collect a kernel abort from the error word.
int bounded_sync(DeviceState *d, cudaStream_t stream, uint32_t timeout_ms) {
    if (timeout_ms == 0) timeout_ms = kDefaultTimeoutMs;
    cudaEvent_t ev;
    ST_CUDA_TRY(cudaEventCreateWithFlags(&ev, cudaEventDisableTiming));
    cudaError_t e = cudaEventRecord(ev, stream);
    if (e != cudaSuccess) {
        cudaEventDestroy(ev);
        return cuda_fail(e, "cudaEventRecord");
    }
    const auto deadline = std::chrono::steady_clock::now() + std::chrono::milliseconds(timeout_ms);
    int sleep_us = 2;
    while ((e = cudaEventQuery(ev)) == cudaErrorNotReady) {
        if (std::chrono::steady_clock::now() > deadline) {
            cudaEventDestroy(ev);
            return fail(ST_ERR_TIMEOUT, "work did not finish within " + std::to_string(timeout_ms) + " ms");
        }
        std::this_thread::sleep_for(std::chrono::microseconds(sleep_us));
        if (sleep_us < 200) sleep_us *= 2;
    }
    cudaEventDestroy(ev);
    if (e != cudaSuccess) return cuda_fail(e, "kernel execution");
    int code = 0;
    ST_CUDA_TRY(cudaMemcpy(&code, d->dev_err, sizeof(int), cudaMemcpyDeviceToHost));
    if (code != 0) {
        ST_CUDA_TRY(cudaMemset(d->dev_err, 0, sizeof(int)));
        sk_reset(d);
        return fail(ST_ERR_DEVICE_ABORT, "a kernel gave up a bounded wait (code " + std::to_string(code) + ")");
    }
    return ST_OK;
}

struct ExecCtx {
    DeviceState *dev = nullptr;
    cudaStream_t stream = nullptr;
    uint32_t timeout_ms = kDefaultTimeoutMs;
    int flags = 0;
};

constexpr const char *kAllDevicesScope =
    "ST_EXEC_ALL_DEVICES applies to st_vector_add_host, st_matmul_host and st_launch with ST_EXEC_HOST_BUFFERS only";

// `split_ok`: the call implements ST_EXEC_ALL_DEVICES (the host-memory
// vector_add and matmul); every other entry point refuses the flag rather
// than running on one device only.
int resolve_exec(st_ctx *ctx, const st_exec *exec, ExecCtx *out, bool split_ok = false) {
    if (exec && (exec->flags & ST_EXEC_ALL_DEVICES) && !split_ok) return fail(ST_ERR_INVALID_ARGUMENT, kAllDevicesScope);
    const int device = exec ? exec->device : -1;
    ST_TRY(get_dev(ctx, device, &out->dev));
    out->stream = (exec && exec->stream) ? static_cast<cudaStream_t>(exec->stream) : out->dev->stream;
    out->timeout_ms = (exec && exec->timeout_ms) ? exec->timeout_ms : kDefaultTimeoutMs;
    out->flags = exec ? exec->flags : 0;
    return ST_OK;
}

// ------------------------------------------------------------ tensor checks
int check_view(const st_tensor *t, const char *name, int rank) {
    if (!t) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
    if (t->rank != rank)
        return fail(ST_ERR_INVALID_ARGUMENT,
                    std::string(name) + " must be rank " + std::to_string(rank) + ", got " + std::to_string(t->rank));
    if (dtype_size(t->dtype) == 0) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has an unknown dtype");
    for (int i = 0; i < rank; ++i) {
        if (t->shape[i] < 0) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative extent");
        if (t->strides[i] < 0) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride");
    }
    bool empty = false;
    for (int i = 0; i < rank; ++i) empty |= t->shape[i] == 0;
    if (!empty && !t->data) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a null data pointer");
    return ST_OK;
}

int64_t view_span(const st_tensor &t) {  // elements from base to last element + 1
    int64_t span = 1;
    for (int i = 0; i < t.rank; ++i) {
        if (t.shape[i] == 0) return 0;
        span += (t.shape[i] - 1) * t.strides[i];
    }
    return span;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ------------------------------------------------------------ vector add
int vector_add_views(const ExecCtx &x, const st_tensor &a, const st_tensor &b, const st_tensor &c, int64_t rows,
                     int64_t cols) {
    if (c.rank == 1)
        return launch_vector_add_1d(static_cast<const float *>(a.data), a.strides[0],
                                    static_cast<const float *>(b.data), b.strides[0], static_cast<float *>(c.data),
                                    c.strides[0], cols, x.dev->sm_count, x.stream);
    return launch_vector_add_2d(static_cast<const float *>(a.data), a.strides, static_cast<const float *>(b.data),
                                b.strides, static_cast<float *>(c.data), c.strides, rows, cols, x.dev->sm_count,
                                x.stream);
}

int check_vector_add(const st_tensor *a, const st_tensor *b, const st_tensor *c) {
    if (!a || !b || !c) return fail(ST_ERR_INVALID_ARGUMENT, "vector_add: null tensor");
    const int rank = c->rank;
    if (rank != 1 && rank != 2) return fail(ST_ERR_INVALID_ARGUMENT, "vector_add: tensors must be rank 1 or 2");
    ST_TRY(check_view(a, "A", rank));
    ST_TRY(check_view(b, "B", rank));
    ST_TRY(check_view(c, "C", rank));
    for (const st_tensor *t : {a, b, c})
        if (t->dtype != ST_F32)
            return fail(ST_ERR_INVALID_ARGUMENT, "vector_add: the lowering is f32-only; tensors must be ST_F32");
    for (int i = 0; i < rank; ++i)
        if (a->shape[i] != c->shape[i] || b->shape[i] != c->shape[i])
            return fail(ST_ERR_INVALID_ARGUMENT, "vector_add: A, B and C must have the same shape");
    return ST_OK;
}

// ------------------------------------------------------------ matmul
int check_matmul(const st_tensor *a, const st_tensor *b, const st_tensor *bias, const st_tensor *c) {
    ST_TRY(check_view(a, "A", 2));
    ST_TRY(check_view(b, "B", 2));
    ST_TRY(check_view(c, "C", 2));
    if (a->shape[1] != b->shape[0])
        return fail(ST_ERR_INVALID_ARGUMENT, "Incompatible matrices: K dimension of A (" + std::to_string(a->shape[1]) +
                                                 ") must match K dimension of B (" + std::to_string(b->shape[0]) + ")");
    if (c->shape[0] != a->shape[0] || c->shape[1] != b->shape[1])
        return fail(ST_ERR_INVALID_ARGUMENT, "C must be [M, N] = [" + std::to_string(a->shape[0]) + ", " +
                                                 std::to_string(b->shape[1]) + "]");
    if (a->dtype != b->dtype) return fail(ST_ERR_INVALID_ARGUMENT, "A and B must have the same dtype");
    if (a->dtype != ST_F32 && a->dtype != ST_F16 && a->dtype != ST_BF16)
        return fail(ST_ERR_INVALID_ARGUMENT, "A and B must be ST_F32, ST_F16 or ST_BF16");
    if (c->dtype != ST_F32 && c->dtype != ST_F16 && c->dtype != ST_BF16)
        return fail(ST_ERR_INVALID_ARGUMENT, "C must be ST_F32, ST_F16 or ST_BF16");
    if (c->shape[0] > 0 && c->shape[1] > 1 && c->strides[1] != 1)
        return fail(ST_ERR_UNSUPPORTED, "C must have unit column stride");
    if (a->shape[0] > INT32_MAX || b->shape[1] > INT32_MAX || a->shape[1] > INT32_MAX)
        return fail(ST_ERR_UNSUPPORTED, "matmul extents must fit in int32 (cuda_tile index type)");
    if (bias) {
        ST_TRY(check_view(bias, "bias", 1));
        if (bias->shape[0] != b->shape[1]) return fail(ST_ERR_INVALID_ARGUMENT, "bias must have N elements");
        if (bias->dtype != ST_F32 && bias->dtype != a->dtype)
            return fail(ST_ERR_INVALID_ARGUMENT, "bias must be ST_F32 or the input dtype");
        if (bias->shape[0] > 1 && bias->strides[0] != 1)
            return fail(ST_ERR_UNSUPPORTED, "bias must be contiguous");
    }
    return ST_OK;
}

__global__ void fill_rows_kernel(void *c, int64_t ldc, int c_dtype, const void *bias, int bias_dtype, int64_t m,
                                 int64_t n) {
    pdl_wait();
    const int64_t total = m * n;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
         i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
        const int64_t r = i / n, q = i - r * n;
        float v = 0.0f;
        if (bias) {
            if (bias_dtype == ST_F32) v = static_cast<const float *>(bias)[q];
            else if (bias_dtype == ST_F16) v = __half2float(static_cast<const __half *>(bias)[q]);
            else v = __bfloat162float(static_cast<const __nv_bfloat16 *>(bias)[q]);
            v = 0.0f + v;
        }
        if (c_dtype == ST_F32) static_cast<float *>(c)[r * ldc + q] = v;
        else if (c_dtype == ST_F16) static_cast<__half *>(c)[r * ldc + q] = __float2half_rn(v);
        else static_cast<__nv_bfloat16 *>(c)[r * ldc + q] = __float2bfloat16_rn(v);
    }
    pdl_trigger();
}

int matmul_device(const ExecCtx &x, const st_tensor &a, const st_tensor &b, const st_tensor *bias,
                  const st_tensor &c, const PeerOutputs *peers = nullptr, bool c_padding = false) {
    const int64_t M = a.shape[0], K = a.shape[1], N = b.shape[1];
    if (M == 0 || N == 0) return ST_OK;
    const void *bias_ptr = bias ? bias->data : nullptr;
    const int bias_dtype = bias ? bias->dtype : ST_F32;
    if (K == 0) {  // empty contraction: C = 0 (+ bias)
        if (peers && peers->n > 0) return fail(ST_ERR_UNSUPPORTED, "K = 0 with peer outputs");
        ST_CUDA_TRY(launch_kernel(fill_rows_kernel, 148, 256, 0, x.stream, c.data, c.strides[0], c.dtype, bias_ptr,
                                  bias_dtype, M, N));
        note_launch();
        const cudaError_t e = cudaPeekAtLastError();
        return e == cudaSuccess ? ST_OK : cuda_fail(cudaGetLastError(), "fill_rows_kernel");
    }
    GemmArgs g{};
    if (peers) g.peers = *peers;
    g.deterministic = (x.flags & ST_EXEC_DETERMINISTIC) != 0;
    g.c_padding = c_padding;
    g.c = c.data;
    g.ldc = c.strides[0];
    g.c_dtype = c.dtype;
    g.bias = bias_ptr;
    g.bias_dtype = bias_dtype;
    g.m = M;
    g.n = N;
    Workspace &ws = x.dev->scratch;
    if (a.dtype == ST_F32) {
        // Opt-in (SPTILES_B200_FP32_FUSED=1): split into tf32 hi/lo inside the
        // GEMM.  Its 128 x 64 tiles are bound by shared-memory bandwidth, so the
        // packed route below -- which can use the 256 x 256 CTA-pair kernel --
        // is faster from 2048^3 up (218 vs 61 TFLOP/s at 4096^3) and ties at 1024^3.
        const bool a_ok = (a.strides[1] == 1 || K == 1) && (a.strides[0] * 4) % 16 == 0 && aligned16(a.data);
        const bool b_rows_ok = (b.strides[1] == 1 || N == 1) && (b.strides[0] * 4) % 16 == 0 && aligned16(b.data);
        const bool b_cols_ok = (b.strides[0] == 1 || K == 1) && (b.strides[1] * 4) % 16 == 0 && aligned16(b.data);
        const char *fused = std::getenv("SPTILES_B200_FP32_FUSED");
        if (fused && fused[0] == '1' && a_ok && (b_rows_ok || b_cols_ok)) {
            g.ab_dtype = ST_F32;
            g.a = a.data;
            g.lda = a.strides[0];
            g.b = b.data;
            g.b_k_major = !b_rows_ok;
            g.ldb = b_rows_ok ? b.strides[0] : b.strides[1];
            g.k = K;
            return launch_gemm_3xtf32(g, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream);
        }
        // Opt-in (SPTILES_B200_FP32=split): operands TMA can address in place, on
        // a CTA-pair plan, are split into tf32 hi / lo by the pair kernel itself,
        // with no packing pass.  Its converter traffic makes it shared-memory
        // bound (~70 % of the MMA rate): it ties with packing at 1024^3 and
        // loses from 2048^3 up (750 vs 578 us at 4096^3), so packing is the default.
        const char *route = std::getenv("SPTILES_B200_FP32");
        if (route && std::strcmp(route, "split") == 0 && a_ok && (b_rows_ok || b_cols_ok)) {
            GemmArgs gs = g;
            gs.ab_dtype = ST_F32;
            gs.a = a.data;
            gs.lda = a.strides[0];
            gs.b = b.data;
            gs.b_k_major = !b_rows_ok;
            gs.ldb = b_rows_ok ? b.strides[0] : b.strides[1];
            gs.k = K;
            gs.split_fp32 = true;
            if (gemm_split_fp32_fits(gs, x.dev->sm_count)) {
                if (gemm_uses_stream_k(gs, x.dev->sm_count)) ST_TRY(sk_acquire(x.dev, x.stream, gs));
                ST_TRY(launch_gemm(gs, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
                if (gs.sk_ws) ST_TRY(ws_release(x.dev->sk, x.stream));
                return ST_OK;
            }
        }
        // otherwise pack [hi|hi|lo] x [hi;lo;hi] into scratch and run one tf32 GEMM
        const int64_t kp = tf32_packed_k(K);
        const size_t need = static_cast<size_t>(M + N) * 3 * kp * sizeof(float);
        void *base = nullptr;
        ST_TRY(ws_acquire(ws, need, x.stream, &base));
        float *ap = static_cast<float *>(base);
        float *bp = ap + M * 3 * kp;
        g.ab_dtype = ST_F32;
        g.a = ap;
        g.lda = 3 * kp;
        g.b = bp;
        g.ldb = 3 * kp;
        g.b_k_major = true;
        g.k = 3 * kp;
        // split tiles that fold in L2 onto a preset C start from C = bias,
        // which the pack writes; the ordered fold and the exchange use the
        // stream-K workspace (an ordered launch captured before the workspace
        // exists presets C by its own kernel instead)
        if (gemm_uses_stream_k(g, x.dev->sm_count)) ST_TRY(sk_acquire(x.dev, x.stream, g));
        CPreset preset;
        if (stream_k_l2add_mode(g, x.dev->sm_count) == 1) {
            preset.c = static_cast<float *>(c.data);
            preset.ldc = c.strides[0];
            preset.bias = bias_ptr;
            preset.bias_dtype = bias_dtype;
            preset.m = static_cast<int>(M);
            preset.n = static_cast<int>(N);
            g.c_preset = true;
        }
        ST_TRY(launch_pack_ab_tf32(static_cast<const float *>(a.data), a.strides[0], a.strides[1], M,
                                   static_cast<const float *>(b.data), b.strides[0], b.strides[1], N, K, ap, bp, kp,
                                   g.c_preset ? &preset : nullptr, x.stream));
        ST_TRY(launch_gemm(g, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
        if (g.sk_ws) ST_TRY(ws_release(x.dev->sk, x.stream));
        return ws_release(ws, x.stream);
    }
    // 16-bit operands: use them in place when TMA can address them
    g.ab_dtype = a.dtype;
    g.k = K;
    const bool a_ok = (a.strides[1] == 1 || K == 1) && (a.strides[0] * 2) % 16 == 0 && aligned16(a.data);
    const bool b_rows_ok = (b.strides[1] == 1 || N == 1) && (b.strides[0] * 2) % 16 == 0 && aligned16(b.data);
    const bool b_cols_ok = (b.strides[0] == 1 || K == 1) && (b.strides[1] * 2) % 16 == 0 && aligned16(b.data);
    size_t need = 0;
    const int64_t lda_p = cdiv(K, 8) * 8, ldb_p = cdiv(N, 8) * 8;
    if (!a_ok) need += static_cast<size_t>(M) * lda_p * 2;
    if (!b_rows_ok && !b_cols_ok) need += static_cast<size_t>(K) * ldb_p * 2;
    void *base = nullptr;
    if (need) ST_TRY(ws_acquire(ws, need + 32, x.stream, &base));
    uint8_t *cursor = static_cast<uint8_t *>(base);
    if (a_ok) {
        g.a = a.data;
        g.lda = a.strides[0];
    } else {
        uint16_t *ap = reinterpret_cast<uint16_t *>(cursor);
        ST_TRY(launch_repack_16(static_cast<const uint16_t *>(a.data), a.strides[0], a.strides[1], M, K, ap, lda_p,
                                x.stream));
        cursor += (static_cast<size_t>(M) * lda_p * 2 + 15) & ~size_t(15);
        g.a = ap;
        g.lda = lda_p;
    }
    if (b_rows_ok) {
        g.b = b.data;
        g.ldb = b.strides[0];
        g.b_k_major = false;
    } else if (b_cols_ok) {  // B stored column-major, i.e. as B^T [N, K] with K contiguous
        g.b = b.data;
        g.ldb = b.strides[1];
        g.b_k_major = true;
    } else {
        uint16_t *bpk = reinterpret_cast<uint16_t *>(cursor);
        ST_TRY(launch_repack_16(static_cast<const uint16_t *>(b.data), b.strides[0], b.strides[1], K, N, bpk, ldb_p,
                                x.stream));
        g.b = bpk;
        g.ldb = ldb_p;
        g.b_k_major = false;
    }
    if (gemm_uses_stream_k(g, x.dev->sm_count)) ST_TRY(sk_acquire(x.dev, x.stream, g));
    ST_TRY(launch_gemm(g, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
    if (g.sk_ws) ST_TRY(ws_release(x.dev->sk, x.stream));
    if (need) return ws_release(ws, x.stream);
    return ST_OK;
}

int finish(const ExecCtx &x) {
    if (x.flags & ST_EXEC_SYNC) return bounded_sync(x.dev, x.stream, x.timeout_ms);
    return ST_OK;
}

// ------------------------------------------------------------ host staging
// Copy a host tensor into a dense device tensor carved from `cursor`.
int stage_in(const ExecCtx &x, const st_tensor &h, uint8_t *&cursor, st_tensor *d) {
    *d = h;
    const size_t es = dtype_size(h.dtype);
    d->data = cursor;
    if (h.rank == 1) {
        d->strides[0] = 1;
        const size_t bytes = static_cast<size_t>(h.shape[0]) * es;
        if (h.shape[0] > 1 && h.strides[0] != 1) return fail(ST_ERR_UNSUPPORTED, "host tensors must be contiguous");
        if (bytes) ST_CUDA_TRY(cudaMemcpyAsync(cursor, h.data, bytes, cudaMemcpyHostToDevice, x.stream));
        cursor += (bytes + 255) & ~size_t(255);
        return ST_OK;
    }
    const int64_t rows = h.shape[0], cols = h.shape[1];
    d->strides[0] = cols;
    d->strides[1] = 1;
    if (rows && cols) {
        if (cols > 1 && h.strides[1] != 1) return fail(ST_ERR_UNSUPPORTED, "host tensors must have unit column stride");
        const int64_t hs0 = rows > 1 ? h.strides[0] : cols;
        ST_CUDA_TRY(cudaMemcpy2DAsync(cursor, cols * es, h.data, hs0 * es, cols * es, rows, cudaMemcpyHostToDevice,
                                      x.stream));
    }
    cursor += (static_cast<size_t>(rows * cols) * es + 255) & ~size_t(255);
    return ST_OK;
}

int stage_out(const ExecCtx &x, const st_tensor &d, const st_tensor &h) {
    const size_t es = dtype_size(h.dtype);
    if (h.rank == 1) {
        if (h.shape[0] > 1 && h.strides[0] != 1) return fail(ST_ERR_UNSUPPORTED, "host tensors must be contiguous");
        if (h.shape[0])
            ST_CUDA_TRY(cudaMemcpyAsync(h.data, d.data, h.shape[0] * es, cudaMemcpyDeviceToHost, x.stream));
        return ST_OK;
    }
    const int64_t rows = h.shape[0], cols = h.shape[1];
    if (!rows || !cols) return ST_OK;
    if (cols > 1 && h.strides[1] != 1) return fail(ST_ERR_UNSUPPORTED, "host tensors must have unit column stride");
    const int64_t hs0 = rows > 1 ? h.strides[0] : cols;
    ST_CUDA_TRY(cudaMemcpy2DAsync(h.data, hs0 * es, d.data, d.strides[0] * es, cols * es, rows,
                                  cudaMemcpyDeviceToHost, x.stream));
    return ST_OK;
}

size_t staged_bytes(const st_tensor &t) {
    size_t n = dtype_size(t.dtype);
    for (int i = 0; i < t.rank; ++i) n *= static_cast<size_t>(t.shape[i]);
    return (n + 255) & ~size_t(255);
}

// ------------------------------------------------------------ pipelined host calls
// Event `i` of the device's pool (created on first use, reused afterwards).
int pool_event(DeviceState *d, size_t i, cudaEvent_t *out) {
    while (d->events.size() <= i) {
        cudaEvent_t e;
        ST_CUDA_TRY(cudaEventCreateWithFlags(&e, cudaEventDisableTiming));
        d->events.push_back(e);
    }
    *out = d->events[i];
    return ST_OK;
}

int ensure_copy_streams(DeviceState *d) {
    if (!d->copy_in) ST_CUDA_TRY(cudaStreamCreateWithFlags(&d->copy_in, cudaStreamNonBlocking));
    if (!d->copy_out) ST_CUDA_TRY(cudaStreamCreateWithFlags(&d->copy_out, cudaStreamNonBlocking));
    return ST_OK;
}

// `waiter` waits for everything issued so far on `signaller`.
int stream_after(DeviceState *d, size_t &ev_i, cudaStream_t waiter, cudaStream_t signaller) {
    cudaEvent_t e;
    ST_TRY(pool_event(d, ev_i++, &e));
    ST_CUDA_TRY(cudaEventRecord(e, signaller));
    ST_CUDA_TRY(cudaStreamWaitEvent(waiter, e, 0));
    return ST_OK;
}

bool host_rows_dense(const st_tensor &t) {  // unit column stride (rows may be padded)
    if (t.rank == 1) return t.shape[0] <= 1 || t.strides[0] == 1;
    return t.shape[1] <= 1 || t.strides[1] == 1;
}

// Block [r0, r1) x [c0, c1) of a rank-2 host tensor <-> the same block of a
// device matrix with row pitch `ld` elements.
int copy_block_in(cudaStream_t s, void *dev, int64_t ld, const st_tensor &h, int64_t r0, int64_t r1, int64_t c0,
                  int64_t c1) {
    const size_t es = dtype_size(h.dtype);
    if (r1 <= r0 || c1 <= c0) return ST_OK;
    const int64_t hs0 = h.shape[0] > 1 ? h.strides[0] : h.shape[1];
    const uint8_t *src = static_cast<const uint8_t *>(h.data) + static_cast<size_t>(r0 * hs0 + c0) * es;
    uint8_t *dst = static_cast<uint8_t *>(dev) + static_cast<size_t>(r0 * ld + c0) * es;
    ST_CUDA_TRY(cudaMemcpy2DAsync(dst, ld * es, src, hs0 * es, (c1 - c0) * es, r1 - r0, cudaMemcpyHostToDevice, s));
    return ST_OK;
}

int copy_block_out(cudaStream_t s, const st_tensor &h, const void *dev, int64_t ld, int64_t r0, int64_t r1,
                   int64_t c0, int64_t c1) {
    const size_t es = dtype_size(h.dtype);
    if (r1 <= r0 || c1 <= c0) return ST_OK;
    const int64_t hs0 = h.shape[0] > 1 ? h.strides[0] : h.shape[1];
    uint8_t *dst = static_cast<uint8_t *>(h.data) + static_cast<size_t>(r0 * hs0 + c0) * es;
    const uint8_t *src = static_cast<const uint8_t *>(dev) + static_cast<size_t>(r0 * ld + c0) * es;
    ST_CUDA_TRY(cudaMemcpy2DAsync(dst, hs0 * es, src, ld * es, (c1 - c0) * es, r1 - r0, cudaMemcpyDeviceToHost, s));
    return ST_OK;
}

// C = A @ B (+ bias) on host tensors with 16-bit A and B.  C[i, j] needs row
// i of A and column j of B, so the received rows of A and columns of B grow
// together: step s brings row block s of A and column block s of B (~16 MB
// each) on copy_in, then computes on the caller's stream
//   C[new rows, all columns so far]  and  C[earlier rows, new columns]
// and sends those blocks of C back on copy_out.  With A and B arriving in
// step, C comes out from the first ~2 blocks on and both PCIe directions
// stay busy (with B first, nothing leaves until all of B is in).  Device
// copies use row pitches rounded up to 8 elements, so every block view is a
// 16-byte-aligned TMA operand.
int matmul_host_pipelined(const ExecCtx &x, const st_tensor &a, const st_tensor &b, const st_tensor *bias,
                          const st_tensor &c, bool wait) {
    DeviceState *d = x.dev;
    ST_TRY(ensure_copy_streams(d));
    const int64_t M = a.shape[0], K = a.shape[1], N = b.shape[1];
    const size_t ein = dtype_size(a.dtype), eout = dtype_size(c.dtype);
    const int64_t lda = cdiv(K, 8) * 8, ldb = cdiv(N, 8) * 8, ldc = cdiv(N, 8) * 8;
    const size_t a_bytes = static_cast<size_t>(M * lda) * ein, b_bytes = static_cast<size_t>(K * ldb) * ein;
    const size_t c_bytes = static_cast<size_t>(M * ldc) * eout;
    const size_t bias_bytes = bias ? static_cast<size_t>(N) * dtype_size(bias->dtype) : 0;
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    void *base = nullptr;
    ST_TRY(ws_acquire(d->stage, up(a_bytes) + up(b_bytes) + up(c_bytes) + up(bias_bytes), x.stream, &base));
    uint8_t *da = static_cast<uint8_t *>(base);
    uint8_t *db = da + up(a_bytes);
    uint8_t *dc = db + up(b_bytes);
    uint8_t *dbias = dc + up(c_bytes);
    size_t ev = 0;
    // the copies start after earlier work on the caller's stream (workspace reuse)
    ST_TRY(stream_after(d, ev, d->copy_in, x.stream));
    ST_TRY(stream_after(d, ev, d->copy_out, x.stream));
    if (bias) ST_CUDA_TRY(cudaMemcpyAsync(dbias, bias->data, bias_bytes, cudaMemcpyHostToDevice, d->copy_in));
    // ~16 MB blocks in whole 256-row / 256-column tiles (measured on B200 at
    // 8192^3: wider column blocks or taller row blocks were 2-4 % slower)
    const int64_t per = static_cast<int64_t>((size_t(16) << 20) / std::max<size_t>(1, static_cast<size_t>(K) * ein));
    const int64_t rows = std::max<int64_t>(256, (per / 256) * 256), cols = rows;
    const int64_t steps = std::max(cdiv(M, rows), cdiv(N, cols));
    auto view = [](const st_tensor &like, void *data, int64_t r, int64_t q, int64_t ld) {
        st_tensor v = like;
        v.data = data;
        v.rank = 2;
        v.shape[0] = r;
        v.shape[1] = q;
        v.strides[0] = ld;
        v.strides[1] = 1;
        return v;
    };
    auto gemm = [&](int64_t r0, int64_t r1, int64_t c0, int64_t c1) -> int {
        if (r1 <= r0 || c1 <= c0) return ST_OK;
        const st_tensor va = view(a, da + static_cast<size_t>(r0 * lda) * ein, r1 - r0, K, lda);
        const st_tensor vb = view(b, db + static_cast<size_t>(c0) * ein, K, c1 - c0, ldb);
        const st_tensor vc = view(c, dc + static_cast<size_t>(r0 * ldc + c0) * eout, r1 - r0, c1 - c0, ldc);
        st_tensor vbias;
        if (bias) {
            vbias = *bias;
            vbias.data = dbias + static_cast<size_t>(c0) * dtype_size(bias->dtype);
            vbias.shape[0] = c1 - c0;
            vbias.strides[0] = 1;
        }
        // the last column block ends in the device copy's own padding, the others on 256 columns
        return matmul_device(x, va, vb, bias ? &vbias : nullptr, vc, nullptr, true);
    };
    for (int64_t st = 0; st < steps; ++st) {
        const int64_t r0 = std::min(M, st * rows), r1 = std::min(M, (st + 1) * rows);
        const int64_t c0 = std::min(N, st * cols), c1 = std::min(N, (st + 1) * cols);
        ST_TRY(copy_block_in(d->copy_in, da, lda, a, r0, r1, 0, K));
        ST_TRY(copy_block_in(d->copy_in, db, ldb, b, 0, K, c0, c1));
        ST_TRY(stream_after(d, ev, x.stream, d->copy_in));
        ST_TRY(gemm(r0, r1, 0, c1));  // new rows x every column so far
        ST_TRY(gemm(0, r0, c0, c1));  // earlier rows x the new columns
        ST_TRY(stream_after(d, ev, d->copy_out, x.stream));
        ST_TRY(copy_block_out(d->copy_out, c, dc, ldc, r0, r1, 0, c1));
        ST_TRY(copy_block_out(d->copy_out, c, dc, ldc, 0, r0, c0, c1));
    }
    ST_TRY(stream_after(d, ev, x.stream, d->copy_out));
    ST_TRY(ws_release(d->stage, x.stream));
    return wait ? bounded_sync(d, x.stream, x.timeout_ms) : ST_OK;
}

// C = A + B on dense host arrays, in element chunks over the three streams.
int vector_add_host_pipelined(const ExecCtx &x, const st_tensor &a, const st_tensor &b, const st_tensor &c,
                              int64_t n, bool wait) {
    DeviceState *d = x.dev;
    ST_TRY(ensure_copy_streams(d));
    const size_t bytes = static_cast<size_t>(n) * 4;
    auto up = [](size_t v) { return (v + 255) & ~size_t(255); };
    void *base = nullptr;
    ST_TRY(ws_acquire(d->stage, 3 * up(bytes), x.stream, &base));
    float *da = static_cast<float *>(base);
    float *db = reinterpret_cast<float *>(static_cast<uint8_t *>(base) + up(bytes));
    float *dc = reinterpret_cast<float *>(static_cast<uint8_t *>(base) + 2 * up(bytes));
    const float *ha = static_cast<const float *>(a.data), *hb = static_cast<const float *>(b.data);
    float *hc = static_cast<float *>(c.data);
    size_t ev = 0;
    ST_TRY(stream_after(d, ev, d->copy_in, x.stream));
    ST_TRY(stream_after(d, ev, d->copy_out, x.stream));
    const int64_t chunk = int64_t(4) << 20;  // 16 MB of each array per chunk
    for (int64_t e0 = 0; e0 < n; e0 += chunk) {
        const int64_t len = std::min(chunk, n - e0);
        ST_CUDA_TRY(cudaMemcpyAsync(da + e0, ha + e0, len * 4, cudaMemcpyHostToDevice, d->copy_in));
        ST_CUDA_TRY(cudaMemcpyAsync(db + e0, hb + e0, len * 4, cudaMemcpyHostToDevice, d->copy_in));
        ST_TRY(stream_after(d, ev, x.stream, d->copy_in));
        ST_TRY(launch_vector_add_1d(da + e0, 1, db + e0, 1, dc + e0, 1, len, d->sm_count, x.stream));
        ST_TRY(stream_after(d, ev, d->copy_out, x.stream));
        ST_CUDA_TRY(cudaMemcpyAsync(hc + e0, dc + e0, len * 4, cudaMemcpyDeviceToHost, d->copy_out));
    }
    ST_TRY(stream_after(d, ev, x.stream, d->copy_out));
    ST_TRY(ws_release(d->stage, x.stream));
    return wait ? bounded_sync(d, x.stream, x.timeout_ms) : ST_OK;
}

// ------------------------------------------------------------ host-memory calls on one device
// Dense arrays of one layout: the add runs over one flat range.
bool vector_add_host_flat(const st_tensor &a, const st_tensor &b, const st_tensor &c) {
    bool flat = true;
    for (const st_tensor *t : {&a, &b, &c}) {
        if (t->rank == 1) flat &= t->shape[0] <= 1 || t->strides[0] == 1;
        else flat &= (t->shape[1] <= 1 || t->strides[1] == 1) && (t->shape[0] <= 1 || t->strides[0] == t->shape[1]);
    }
    return flat;
}

// C = A + B on host memory through the device of `x`; waits (bounded) when `wait`.
int vector_add_host_one(const ExecCtx &x, const st_tensor &a, const st_tensor &b, const st_tensor &c, bool wait) {
    int64_t n = 1;
    for (int i = 0; i < c.rank; ++i) n *= c.shape[i];
    if (vector_add_host_flat(a, b, c) && n > 0) return vector_add_host_pipelined(x, a, b, c, n, wait);
    void *base = nullptr;
    ST_TRY(ws_acquire(x.dev->stage, staged_bytes(a) + staged_bytes(b) + staged_bytes(c), x.stream, &base));
    uint8_t *cursor = static_cast<uint8_t *>(base);
    st_tensor da, db, dc;
    ST_TRY(stage_in(x, a, cursor, &da));
    ST_TRY(stage_in(x, b, cursor, &db));
    dc = c;
    dc.data = cursor;
    if (c.rank == 1) dc.strides[0] = 1;
    else {
        dc.strides[0] = c.shape[1];
        dc.strides[1] = 1;
    }
    const int64_t rows = c.rank == 2 ? c.shape[0] : 1;
    const int64_t cols = c.rank == 2 ? c.shape[1] : c.shape[0];
    ST_TRY(vector_add_views(x, da, db, dc, rows, cols));
    ST_TRY(stage_out(x, dc, c));
    ST_TRY(ws_release(x.dev->stage, x.stream));
    return wait ? bounded_sync(x.dev, x.stream, x.timeout_ms) : ST_OK;
}

// C = A @ B (+ bias) on host memory through the device of `x`; waits (bounded) when `wait`.
int matmul_host_one(const ExecCtx &x, const st_tensor &a, const st_tensor &b, const st_tensor *bias,
                    const st_tensor &c, bool wait) {
    // 16-bit operands with unit column strides: chunked and overlapped (the
    // fp32 path packs B once per call, so it stays unchunked)
    if (a.dtype != ST_F32 && a.shape[0] > 0 && b.shape[1] > 0 && a.shape[1] > 0 && host_rows_dense(a) &&
        host_rows_dense(b) && host_rows_dense(c))
        return matmul_host_pipelined(x, a, b, bias, c, wait);
    size_t need = staged_bytes(a) + staged_bytes(b) + staged_bytes(c) + (bias ? staged_bytes(*bias) : 0);
    void *base = nullptr;
    ST_TRY(ws_acquire(x.dev->stage, need, x.stream, &base));
    uint8_t *cursor = static_cast<uint8_t *>(base);
    st_tensor da, db, dbias, dc;
    ST_TRY(stage_in(x, a, cursor, &da));
    ST_TRY(stage_in(x, b, cursor, &db));
    if (bias) ST_TRY(stage_in(x, *bias, cursor, &dbias));
    dc = c;
    dc.data = cursor;
    dc.strides[0] = c.shape[1];
    dc.strides[1] = 1;
    ST_TRY(matmul_device(x, da, db, bias ? &dbias : nullptr, dc));
    ST_TRY(stage_out(x, dc, c));
    ST_TRY(ws_release(x.dev->stage, x.stream));
    return wait ? bounded_sync(x.dev, x.stream, x.timeout_ms) : ST_OK;
}

// ------------------------------------------------------------ single-box partitioner (one process)
// ST_EXEC_ALL_DEVICES: each device runs on its own stream of the context.
int check_all_devices(const st_exec *exec) {
    if (exec->stream != nullptr)
        return fail(ST_ERR_INVALID_ARGUMENT,
                    "ST_EXEC_ALL_DEVICES runs every device on the context's own stream: exec->stream must be NULL");
    if (exec->device >= 0)
        return fail(ST_ERR_INVALID_ARGUMENT, "ST_EXEC_ALL_DEVICES uses every device: exec->device must be -1");
    return ST_OK;
}

// Rows [r0, r1) of a host view (elements, for rank 1).
st_tensor host_rows(const st_tensor &t, int64_t r0, int64_t r1) {
    st_tensor v = t;
    v.data = static_cast<uint8_t *>(t.data) + static_cast<size_t>(r0 * t.strides[0]) * dtype_size(t.dtype);
    v.shape[0] = r1 - r0;
    return v;
}

// Elements [e0, e1) of a dense host array, as a rank-1 view.
st_tensor flat_range(const st_tensor &t, int64_t e0, int64_t e1) {
    st_tensor v = t;
    v.data = static_cast<uint8_t *>(t.data) + static_cast<size_t>(e0) * dtype_size(t.dtype);
    v.rank = 1;
    v.shape[0] = e1 - e0;
    v.strides[0] = 1;
    v.shape[1] = 0;
    v.strides[1] = 0;
    return v;
}

// Split [0, total) into one contiguous range per device of the context
// (boundaries on multiples of `align`, as st_shard_range), enqueue each
// range's work on its device, then wait (bounded) for every device that got
// work -- also after a failure, so that nothing is left in flight.
template <typename Enqueue>
int for_each_device_shard(st_ctx *ctx, const ExecCtx &x0, int64_t total, int64_t align, Enqueue enqueue) {
    const int g_count = static_cast<int>(ctx->devs.size());
    const int64_t units = cdiv(total, align);
    std::vector<ExecCtx> busy;
    int rc = ST_OK;
    for (int g = 0; g < g_count && rc == ST_OK; ++g) {
        const int64_t b = std::min(units * g / g_count * align, total);
        const int64_t e = std::min(units * (g + 1) / g_count * align, total);
        if (e <= b) continue;
        ExecCtx xg = x0;
        xg.dev = &ctx->devs[g];
        xg.stream = xg.dev->stream;
        DeviceGuard guard(xg.dev->ordinal);
        rc = enqueue(xg, b, e);
        busy.push_back(xg);
    }
    for (const ExecCtx &xg : busy) {
        DeviceGuard guard(xg.dev->ordinal);
        const int r = bounded_sync(xg.dev, xg.stream, xg.timeout_ms);
        if (rc == ST_OK) rc = r;
    }
    return rc;
}

// C = A + B on host memory over every device of the context: element
// ranges on 16-byte boundaries for dense arrays, rows otherwise.
int vector_add_host_split(st_ctx *ctx, const ExecCtx &x, const st_tensor &a, const st_tensor &b,
                          const st_tensor &c) {
    if (vector_add_host_flat(a, b, c)) {
        int64_t n = 1;
        for (int i = 0; i < c.rank; ++i) n *= c.shape[i];
        return for_each_device_shard(ctx, x, n, 4, [&](const ExecCtx &xg, int64_t e0, int64_t e1) {
            return vector_add_host_one(xg, flat_range(a, e0, e1), flat_range(b, e0, e1), flat_range(c, e0, e1),
                                       false);
        });
    }
    return for_each_device_shard(ctx, x, c.shape[0], 1, [&](const ExecCtx &xg, int64_t r0, int64_t r1) {
        return vector_add_host_one(xg, host_rows(a, r0, r1), host_rows(b, r0, r1), host_rows(c, r0, r1), false);
    });
}

// C = A @ B (+ bias) on host memory over every device of the context: 128-row
// blocks of A and C per device, all of B and the bias to each.
int matmul_host_split(st_ctx *ctx, const ExecCtx &x, const st_tensor &a, const st_tensor &b, const st_tensor *bias,
                      const st_tensor &c) {
    return for_each_device_shard(ctx, x, a.shape[0], 128, [&](const ExecCtx &xg, int64_t r0, int64_t r1) {
        return matmul_host_one(xg, host_rows(a, r0, r1), b, bias, host_rows(c, r0, r1), false);
    });
}

// ------------------------------------------------------------ 8-bit blocks and norms
constexpr int64_t kScaleBlock = 128;

int check_matrix(const st_tensor *t, const char *name) {
    if (!t) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
    if (t->rank != 2)
        return fail(ST_ERR_INVALID_ARGUMENT,
                    std::string(name) + " must be rank 2, got " + std::to_string(t->rank));
    for (int i = 0; i < 2; ++i) {
        if (t->shape[i] < 0) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative extent");
        if (t->strides[i] < 0) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a negative stride");
        if (t->shape[i] > INT32_MAX) return fail(ST_ERR_UNSUPPORTED, std::string(name) + ": extents must fit in int32");
    }
    if (t->shape[0] > 0 && t->shape[1] > 0 && !t->data)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a null data pointer");
    return ST_OK;
}

// An output: no two of its elements may share an address.
int check_output(const st_tensor &t, const char *name) {
    const int64_t a = t.shape[0], b = t.shape[1], sa = t.strides[0], sb = t.strides[1];
    if (a == 0 || b == 0) return ST_OK;
    const bool ok = (a == 1 && b == 1) || (a == 1 && sb >= 1) || (b == 1 && sa >= 1) ||
                    (sb >= 1 && sa >= (b - 1) * sb + 1) || (sa >= 1 && sb >= (a - 1) * sa + 1);
    return ok ? ST_OK : fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has overlapping elements");
}

bool is_fp8(int dtype) { return dtype == ST_E4M3 || dtype == ST_E5M2; }
bool is_float(int dtype) { return dtype == ST_F32 || dtype == ST_F16 || dtype == ST_BF16; }
// element (0, 1) of a row lies next to (0, 0)
bool unit_columns(const st_tensor &t) { return t.shape[1] <= 1 || t.strides[1] == 1; }

int check_fp8_operands(const st_tensor *a, const st_tensor *b) {
    ST_TRY(check_matrix(a, "A"));
    ST_TRY(check_matrix(b, "B"));
    if (!is_fp8(a->dtype) || !is_fp8(b->dtype))
        return fail(ST_ERR_INVALID_ARGUMENT, "matmul_fp8: A and B must be ST_E4M3 or ST_E5M2");
    if (a->shape[1] != b->shape[0])
        return fail(ST_ERR_INVALID_ARGUMENT, "Incompatible matrices: K dimension of A (" + std::to_string(a->shape[1]) +
                                                 ") must match K dimension of B (" + std::to_string(b->shape[0]) + ")");
    return ST_OK;
}

Fp8Operand fp8_operand(const st_tensor &t, bool is_b) {
    Fp8Operand o{};
    o.data = t.data;
    o.rows = t.shape[is_b ? 1 : 0];
    o.k = t.shape[is_b ? 0 : 1];
    o.s_row = t.strides[is_b ? 1 : 0];
    o.s_k = t.strides[is_b ? 0 : 1];
    o.e5m2 = t.dtype == ST_E5M2 ? 1 : 0;
    return o;
}

// Scales of an operand: [rows or their blocks of 128, K blocks] for A, the transpose for B.
int set_scale(const st_tensor *t, const char *name, bool is_b, Fp8Operand *o) {
    ST_TRY(check_matrix(t, name));
    if (t->dtype != ST_F32) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be ST_F32");
    const int ri = is_b ? 1 : 0;
    const int64_t rows = t->shape[ri], blocks = t->shape[1 - ri];
    if (blocks != cdiv(o->k, kScaleBlock) || (rows != o->rows && rows != cdiv(o->rows, kScaleBlock)))
        return fail(ST_ERR_INVALID_ARGUMENT,
                    std::string(name) + " must have one scale for each 128 elements along K (" +
                        std::to_string(cdiv(o->k, kScaleBlock)) + ") and for each " + (is_b ? "column (" : "row (") +
                        std::to_string(o->rows) + ") or 128 of them (" + std::to_string(cdiv(o->rows, kScaleBlock)) +
                        "), got [" + std::to_string(t->shape[0]) + ", " + std::to_string(t->shape[1]) + "]");
    o->scale = t->data;
    o->scale_row = t->strides[ri];
    o->scale_k = t->strides[1 - ri];
    o->scale_shift = rows == o->rows ? 0 : 7;
    return ST_OK;
}

// ---- 4-bit blocks
int check_codes(const st_tensor *t, const char *name) {
    ST_TRY(check_matrix(t, name));
    if (t->dtype != ST_E2M1X2) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be ST_E2M1X2");
    if (t->shape[0] > INT32_MAX / 4 || t->shape[1] > INT32_MAX / 4)
        return fail(ST_ERR_UNSUPPORTED, std::string(name) + ": at most " + std::to_string(INT32_MAX / 4) + " bytes a row or column");
    return ST_OK;
}

// A load or store of an element off its boundary is a fault of the device.
int check_elements(const st_tensor &t, const char *name) {
    const size_t es = dtype_size(t.dtype);
    if (es > 1 && reinterpret_cast<uintptr_t>(t.data) % es != 0)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must start on a boundary of its elements");
    return ST_OK;
}

// The scales of `rows` rows of `bytes` bytes of codes.
int check_fp4_scale(const st_tensor *t, const char *name, int64_t rows, int64_t bytes) {
    if (!t) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " is null");
    if (t->dtype != ST_E4M3 && t->dtype != ST_E8M0)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be ST_E4M3 (blocks of 16) or ST_E8M0 (blocks of 32)");
    const int64_t need = fp4_scale_bytes(rows, cdiv(bytes, t->dtype == ST_E8M0 ? 16 : 8));
    if (t->rank != 1 || t->shape[0] != need || (need > 1 && t->strides[0] != 1))
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be contiguous, with " + std::to_string(need) +
                                                 " scales: [ceil(rows / 128)][ceil(blocks / 4)][32][4][4]");
    if (need > 0 && !t->data) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a null data pointer");
    if (need > 0 && !aligned16(t->data)) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must start on a 16-byte boundary");
    return ST_OK;
}

// One f32 on the device, or null.
int scalar_of(const st_tensor *t, const char *name, float **out) {
    *out = nullptr;
    if (!t) return ST_OK;
    if (t->dtype != ST_F32 || t->rank != 1 || t->shape[0] != 1 || !t->data)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be one ST_F32");
    ST_TRY(check_elements(*t, name));
    *out = static_cast<float *>(t->data);
    return ST_OK;
}

int check_fp4_operands(const st_tensor *a, const st_tensor *b) {
    ST_TRY(check_codes(a, "A"));
    ST_TRY(check_codes(b, "B"));
    if (a->shape[1] != b->shape[0])
        return fail(ST_ERR_INVALID_ARGUMENT, "Incompatible matrices: K dimension of A (" + std::to_string(a->shape[1]) +
                                                 " bytes) must match K dimension of B (" + std::to_string(b->shape[0]) + ")");
    return ST_OK;
}

Fp4Operand fp4_operand(const st_tensor &t, bool is_b) {
    Fp4Operand o{};
    o.data = t.data;
    o.rows = t.shape[is_b ? 1 : 0];
    o.k = t.shape[is_b ? 0 : 1];
    o.s_row = t.strides[is_b ? 1 : 0];
    o.s_k = t.strides[is_b ? 0 : 1];
    return o;
}

int check_workspace(const char *what, int64_t need, const void *workspace, uint64_t bytes, uintptr_t align) {
    if (need <= 0) return ST_OK;
    if (!workspace || bytes < static_cast<uint64_t>(need))
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(what) + " needs a workspace of " + std::to_string(need) + " bytes");
    if (reinterpret_cast<uintptr_t>(workspace) % align != 0)
        return fail(ST_ERR_INVALID_ARGUMENT, "workspace must be " + std::to_string(align) + "-byte aligned");
    return ST_OK;
}

// ---- products by groups of rows
int check_ends(const st_tensor *t) {
    if (!t) return fail(ST_ERR_INVALID_ARGUMENT, "ends is null");
    if (t->dtype != ST_I32 || t->rank != 1) return fail(ST_ERR_INVALID_ARGUMENT, "ends must be rank 1 of ST_I32");
    if (t->shape[0] < 0) return fail(ST_ERR_INVALID_ARGUMENT, "ends has a negative extent");
    if (t->shape[0] > kGroupedMaxGroups)
        return fail(ST_ERR_UNSUPPORTED, "at most " + std::to_string(kGroupedMaxGroups) + " groups, got " + std::to_string(t->shape[0]));
    if (t->shape[0] > 1 && t->strides[0] != 1) return fail(ST_ERR_INVALID_ARGUMENT, "ends must be contiguous");
    if (t->shape[0] > 0 && !t->data) return fail(ST_ERR_INVALID_ARGUMENT, "ends has a null data pointer");
    return check_elements(*t, "ends");
}

// A [rows, k] and, for one group, B [k, n] (weights: B [rows, n]).
int grouped_operands(const char *what, const st_tensor *a, const st_tensor *b, const char *b_name, bool weights, int64_t groups,
                     int64_t b_group_stride, GroupedArgs *g) {
    ST_TRY(check_matrix(a, "A"));
    st_tensor shape_of_b{};
    if (b && !weights && groups == 0) {  // no matrix, but the extents of one
        shape_of_b = *b;
        shape_of_b.data = &shape_of_b;
        b = &shape_of_b;
    }
    ST_TRY(check_matrix(b, b_name));
    if (a->dtype == ST_F32 && b->dtype == ST_F32)
        return fail(ST_ERR_UNSUPPORTED, std::string(what) + ": operands must be ST_F16 or ST_BF16");
    if ((a->dtype != ST_F16 && a->dtype != ST_BF16) || a->dtype != b->dtype)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(what) + ": A and " + b_name + " must both be ST_F16 or both ST_BF16");
    if (weights && a->shape[0] != b->shape[0])
        return fail(ST_ERR_INVALID_ARGUMENT, "A and C must have the same rows, got " + std::to_string(a->shape[0]) + " and " +
                                                 std::to_string(b->shape[0]));
    if (!weights && a->shape[1] != b->shape[0])
        return fail(ST_ERR_INVALID_ARGUMENT, "Incompatible matrices: K dimension of A (" + std::to_string(a->shape[1]) +
                                                 ") must match K dimension of B (" + std::to_string(b->shape[0]) + ")");
    if (b_group_stride < 0) return fail(ST_ERR_INVALID_ARGUMENT, std::string(b_name) + " has a negative group stride");
    for (const int64_t extent : {a->shape[0], a->shape[1], b->shape[1]})  // sums of an extent and a tile's stay in int32
        if (extent > INT32_MAX / 2) return fail(ST_ERR_UNSUPPORTED, std::string(what) + ": extents of at most " + std::to_string(INT32_MAX / 2));
    ST_TRY(check_elements(*a, "A"));
    if (b != &shape_of_b) ST_TRY(check_elements(*b, b_name));
    g->weights = weights;
    g->dtype = a->dtype;
    g->groups = groups;
    g->rows = a->shape[0];
    g->k = a->shape[1];
    g->n = b->shape[1];
    g->a = a->data;
    g->a_s0 = a->strides[0];
    g->a_s1 = a->strides[1];
    g->b = b->data;
    g->b_g = b_group_stride;
    g->b_s0 = b->strides[0];
    g->b_s1 = b->strides[1];
    return ST_OK;
}

int check_grouped_output(const st_tensor *c, const char *name, int64_t rows, int64_t cols) {
    ST_TRY(check_matrix(c, name));
    if (c->shape[0] != rows || c->shape[1] != cols)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be [" + std::to_string(rows) + ", " + std::to_string(cols) + "]");
    if (!is_float(c->dtype)) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be ST_F32, ST_F16 or ST_BF16");
    if (!unit_columns(*c)) return fail(ST_ERR_UNSUPPORTED, std::string(name) + " must have unit column stride");
    ST_TRY(check_elements(*c, name));
    return check_output(*c, name);
}

// A tensor of the norms: [rows, cols] with unit column stride.
int norm_view(const st_tensor *t, const char *name, int64_t rows, int64_t cols, bool output, NormView *out) {
    if (!t) return ST_OK;
    ST_TRY(check_matrix(t, name));
    if (t->shape[0] != rows || t->shape[1] != cols)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must be [" + std::to_string(rows) + ", " +
                                                 std::to_string(cols) + "], got [" + std::to_string(t->shape[0]) + ", " +
                                                 std::to_string(t->shape[1]) + "]");
    if (!unit_columns(*t)) return fail(ST_ERR_UNSUPPORTED, std::string(name) + " must have unit column stride");
    if (output) ST_TRY(check_output(*t, name));
    out->p = rows > 0 ? t->data : const_cast<char *>("");  // present, though without rows
    out->dtype = t->dtype;
    out->ld = t->strides[0];
    return ST_OK;
}

int norm_weight(const st_tensor *t, const char *name, int64_t cols, NormView *out) {
    if (!t) return ST_OK;
    if (t->rank != 1 || t->shape[0] != cols)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " must have one element per column (" +
                                                 std::to_string(cols) + ")");
    if (!t->data) return fail(ST_ERR_INVALID_ARGUMENT, std::string(name) + " has a null data pointer");
    if (cols > 1 && t->strides[0] != 1) return fail(ST_ERR_UNSUPPORTED, std::string(name) + " must be contiguous");
    out->p = t->data;
    out->dtype = t->dtype;
    out->ld = 0;
    return ST_OK;
}

// gate: [cols] or [1, cols] (channel), [rows, 1] (token), [rows, cols] (full)
int norm_gate(const st_tensor *t, int64_t rows, int64_t cols, NormView *out, int *mode) {
    *mode = kGateNone;
    if (!t) return ST_OK;
    if (t->rank == 1) {
        *mode = kGateChannel;
        return norm_weight(t, "gate", cols, out);
    }
    ST_TRY(check_matrix(t, "gate"));
    const int64_t r = t->shape[0], c = t->shape[1];
    if (r == rows && c == cols) *mode = kGateFull;
    else if (r == 1 && c == cols) *mode = kGateChannel;
    else if (r == rows && c == 1) *mode = kGateToken;
    else
        return fail(ST_ERR_INVALID_ARGUMENT, "gate must be [" + std::to_string(cols) + "], [1, " + std::to_string(cols) +
                                                 "], [" + std::to_string(rows) + ", 1] or [" + std::to_string(rows) + ", " +
                                                 std::to_string(cols) + "], got [" + std::to_string(r) + ", " +
                                                 std::to_string(c) + "]");
    if (*mode != kGateToken && !unit_columns(*t)) return fail(ST_ERR_UNSUPPORTED, "gate must have unit column stride");
    out->p = t->data;
    out->dtype = t->dtype;
    out->ld = *mode == kGateChannel ? 0 : t->strides[0];
    return ST_OK;
}

int check_norm_options(const char *what, const st_norm_options *o, int64_t cols) {
    if (!o) return fail(ST_ERR_INVALID_ARGUMENT, std::string(what) + ": null options");
    if (!std::isfinite(o->alpha) || !std::isfinite(o->weight_offset) || !std::isfinite(o->eps) || o->eps < 0.0f)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(what) + ": alpha, weight_offset and eps must be finite, eps >= 0");
    if (cols < 1) return fail(ST_ERR_INVALID_ARGUMENT, std::string(what) + ": rows must have at least one element");
    return ST_OK;
}

// The branch's type T (x, h, their gradients) and the stream's S: S is T or ST_F32.
int check_norm_types(const char *what, int t, int s) {
    if (!is_float(t) || !is_float(s) || (s != t && s != ST_F32))
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(what) + ": tensors must be ST_F32, ST_F16 or ST_BF16, and the "
                                                                 "residual stream of the branch's type or ST_F32");
    return ST_OK;
}

int check_side_types(const char *what, int t, std::initializer_list<std::pair<const NormView *, const char *>> views) {
    for (const auto &v : views)
        if (v.first->p && v.first->dtype != ST_F32 && v.first->dtype != t)
            return fail(ST_ERR_INVALID_ARGUMENT, std::string(what) + ": " + v.second + " must be ST_F32 or of the branch's type");
    return ST_OK;
}

// ------------------------------------------------------------ entry registry
enum class Kind { VectorAdd1D, VectorAdd2D, Matmul, Fma1D, Fma2D, Cast1D, Cast2D };

struct Entry {
    const char *name;
    Kind kind;
    int in_dtype;
    bool bias;
    bool persistent;
    int n_constants;
    int defaults[3];
};

// cuda_tile symbols this backend serves (vecadd.py:39-48 exports
// "vector_add"; matmul.py:287-296 exports "matmul_fp32").
const Entry kEntries[] = {
    {"vector_add", Kind::VectorAdd1D, ST_F32, false, false, 1, {1024, 0, 0}},
    {"vector_add_2d", Kind::VectorAdd2D, ST_F32, false, false, 2, {64, 64, 0}},
    {"matmul_fp32", Kind::Matmul, ST_F32, false, false, 3, {32, 32, 32}},
    {"matmul_f16", Kind::Matmul, ST_F16, false, false, 3, {128, 256, 64}},
    {"matmul_bf16", Kind::Matmul, ST_BF16, false, false, 3, {128, 256, 64}},
    {"matmul_fp32_bias", Kind::Matmul, ST_F32, true, false, 3, {32, 32, 32}},
    {"matmul_f16_bias", Kind::Matmul, ST_F16, true, false, 3, {128, 256, 64}},
    {"matmul_bf16_bias", Kind::Matmul, ST_BF16, true, false, 3, {128, 256, 64}},
    {"persistent_matmul_fp32", Kind::Matmul, ST_F32, false, true, 3, {32, 32, 32}},
    {"persistent_matmul_f16", Kind::Matmul, ST_F16, false, true, 3, {128, 256, 64}},
    {"persistent_matmul_bf16", Kind::Matmul, ST_BF16, false, true, 3, {128, 256, 64}},
    // the other elementwise ops the lowering materialises (tileops.hpp:616-623, 257-258)
    {"vector_fma", Kind::Fma1D, ST_F32, false, false, 1, {1024, 0, 0}},
    {"vector_fma_2d", Kind::Fma2D, ST_F32, false, false, 2, {64, 64, 0}},
    {"cast", Kind::Cast1D, ST_F32, false, false, 1, {1024, 0, 0}},
    {"cast_2d", Kind::Cast2D, ST_F32, false, false, 2, {64, 64, 0}},
};

const Entry *find_entry(const char *name) {
    if (!name) return nullptr;
    for (const Entry &e : kEntries)
        if (std::strcmp(e.name, name) == 0) return &e;
    return nullptr;
}

// Rebuild tensor views from the flattened cutile_python_v1 bindings:
// rank 1 = (data, size, stride); rank 2 = (data, dim0, dim1, stride0, stride1).
int parse_params(const Entry &e, const st_param *params, int n_params, std::vector<st_tensor> *views,
                 std::vector<int> *buffer_index, int consts[3]) {
    std::vector<int> ranks;
    switch (e.kind) {
    case Kind::VectorAdd1D: ranks = {1, 1, 1}; break;
    case Kind::VectorAdd2D: ranks = {2, 2, 2}; break;
    case Kind::Fma1D: ranks = {1, 1, 1, 1}; break;   // A, B, D, C
    case Kind::Fma2D: ranks = {2, 2, 2, 2}; break;
    case Kind::Cast1D: ranks = {1, 1}; break;         // A, C
    case Kind::Cast2D: ranks = {2, 2}; break;
    case Kind::Matmul: ranks = e.bias ? std::vector<int>{2, 2, 2, 1} : std::vector<int>{2, 2, 2}; break;
    }
    const int n_arrays = static_cast<int>(ranks.size());
    int pos = 0;
    for (int i = 0; i < n_arrays; ++i) {
        const int r = ranks[i];
        const int need = 1 + 2 * r;
        if (pos + need > n_params)
            return fail(ST_ERR_INVALID_ARGUMENT, std::string(e.name) + " expects " +
                                                     std::to_string(n_arrays) + " array descriptors (got " +
                                                     std::to_string(n_params) + " params)");
        const st_param &buf = params[pos];
        if (buf.kind != ST_PARAM_BUFFER)
            return fail(ST_ERR_INVALID_ARGUMENT, "param " + std::to_string(pos) + " must be a buffer");
        for (int j = 1; j < need; ++j)
            if (params[pos + j].kind != ST_PARAM_I32)
                return fail(ST_ERR_INVALID_ARGUMENT, "param " + std::to_string(pos + j) + " must be an i32 scalar");
        st_tensor t{};
        t.data = buf.data;
        t.dtype = buf.dtype;
        t.rank = r;
        for (int d = 0; d < r; ++d) {
            t.shape[d] = params[pos + 1 + d].value;
            t.strides[d] = params[pos + 1 + r + d].value;
        }
        ST_TRY(check_view(&t, "array", r));
        if (buf.bytes) {
            const int64_t span = view_span(t);
            if (static_cast<uint64_t>(span) * dtype_size(t.dtype) > buf.bytes)
                return fail(ST_ERR_INVALID_ARGUMENT, "array " + std::to_string(i) + " descriptor reaches past its buffer");
        }
        views->push_back(t);
        buffer_index->push_back(pos);
        pos += need;
    }
    const int extra = n_params - pos;
    if (extra > e.n_constants)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(e.name) + " takes at most " + std::to_string(e.n_constants) +
                                                 " trailing constants");
    for (int i = 0; i < 3; ++i) consts[i] = e.defaults[i];
    for (int i = 0; i < extra; ++i) {
        if (params[pos + i].kind != ST_PARAM_I32 || params[pos + i].value <= 0 || params[pos + i].value > (1 << 20))
            return fail(ST_ERR_INVALID_ARGUMENT, "kernel constants must be positive i32 tile sizes");
        consts[i] = static_cast<int>(params[pos + i].value);
    }
    return ST_OK;
}

int run_entry(const ExecCtx &x, const Entry &e, const st_grid &grid, std::vector<st_tensor> &v, const int consts[3]) {
    const int64_t blocks = static_cast<int64_t>(grid.x) * grid.y * grid.z;
    if (e.kind == Kind::VectorAdd1D) {
        for (int i = 0; i < 3; ++i)
            if (v[i].dtype != ST_F32) return fail(ST_ERR_INVALID_ARGUMENT, "vector_add is f32-only");
        const int64_t tile = consts[0];
        int64_t n = blocks * tile;
        if (n > v[2].shape[0]) n = v[2].shape[0];
        if (n > v[0].shape[0] || n > v[1].shape[0])
            return fail(ST_ERR_INVALID_ARGUMENT, "vector_add: A and B must cover every stored element");
        return launch_vector_add_1d(static_cast<const float *>(v[0].data), v[0].strides[0],
                                    static_cast<const float *>(v[1].data), v[1].strides[0],
                                    static_cast<float *>(v[2].data), v[2].strides[0], n, x.dev->sm_count, x.stream);
    }
    if (e.kind == Kind::VectorAdd2D) {
        for (int i = 0; i < 3; ++i)
            if (v[i].dtype != ST_F32) return fail(ST_ERR_INVALID_ARGUMENT, "vector_add_2d is f32-only");
        int64_t rows = static_cast<int64_t>(grid.x) * consts[0], cols = static_cast<int64_t>(grid.y) * consts[1];
        if (grid.z == 0) rows = 0;
        rows = std::min(rows, v[2].shape[0]);
        cols = std::min(cols, v[2].shape[1]);
        for (int i = 0; i < 2; ++i)
            if (rows > v[i].shape[0] || cols > v[i].shape[1])
                return fail(ST_ERR_INVALID_ARGUMENT, "vector_add_2d: A and B must cover every stored element");
        return launch_vector_add_2d(static_cast<const float *>(v[0].data), v[0].strides,
                                    static_cast<const float *>(v[1].data), v[1].strides,
                                    static_cast<float *>(v[2].data), v[2].strides, rows, cols, x.dev->sm_count,
                                    x.stream);
    }
    if (e.kind == Kind::Fma1D || e.kind == Kind::Cast1D || e.kind == Kind::Fma2D || e.kind == Kind::Cast2D) {
        const bool fma = e.kind == Kind::Fma1D || e.kind == Kind::Fma2D;
        const size_t n_in = fma ? 3 : 1;
        st_tensor &out = v[n_in];
        if (fma)
            for (size_t i = 0; i <= n_in; ++i)
                if (v[i].dtype != ST_F32) return fail(ST_ERR_INVALID_ARGUMENT, std::string(e.name) + " is f32-only");
        int64_t rows, cols;
        if (out.rank == 1) {
            rows = 1;
            cols = std::min<int64_t>(blocks * consts[0], out.shape[0]);
            for (size_t i = 0; i < n_in; ++i)
                if (cols > v[i].shape[0])
                    return fail(ST_ERR_INVALID_ARGUMENT, std::string(e.name) + ": inputs must cover every stored element");
        } else {
            rows = std::min<int64_t>(static_cast<int64_t>(grid.x) * consts[0], out.shape[0]);
            cols = std::min<int64_t>(static_cast<int64_t>(grid.y) * consts[1], out.shape[1]);
            if (grid.z == 0) rows = 0;
            for (size_t i = 0; i < n_in; ++i)
                if (rows > v[i].shape[0] || cols > v[i].shape[1])
                    return fail(ST_ERR_INVALID_ARGUMENT, std::string(e.name) + ": inputs must cover every stored element");
        }
        int64_t s[4][2];
        for (size_t i = 0; i <= n_in; ++i) {
            s[i][0] = v[i].rank == 1 ? cols : v[i].strides[0];
            s[i][1] = v[i].rank == 1 ? v[i].strides[0] : v[i].strides[1];
        }
        if (fma)
            return launch_vector_fma(static_cast<const float *>(v[0].data), s[0], static_cast<const float *>(v[1].data),
                                     s[1], static_cast<const float *>(v[2].data), s[2], static_cast<float *>(v[3].data),
                                     s[3], rows, cols, x.dev->sm_count, x.stream);
        return launch_cast(v[0].data, v[0].dtype, s[0], v[1].data, v[1].dtype, s[1], rows, cols, x.dev->sm_count,
                           x.stream);
    }
    const st_tensor *bias = e.bias ? &v[3] : nullptr;
    ST_TRY(check_matmul(&v[0], &v[1], bias, &v[2]));
    if (v[0].dtype != e.in_dtype)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(e.name) + ": A/B dtype does not match the entry");
    const int64_t tiles = cdiv(v[0].shape[0], consts[0]) * cdiv(v[1].shape[1], consts[1]);
    if (blocks < 1) return fail(ST_ERR_INVALID_ARGUMENT, "empty grid");
    if (!e.persistent && blocks < tiles)
        return fail(ST_ERR_UNSUPPORTED, std::string(e.name) + ": the grid must cover all " + std::to_string(tiles) +
                                            " output tiles (the runtime picks its own tile shape)");
    return matmul_device(x, v[0], v[1], bias, v[2]);
}

// A host-buffer launch split over every device of the context
// (ST_EXEC_ALL_DEVICES): the region the tile grid covers, by the same rules
// as run_entry, goes to the split host calls, which write C in place.
int run_entry_split(st_ctx *ctx, const ExecCtx &x, const Entry &e, const st_grid &grid, std::vector<st_tensor> &v,
                    const int consts[3]) {
    const int64_t blocks = static_cast<int64_t>(grid.x) * grid.y * grid.z;
    if (e.kind == Kind::VectorAdd1D) {
        for (int i = 0; i < 3; ++i)
            if (v[i].dtype != ST_F32) return fail(ST_ERR_INVALID_ARGUMENT, "vector_add is f32-only");
        const int64_t n = std::min<int64_t>(blocks * consts[0], v[2].shape[0]);
        if (n > v[0].shape[0] || n > v[1].shape[0])
            return fail(ST_ERR_INVALID_ARGUMENT, "vector_add: A and B must cover every stored element");
        for (int i = 0; i < 3; ++i) v[i].shape[0] = n;
        return vector_add_host_split(ctx, x, v[0], v[1], v[2]);
    }
    if (e.kind == Kind::VectorAdd2D) {
        for (int i = 0; i < 3; ++i)
            if (v[i].dtype != ST_F32) return fail(ST_ERR_INVALID_ARGUMENT, "vector_add_2d is f32-only");
        int64_t rows = grid.z == 0 ? 0 : std::min<int64_t>(static_cast<int64_t>(grid.x) * consts[0], v[2].shape[0]);
        const int64_t cols = std::min<int64_t>(static_cast<int64_t>(grid.y) * consts[1], v[2].shape[1]);
        for (int i = 0; i < 2; ++i)
            if (rows > v[i].shape[0] || cols > v[i].shape[1])
                return fail(ST_ERR_INVALID_ARGUMENT, "vector_add_2d: A and B must cover every stored element");
        for (int i = 0; i < 3; ++i) {
            v[i].shape[0] = rows;
            v[i].shape[1] = cols;
        }
        return vector_add_host_split(ctx, x, v[0], v[1], v[2]);
    }
    if (e.kind != Kind::Matmul)
        return fail(ST_ERR_UNSUPPORTED, std::string(e.name) +
                                            ": ST_EXEC_ALL_DEVICES splits vector_add, vector_add_2d and matmul entries");
    const st_tensor *bias = e.bias ? &v[3] : nullptr;
    ST_TRY(check_matmul(&v[0], &v[1], bias, &v[2]));
    if (v[0].dtype != e.in_dtype)
        return fail(ST_ERR_INVALID_ARGUMENT, std::string(e.name) + ": A/B dtype does not match the entry");
    const int64_t tiles = cdiv(v[0].shape[0], consts[0]) * cdiv(v[1].shape[1], consts[1]);
    if (blocks < 1) return fail(ST_ERR_INVALID_ARGUMENT, "empty grid");
    if (!e.persistent && blocks < tiles)
        return fail(ST_ERR_UNSUPPORTED, std::string(e.name) + ": the grid must cover all " + std::to_string(tiles) +
                                            " output tiles (the runtime picks its own tile shape)");
    return matmul_host_split(ctx, x, v[0], v[1], bias, v[2]);
}

}  // namespace
}  // namespace st

// ============================================================ C ABI
using namespace st;

extern "C" {

const char *st_version(void) { return "sptiles_b200 0.1.0 (sm_100a)"; }

const char *st_last_error(void) { return g_last_error.c_str(); }

int st_device_count(int32_t *count) {
    if (!count) return fail(ST_ERR_INVALID_ARGUMENT, "count is null");
    int n = 0;
    const cudaError_t e = cudaGetDeviceCount(&n);
    if (e != cudaSuccess) {
        cudaGetLastError();
        *count = 0;
        g_last_error = std::string("cudaGetDeviceCount: ") + cudaGetErrorString(e);
        return ST_OK;
    }
    *count = n;
    return ST_OK;
}

int st_kernel_launches(uint64_t *count) {
    if (!count) return fail(ST_ERR_INVALID_ARGUMENT, "count is null");
    *count = g_launches.load(std::memory_order_relaxed);
    return ST_OK;
}

int st_init(const int32_t *devices, int32_t n_devices, st_ctx **out) {
    if (!out) return fail(ST_ERR_INVALID_ARGUMENT, "out is null");
    *out = nullptr;
    if (n_devices < 0 || (n_devices > 0 && !devices))
        return fail(ST_ERR_INVALID_ARGUMENT, "bad device list");
    int count = 0;
    cudaError_t e = cudaGetDeviceCount(&count);
    if (e != cudaSuccess || count == 0) {
        cudaGetLastError();
        return fail(ST_ERR_NO_DEVICE, "no CUDA device is visible");
    }
    std::vector<int> ords;
    if (n_devices == 0) ords.push_back(0);
    for (int i = 0; i < n_devices; ++i) ords.push_back(devices[i]);
    auto *ctx = new st_ctx();
    for (int ord : ords) {
        if (ord < 0 || ord >= count) {
            st_shutdown(ctx);
            return fail(ST_ERR_INVALID_ARGUMENT, "device ordinal " + std::to_string(ord) + " out of range");
        }
        DeviceGuard guard(ord);
        cudaDeviceProp prop;
        e = cudaGetDeviceProperties(&prop, ord);
        if (e != cudaSuccess) {
            st_shutdown(ctx);
            return cuda_fail(e, "cudaGetDeviceProperties");
        }
        if (prop.major != 10) {
            st_shutdown(ctx);
            return fail(ST_ERR_NO_DEVICE, std::string("device ") + std::to_string(ord) + " (" + prop.name +
                                              ") is not sm_100; these kernels are built for sm_100a only");
        }
        DeviceState d;
        d.ordinal = ord;
        d.sm_count = prop.multiProcessorCount;
        if ((e = cudaStreamCreateWithFlags(&d.stream, cudaStreamNonBlocking)) != cudaSuccess ||
            (e = cudaMalloc(&d.dev_err, sizeof(int))) != cudaSuccess ||
            (e = cudaMemset(d.dev_err, 0, sizeof(int))) != cudaSuccess) {
            ctx->devs.push_back(d);
            st_shutdown(ctx);
            return cuda_fail(e, "device set-up");
        }
        ctx->devs.push_back(d);
    }
    // peer access between the context's devices (NVLink), for peer copies and
    // for GEMM epilogues that store into another device's copy of C
    for (int i : ords)
        for (int j : ords) {
            int can = 0;
            if (i == j || cudaDeviceCanAccessPeer(&can, i, j) != cudaSuccess || !can) {
                cudaGetLastError();
                continue;
            }
            DeviceGuard guard(i);
            if (cudaDeviceEnablePeerAccess(j, 0) != cudaSuccess) cudaGetLastError();  // already enabled is fine
        }
    *out = ctx;
    return ST_OK;
}

int st_shutdown(st_ctx *ctx) {
    if (!ctx) return ST_OK;
    for (auto &d : ctx->devs) {
        DeviceGuard guard(d.ordinal);
        if (d.stream) cudaStreamSynchronize(d.stream);
        if (d.copy_in) cudaStreamSynchronize(d.copy_in);
        if (d.copy_out) cudaStreamSynchronize(d.copy_out);
        ws_free(d.scratch);
        ws_free(d.stage);
        ws_free(d.sk);
        for (cudaEvent_t e : d.events) cudaEventDestroy(e);
        if (d.copy_in) cudaStreamDestroy(d.copy_in);
        if (d.copy_out) cudaStreamDestroy(d.copy_out);
        if (d.dev_err) cudaFree(d.dev_err);
        if (d.stream) cudaStreamDestroy(d.stream);
    }
    delete ctx;
    return ST_OK;
}

int st_sync(st_ctx *ctx, int32_t device, uint32_t timeout_ms) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    DeviceGuard guard(d->ordinal);
    return bounded_sync(d, d->stream, timeout_ms);
}

int st_stream(st_ctx *ctx, int32_t device, void **stream) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    if (!stream) return fail(ST_ERR_INVALID_ARGUMENT, "stream is null");
    *stream = d->stream;
    return ST_OK;
}

int st_alloc(st_ctx *ctx, int32_t device, uint64_t bytes, void **out) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    if (!out) return fail(ST_ERR_INVALID_ARGUMENT, "out is null");
    DeviceGuard guard(d->ordinal);
    *out = nullptr;
    if (bytes == 0) return ST_OK;
    ST_CUDA_TRY(cudaMalloc(out, bytes));
    return ST_OK;
}

int st_free(st_ctx *ctx, int32_t device, void *ptr) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    DeviceGuard guard(d->ordinal);
    if (ptr) ST_CUDA_TRY(cudaFree(ptr));
    return ST_OK;
}

int st_upload(st_ctx *ctx, int32_t device, void *dst, const void *src, uint64_t bytes) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    if (bytes && (!dst || !src)) return fail(ST_ERR_INVALID_ARGUMENT, "null pointer");
    DeviceGuard guard(d->ordinal);
    if (bytes) ST_CUDA_TRY(cudaMemcpyAsync(dst, src, bytes, cudaMemcpyHostToDevice, d->stream));
    return bounded_sync(d, d->stream, 0);
}

int st_download(st_ctx *ctx, int32_t device, void *dst, const void *src, uint64_t bytes) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    if (bytes && (!dst || !src)) return fail(ST_ERR_INVALID_ARGUMENT, "null pointer");
    DeviceGuard guard(d->ordinal);
    if (bytes) ST_CUDA_TRY(cudaMemcpyAsync(dst, src, bytes, cudaMemcpyDeviceToHost, d->stream));
    return bounded_sync(d, d->stream, 0);
}

int st_grid_from_dispatch(const char *entry_name, const uint32_t dispatch[3], int64_t tile_elems, st_grid *out) {
    const Entry *e = find_entry(entry_name);
    if (!e) return fail(ST_ERR_UNKNOWN_ENTRY, std::string("unknown entry '") + (entry_name ? entry_name : "") + "'");
    if (!dispatch || !out || tile_elems <= 0) return fail(ST_ERR_INVALID_ARGUMENT, "bad dispatch conversion arguments");
    if (e->kind == Kind::VectorAdd2D)
        return fail(ST_ERR_UNSUPPORTED, "a 2D tile grid cannot be recovered from a linear dispatch");
    const int64_t inv = static_cast<int64_t>(dispatch[0]) * dispatch[1] * dispatch[2] * 1024;
    const int64_t tiles = cdiv(inv, tile_elems);
    if (tiles > UINT32_MAX) return fail(ST_ERR_INVALID_ARGUMENT, "dispatch too large");
    *out = st_grid{static_cast<uint32_t>(tiles), 1, 1};
    return ST_OK;
}

int st_launch(st_ctx *ctx, const char *entry_name, const st_grid *grid, const st_param *params, int32_t n_params,
              const st_exec *exec) {
    const Entry *e = find_entry(entry_name);
    if (!e) return fail(ST_ERR_UNKNOWN_ENTRY, std::string("Entry point ") + (entry_name ? entry_name : "(null)") +
                                                  " was not found in the kernel registry.");
    if (!grid || (!params && n_params > 0) || n_params < 0)
        return fail(ST_ERR_INVALID_ARGUMENT, "grid and params are required");
    const bool split = exec && (exec->flags & ST_EXEC_ALL_DEVICES);
    if (split && !(exec->flags & ST_EXEC_HOST_BUFFERS))
        return fail(ST_ERR_INVALID_ARGUMENT, kAllDevicesScope);
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x, true));
    std::vector<st_tensor> views;
    std::vector<int> bufpos;
    int consts[3];
    ST_TRY(parse_params(*e, params, n_params, &views, &bufpos, consts));
    if (split) {  // host buffers split over every device: C is written in place
        ST_TRY(check_all_devices(exec));
        return run_entry_split(ctx, x, *e, *grid, views, consts);
    }
    DeviceGuard guard(x.dev->ordinal);
    if (!(x.flags & ST_EXEC_HOST_BUFFERS)) {
        ST_TRY(run_entry(x, *e, *grid, views, consts));
        return finish(x);
    }
    // host buffers: stage every array, run, copy the requested outputs back
    // (the run_spirv_kernel contract, spirv_runtime.py:153-174)
    for (size_t i = 0; i < views.size(); ++i)
        if (params[bufpos[i]].bytes == 0)
            return fail(ST_ERR_INVALID_ARGUMENT, "host-buffer launches need the size of every buffer");
    size_t total = 0;
    for (size_t i = 0; i < views.size(); ++i) total += (params[bufpos[i]].bytes + 255) & ~uint64_t(255);
    void *base = nullptr;
    ST_TRY(ws_acquire(x.dev->stage, total, x.stream, &base));
    uint8_t *cursor = static_cast<uint8_t *>(base);
    std::vector<st_tensor> dev_views = views;
    std::vector<uint8_t *> dev_bufs;
    for (size_t i = 0; i < views.size(); ++i) {
        const st_param &p = params[bufpos[i]];
        ST_CUDA_TRY(cudaMemcpyAsync(cursor, p.data, p.bytes, cudaMemcpyHostToDevice, x.stream));
        dev_views[i].data = cursor;
        dev_bufs.push_back(cursor);
        cursor += (p.bytes + 255) & ~uint64_t(255);
    }
    ST_TRY(run_entry(x, *e, *grid, dev_views, consts));
    // default output: C, the third array of the add/matmul signatures, the last one otherwise
    const int32_t default_out[1] = {(e->kind == Kind::VectorAdd1D || e->kind == Kind::VectorAdd2D ||
                                     e->kind == Kind::Matmul)
                                        ? bufpos[2]
                                        : bufpos.back()};
    const int32_t *outs = exec && exec->n_outputs > 0 ? exec->output_indices : default_out;
    const int n_outs = exec && exec->n_outputs > 0 ? exec->n_outputs : 1;
    for (int i = 0; i < n_outs; ++i) {
        const int idx = outs[i];
        size_t which = views.size();
        for (size_t j = 0; j < bufpos.size(); ++j)
            if (bufpos[j] == idx) which = j;
        if (which == views.size()) return fail(ST_ERR_INVALID_ARGUMENT, "output index must name a buffer param");
        ST_CUDA_TRY(cudaMemcpyAsync(params[idx].data, dev_bufs[which], params[idx].bytes, cudaMemcpyDeviceToHost,
                                    x.stream));
    }
    ST_TRY(ws_release(x.dev->stage, x.stream));
    return bounded_sync(x.dev, x.stream, x.timeout_ms);
}

int st_vector_add(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *c, const st_exec *exec) {
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    ST_TRY(check_vector_add(a, b, c));
    DeviceGuard guard(x.dev->ordinal);
    const int64_t rows = c->rank == 2 ? c->shape[0] : 1;
    const int64_t cols = c->rank == 2 ? c->shape[1] : c->shape[0];
    ST_TRY(vector_add_views(x, *a, *b, *c, rows, cols));
    return finish(x);
}

int st_matmul(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *bias, const st_tensor *c,
              const st_exec *exec) {
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    ST_TRY(check_matmul(a, b, bias, c));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(matmul_device(x, *a, *b, bias, *c));
    return finish(x);
}

int st_vector_fma(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *d, const st_tensor *c,
                  const st_exec *exec) {
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    ST_TRY(check_vector_add(a, b, c));
    ST_TRY(check_vector_add(a, d, c));
    DeviceGuard guard(x.dev->ordinal);
    const int64_t rows = c->rank == 2 ? c->shape[0] : 1;
    const int64_t cols = c->rank == 2 ? c->shape[1] : c->shape[0];
    int64_t s[4][2];
    const st_tensor *t[4] = {a, b, d, c};
    for (int i = 0; i < 4; ++i) {
        s[i][0] = t[i]->rank == 1 ? cols : t[i]->strides[0];
        s[i][1] = t[i]->rank == 1 ? t[i]->strides[0] : t[i]->strides[1];
    }
    ST_TRY(launch_vector_fma(static_cast<const float *>(a->data), s[0], static_cast<const float *>(b->data), s[1],
                             static_cast<const float *>(d->data), s[2], static_cast<float *>(c->data), s[3], rows, cols,
                             x.dev->sm_count, x.stream));
    return finish(x);
}

int st_quantize_fp8(st_ctx *ctx, const st_tensor *a, const st_tensor *q, const st_tensor *scale, int32_t block_rows,
                    int32_t block_cols, const st_exec *exec) {
    ST_TRY(check_matrix(a, "A"));
    ST_TRY(check_matrix(q, "Q"));
    ST_TRY(check_matrix(scale, "scale"));
    const bool known = (block_rows == 1 && block_cols == 128) || (block_rows == 128 && block_cols == 1) ||
                       (block_rows == 128 && block_cols == 128);
    if (!known) return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp8: blocks are 1 x 128, 128 x 1 or 128 x 128");
    if (!is_float(a->dtype)) return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp8: A must be ST_F32, ST_F16 or ST_BF16");
    if (!is_fp8(q->dtype)) return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp8: Q must be ST_E4M3 or ST_E5M2");
    if (scale->dtype != ST_F32) return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp8: scale must be ST_F32");
    if (q->shape[0] != a->shape[0] || q->shape[1] != a->shape[1])
        return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp8: A and Q must have the same shape");
    if (scale->shape[0] != cdiv(a->shape[0], block_rows) || scale->shape[1] != cdiv(a->shape[1], block_cols))
        return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp8: scale must be [" +
                                                 std::to_string(cdiv(a->shape[0], block_rows)) + ", " +
                                                 std::to_string(cdiv(a->shape[1], block_cols)) + "]");
    ST_TRY(check_output(*q, "Q"));
    ST_TRY(check_output(*scale, "scale"));
    QuantizeArgs g{};
    g.a = a->data;
    g.a_dtype = a->dtype;
    g.sa0 = a->strides[0];
    g.sa1 = a->strides[1];
    g.q = q->data;
    g.e5m2 = q->dtype == ST_E5M2;
    g.sq0 = q->strides[0];
    g.sq1 = q->strides[1];
    g.scale = static_cast<float *>(scale->data);
    g.ss0 = scale->strides[0];
    g.ss1 = scale->strides[1];
    g.rows = a->shape[0];
    g.cols = a->shape[1];
    g.block_rows = block_rows;
    g.block_cols = block_cols;
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_quantize_fp8(g, x.stream));
    return finish(x);
}

int st_matmul_fp8_workspace(const st_tensor *a, const st_tensor *b, uint64_t *bytes) {
    if (!bytes) return fail(ST_ERR_INVALID_ARGUMENT, "bytes is null");
    ST_TRY(check_fp8_operands(a, b));
    *bytes = static_cast<uint64_t>(gemm_fp8_workspace_bytes(fp8_operand(*a, false), fp8_operand(*b, true)));
    return ST_OK;
}

int st_matmul_fp8(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *a_scale,
                  const st_tensor *b_scale, const st_tensor *bias, const st_tensor *c, void *workspace,
                  uint64_t workspace_bytes, const st_exec *exec) {
    ST_TRY(check_fp8_operands(a, b));
    ST_TRY(check_matrix(c, "C"));
    GemmFp8Args g{};
    g.a = fp8_operand(*a, false);
    g.b = fp8_operand(*b, true);
    ST_TRY(set_scale(a_scale, "a_scale", false, &g.a));
    ST_TRY(set_scale(b_scale, "b_scale", true, &g.b));
    if (c->shape[0] != g.a.rows || c->shape[1] != g.b.rows)
        return fail(ST_ERR_INVALID_ARGUMENT, "C must be [M, N] = [" + std::to_string(g.a.rows) + ", " +
                                                 std::to_string(g.b.rows) + "]");
    if (!is_float(c->dtype)) return fail(ST_ERR_INVALID_ARGUMENT, "C must be ST_F32, ST_F16 or ST_BF16");
    if (!unit_columns(*c)) return fail(ST_ERR_UNSUPPORTED, "C must have unit column stride");
    ST_TRY(check_output(*c, "C"));
    if (bias) {
        if (bias->rank != 1 || bias->shape[0] != g.b.rows)
            return fail(ST_ERR_INVALID_ARGUMENT, "bias must have N elements");
        if (bias->dtype != ST_F32 && (bias->dtype != c->dtype || !is_float(bias->dtype)))
            return fail(ST_ERR_INVALID_ARGUMENT, "bias must be ST_F32 or C's dtype");
        if (bias->shape[0] > 1 && bias->strides[0] != 1) return fail(ST_ERR_UNSUPPORTED, "bias must be contiguous");
        if (bias->shape[0] > 0 && !bias->data) return fail(ST_ERR_INVALID_ARGUMENT, "bias has a null data pointer");
        g.bias = bias->data;
        g.bias_dtype = bias->dtype;
    }
    const int64_t need = gemm_fp8_workspace_bytes(g.a, g.b);
    if (need > 0 && (!workspace || workspace_bytes < static_cast<uint64_t>(need)))
        return fail(ST_ERR_INVALID_ARGUMENT, "matmul_fp8 needs a workspace of " + std::to_string(need) +
                                                 " bytes for operands that are not on 16-byte boundaries");
    if (need > 0 && !aligned16(workspace)) return fail(ST_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    g.c = c->data;
    g.ldc = c->strides[0];
    g.c_dtype = c->dtype;
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_gemm_fp8(g, workspace, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
    return finish(x);
}

int st_quantize_fp4_workspace(uint64_t *bytes) {
    if (!bytes) return fail(ST_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = static_cast<uint64_t>(quantize_fp4_workspace_bytes());
    return ST_OK;
}

int st_quantize_fp4(st_ctx *ctx, const st_tensor *a, const st_tensor *q, const st_tensor *scale, const st_tensor *amax,
                    const st_tensor *tensor_scale, void *workspace, uint64_t workspace_bytes, const st_exec *exec) {
    ST_TRY(check_matrix(a, "A"));
    ST_TRY(check_codes(q, "Q"));
    if (!is_float(a->dtype)) return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp4: A must be ST_F32, ST_F16 or ST_BF16");
    ST_TRY(check_elements(*a, "A"));
    if (q->shape[0] != a->shape[0] || q->shape[1] != cdiv(a->shape[1], 2))
        return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp4: Q must be [rows, ceil(cols / 2)] = [" + std::to_string(a->shape[0]) + ", " +
                                                 std::to_string(cdiv(a->shape[1], 2)) + "]");
    if (!unit_columns(*q)) return fail(ST_ERR_UNSUPPORTED, "quantize_fp4: Q must have unit column stride");
    ST_TRY(check_output(*q, "Q"));
    ST_TRY(check_fp4_scale(scale, "scale", q->shape[0], q->shape[1]));
    Quantize4Args g{};
    float *known = nullptr;
    ST_TRY(scalar_of(amax, "amax", &known));
    ST_TRY(scalar_of(tensor_scale, "tensor_scale", &g.tensor_scale));
    g.wide = scale->dtype == ST_E8M0;
    if (g.wide && (amax || tensor_scale))
        return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp4: amax and tensor_scale go with ST_E4M3 scales");
    if (!g.wide && !tensor_scale) return fail(ST_ERR_INVALID_ARGUMENT, "quantize_fp4: ST_E4M3 scales need tensor_scale");
    if (!g.wide && !known && a->shape[0] > 0 && a->shape[1] > 0)
        ST_TRY(check_workspace("quantize_fp4", quantize_fp4_workspace_bytes(), workspace, workspace_bytes, 4));
    g.a = a->data;
    g.a_dtype = a->dtype;
    g.sa0 = a->strides[0];
    g.sa1 = a->strides[1];
    g.rows = a->shape[0];
    g.cols = a->shape[1];
    g.q = static_cast<uint8_t *>(q->data);
    g.sq0 = q->strides[0];
    g.scale = static_cast<uint8_t *>(scale->data);
    g.maxima = known;
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_quantize_fp4(g, workspace, x.dev->sm_count, x.stream));
    return finish(x);
}

int st_dequantize_fp4(st_ctx *ctx, const st_tensor *q, const st_tensor *scale, const st_tensor *tensor_scale,
                      const st_tensor *out, const st_exec *exec) {
    ST_TRY(check_codes(q, "Q"));
    ST_TRY(check_matrix(out, "out"));
    ST_TRY(check_fp4_scale(scale, "scale", q->shape[0], q->shape[1]));
    if (!is_float(out->dtype)) return fail(ST_ERR_INVALID_ARGUMENT, "dequantize_fp4: out must be ST_F32, ST_F16 or ST_BF16");
    if (out->shape[0] != q->shape[0] || cdiv(out->shape[1], 2) != q->shape[1])
        return fail(ST_ERR_INVALID_ARGUMENT, "dequantize_fp4: out must be [" + std::to_string(q->shape[0]) + ", " +
                                                 std::to_string(2 * q->shape[1]) + "], or a column less");
    ST_TRY(check_elements(*out, "out"));
    ST_TRY(check_output(*out, "out"));
    Dequantize4Args g{};
    float *t = nullptr;
    ST_TRY(scalar_of(tensor_scale, "tensor_scale", &t));
    g.wide = scale->dtype == ST_E8M0;
    if (g.wide && t) return fail(ST_ERR_INVALID_ARGUMENT, "dequantize_fp4: tensor_scale goes with ST_E4M3 scales");
    g.q = static_cast<const uint8_t *>(q->data);
    g.sq0 = q->strides[0];
    g.sq1 = q->shape[1] > 1 ? q->strides[1] : 1;
    g.rows = out->shape[0];
    g.cols = out->shape[1];
    g.scale = static_cast<const uint8_t *>(scale->data);
    g.tensor_scale = t;
    g.out = out->data;
    g.out_dtype = out->dtype;
    g.so0 = out->strides[0];
    g.so1 = out->shape[1] > 1 ? out->strides[1] : 1;
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_dequantize_fp4(g, x.dev->sm_count, x.stream));
    return finish(x);
}

int st_matmul_fp4_workspace(const st_tensor *a, const st_tensor *b, uint64_t *bytes) {
    if (!bytes) return fail(ST_ERR_INVALID_ARGUMENT, "bytes is null");
    ST_TRY(check_fp4_operands(a, b));
    *bytes = static_cast<uint64_t>(gemm_fp4_workspace_bytes(fp4_operand(*a, false), fp4_operand(*b, true)));
    return ST_OK;
}

int st_matmul_fp4(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *a_scale, const st_tensor *b_scale,
                  const st_tensor *a_tensor_scale, const st_tensor *b_tensor_scale, const st_tensor *bias,
                  const st_tensor *c, void *workspace, uint64_t workspace_bytes, const st_exec *exec) {
    ST_TRY(check_fp4_operands(a, b));
    GemmFp4Args g{};
    g.a = fp4_operand(*a, false);
    g.b = fp4_operand(*b, true);
    ST_TRY(check_fp4_scale(a_scale, "a_scale", g.a.rows, g.a.k));
    ST_TRY(check_fp4_scale(b_scale, "b_scale", g.b.rows, g.b.k));
    if (a_scale->dtype != b_scale->dtype)
        return fail(ST_ERR_INVALID_ARGUMENT, "matmul_fp4: a_scale and b_scale must have one type");
    g.wide = a_scale->dtype == ST_E8M0;
    g.a.scale = a_scale->data;
    g.b.scale = b_scale->data;
    float *t = nullptr;
    ST_TRY(scalar_of(a_tensor_scale, "a_tensor_scale", &t));
    g.a.tensor_scale = t;
    ST_TRY(scalar_of(b_tensor_scale, "b_tensor_scale", &t));
    g.b.tensor_scale = t;
    if (g.wide && (a_tensor_scale || b_tensor_scale))
        return fail(ST_ERR_INVALID_ARGUMENT, "matmul_fp4: tensor scales go with ST_E4M3 scales");
    ST_TRY(check_matrix(c, "C"));
    if (c->shape[0] != g.a.rows || c->shape[1] != g.b.rows)
        return fail(ST_ERR_INVALID_ARGUMENT, "C must be [M, N] = [" + std::to_string(g.a.rows) + ", " +
                                                 std::to_string(g.b.rows) + "]");
    if (!is_float(c->dtype)) return fail(ST_ERR_INVALID_ARGUMENT, "C must be ST_F32, ST_F16 or ST_BF16");
    if (!unit_columns(*c)) return fail(ST_ERR_UNSUPPORTED, "C must have unit column stride");
    ST_TRY(check_elements(*c, "C"));
    ST_TRY(check_output(*c, "C"));
    if (bias) {
        if (bias->rank != 1 || bias->shape[0] != g.b.rows)
            return fail(ST_ERR_INVALID_ARGUMENT, "bias must have N elements");
        if (bias->dtype != ST_F32 && (bias->dtype != c->dtype || !is_float(bias->dtype)))
            return fail(ST_ERR_INVALID_ARGUMENT, "bias must be ST_F32 or C's dtype");
        if (bias->shape[0] > 1 && bias->strides[0] != 1) return fail(ST_ERR_UNSUPPORTED, "bias must be contiguous");
        if (bias->shape[0] > 0 && !bias->data) return fail(ST_ERR_INVALID_ARGUMENT, "bias has a null data pointer");
        ST_TRY(check_elements(*bias, "bias"));
        g.bias = bias->data;
        g.bias_dtype = bias->dtype;
    }
    ST_TRY(check_workspace("matmul_fp4", gemm_fp4_workspace_bytes(g.a, g.b), workspace, workspace_bytes, 16));
    g.c = c->data;
    g.ldc = c->strides[0];
    g.c_dtype = c->dtype;
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_gemm_fp4(g, workspace, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
    return finish(x);
}

int st_matmul_grouped_workspace(const st_tensor *a, const st_tensor *b, int64_t b_group_stride, int64_t groups, uint64_t *bytes) {
    if (!bytes) return fail(ST_ERR_INVALID_ARGUMENT, "bytes is null");
    if (groups < 0 || groups > kGroupedMaxGroups) return fail(ST_ERR_INVALID_ARGUMENT, "groups must be in [0, 1024]");
    GroupedArgs g{};
    ST_TRY(grouped_operands("matmul_grouped", a, b, "B", false, groups, b_group_stride, &g));
    *bytes = static_cast<uint64_t>(gemm_grouped_workspace_bytes(g));
    return ST_OK;
}

int st_matmul_grouped(st_ctx *ctx, const st_tensor *a, const st_tensor *b, int64_t b_group_stride, const st_tensor *ends,
                      const st_tensor *c, int32_t zero_rest, void *workspace, uint64_t workspace_bytes, const st_exec *exec) {
    ST_TRY(check_ends(ends));
    GroupedArgs g{};
    ST_TRY(grouped_operands("matmul_grouped", a, b, "B", false, ends->shape[0], b_group_stride, &g));
    ST_TRY(check_grouped_output(c, "C", g.rows, g.n));
    ST_TRY(check_workspace("matmul_grouped", gemm_grouped_workspace_bytes(g), workspace, workspace_bytes, 16));
    g.ends = static_cast<const int *>(ends->data);
    g.c = c->data;
    g.ldc = c->strides[0];
    g.c_dtype = c->dtype;
    g.zero_rest = zero_rest != 0;
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_gemm_grouped(g, workspace, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
    return finish(x);
}

int st_matmul_grouped_weights_workspace(const st_tensor *a, const st_tensor *c, int64_t groups, uint64_t *bytes) {
    if (!bytes) return fail(ST_ERR_INVALID_ARGUMENT, "bytes is null");
    if (groups < 0 || groups > kGroupedMaxGroups) return fail(ST_ERR_INVALID_ARGUMENT, "groups must be in [0, 1024]");
    GroupedArgs g{};
    ST_TRY(grouped_operands("matmul_grouped_weights", a, c, "C", true, groups, 0, &g));
    *bytes = static_cast<uint64_t>(gemm_grouped_workspace_bytes(g));
    return ST_OK;
}

int st_matmul_grouped_weights(st_ctx *ctx, const st_tensor *a, const st_tensor *c, const st_tensor *ends, const st_tensor *d,
                              int64_t d_group_stride, void *workspace, uint64_t workspace_bytes, const st_exec *exec) {
    ST_TRY(check_ends(ends));
    GroupedArgs g{};
    ST_TRY(grouped_operands("matmul_grouped_weights", a, c, "C", true, ends->shape[0], 0, &g));
    st_tensor shape_of_d{};
    if (d && g.groups == 0) {  // no matrix, but the extents of one
        shape_of_d = *d;
        shape_of_d.data = &shape_of_d;
        d = &shape_of_d;
    }
    ST_TRY(check_grouped_output(d, "D", g.k, g.n));
    const int64_t span = g.k > 0 && g.n > 0 ? (g.k - 1) * d->strides[0] + g.n : 0;
    // one group behind the other, or the groups' rows in turn ([K, G, N])
    const bool in_turn = g.groups > 1 && d_group_stride >= g.n && (d->strides[0] - g.n) / (g.groups - 1) >= d_group_stride;
    if (g.groups > 1 && d_group_stride < span && !in_turn)
        return fail(ST_ERR_INVALID_ARGUMENT, "D has overlapping groups: their stride is " + std::to_string(d_group_stride) +
                                                 ", one spans " + std::to_string(span) + " elements");
    ST_TRY(check_workspace("matmul_grouped_weights", gemm_grouped_workspace_bytes(g), workspace, workspace_bytes, 16));
    g.ends = static_cast<const int *>(ends->data);
    g.c = d->data;
    g.c_g = d_group_stride;
    g.ldc = d->strides[0];
    g.c_dtype = d->dtype;
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_gemm_grouped(g, workspace, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
    return finish(x);
}

int st_residual_norm(st_ctx *ctx, const st_tensor *x_in, const st_tensor *residual, const st_tensor *post,
                     const st_tensor *gate, const st_tensor *pre, const st_tensor *residual_out,
                     const st_tensor *normed, const st_tensor *normed_scale, const st_norm_options *options,
                     const st_exec *exec) {
    ST_TRY(check_matrix(residual, "residual"));
    NormArgs g{};
    g.rows = residual->shape[0];
    g.cols = residual->shape[1];
    ST_TRY(check_norm_options("residual_norm", options, g.cols));
    g.alpha = options->alpha;
    g.eps = options->eps;
    g.offset = options->weight_offset;
    ST_TRY(norm_view(residual, "residual", g.rows, g.cols, false, &g.r));
    ST_TRY(norm_view(x_in, "x", g.rows, g.cols, false, &g.x));
    ST_TRY(norm_view(residual_out, "residual_out", g.rows, g.cols, true, &g.r_out));
    ST_TRY(norm_view(normed, "normed", g.rows, g.cols, true, &g.h));
    ST_TRY(norm_weight(post, "post_weight", g.cols, &g.post));
    ST_TRY(norm_weight(pre, "pre_weight", g.cols, &g.pre));
    ST_TRY(norm_gate(gate, g.rows, g.cols, &g.gate, &g.gate_mode));
    if (!x_in && (post || gate)) return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm: post_weight and gate need x");
    if ((pre != nullptr) != (normed != nullptr))
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm: pre_weight and normed come together");
    if (!residual_out && !normed) return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm: nothing to compute");
    g.h_fp8 = normed && is_fp8(normed->dtype);
    g.h_e5m2 = normed && normed->dtype == ST_E5M2;
    const int t = x_in ? x_in->dtype : (normed && !g.h_fp8 ? normed->dtype : residual->dtype);
    ST_TRY(check_norm_types("residual_norm", t, residual->dtype));
    g.branch = t;
    g.stream = residual->dtype;
    if (residual_out && residual_out->dtype != residual->dtype)
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm: residual and residual_out must have the same dtype");
    if (normed && !g.h_fp8 && normed->dtype != t)
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm: normed must have x's dtype, ST_E4M3 or ST_E5M2");
    ST_TRY(check_side_types("residual_norm", t, {{&g.post, "post_weight"}, {&g.pre, "pre_weight"}, {&g.gate, "gate"}}));
    if (g.h_fp8 != (normed_scale != nullptr))
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm: 8-bit blocks come with their scales, and only they do");
    if (g.h_fp8) {
        ST_TRY(check_matrix(normed_scale, "normed_scale"));
        if (normed_scale->dtype != ST_F32 || normed_scale->shape[0] != g.rows ||
            normed_scale->shape[1] != cdiv(g.cols, kScaleBlock))
            return fail(ST_ERR_INVALID_ARGUMENT, "normed_scale must be ST_F32 [" + std::to_string(g.rows) + ", " +
                                                     std::to_string(cdiv(g.cols, kScaleBlock)) + "]");
        ST_TRY(check_output(*normed_scale, "normed_scale"));
        g.h_scale = static_cast<float *>(normed_scale->data);
        g.hs0 = normed_scale->strides[0];
        g.hs1 = normed_scale->strides[1];
    }
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_residual_norm(g, x.dev->sm_count, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
    return finish(x);
}

int st_residual_norm_backward_workspace(int64_t rows, int64_t cols, uint64_t *bytes) {
    if (!bytes) return fail(ST_ERR_INVALID_ARGUMENT, "bytes is null");
    if (rows < 0 || cols < 1 || rows > INT32_MAX || cols > INT32_MAX)
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: bad extents");
    *bytes = static_cast<uint64_t>(residual_norm_backward_workspace(rows, cols));
    return ST_OK;
}

int st_residual_norm_backward(st_ctx *ctx, const st_tensor *d_residual, const st_tensor *d_normed,
                              const st_tensor *x_in, const st_tensor *residual, const st_tensor *post,
                              const st_tensor *gate, const st_tensor *pre, const st_tensor *dx, const st_tensor *dr,
                              const st_tensor *dpost, const st_tensor *dgate, const st_tensor *dpre, void *workspace,
                              uint64_t workspace_bytes, const st_norm_options *options, const st_exec *exec) {
    const char *const what = "residual_norm_backward";
    if (!d_residual && !d_normed) return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: no gradient to take back");
    const st_tensor *like = d_residual ? d_residual : d_normed;
    ST_TRY(check_matrix(like, d_residual ? "d_residual" : "d_normed"));
    NormBackwardArgs g{};
    g.rows = like->shape[0];
    g.cols = like->shape[1];
    ST_TRY(check_norm_options(what, options, g.cols));
    g.alpha = options->alpha;
    g.eps = options->eps;
    g.offset = options->weight_offset;
    ST_TRY(norm_view(d_residual, "d_residual", g.rows, g.cols, false, &g.d_residual));
    ST_TRY(norm_view(d_normed, "d_normed", g.rows, g.cols, false, &g.d_normed));
    ST_TRY(norm_view(x_in, "x", g.rows, g.cols, false, &g.x));
    ST_TRY(norm_view(residual, "residual", g.rows, g.cols, false, &g.r));
    ST_TRY(norm_view(dx, "dx", g.rows, g.cols, true, &g.dx));
    ST_TRY(norm_view(dr, "dr", g.rows, g.cols, true, &g.dr));
    ST_TRY(norm_weight(post, "post_weight", g.cols, &g.post));
    ST_TRY(norm_weight(pre, "pre_weight", g.cols, &g.pre));
    ST_TRY(norm_gate(gate, g.rows, g.cols, &g.gate, &g.gate_mode));
    if (!x_in && (post || gate)) return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: post_weight and gate need x");
    if ((x_in != nullptr) != (dx != nullptr)) return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: x and dx come together");
    if ((pre != nullptr) != (d_normed != nullptr))
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: pre_weight and d_normed come together");
    if (pre && !residual) return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: pre_weight needs the updated residual");
    if (!pre) g.r = NormView{};
    const int t = x_in ? x_in->dtype : (d_normed ? d_normed->dtype : d_residual->dtype);
    const int s = residual && pre ? residual->dtype : (d_residual ? d_residual->dtype : t);
    ST_TRY(check_norm_types(what, t, s));
    g.branch = t;
    g.stream = s;
    if ((d_residual && d_residual->dtype != s) || (dr && dr->dtype != s) || (d_normed && d_normed->dtype != t) ||
        (dx && dx->dtype != t))
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: a gradient must have the dtype of its tensor");
    ST_TRY(check_side_types(what, t, {{&g.post, "post_weight"}, {&g.pre, "pre_weight"}, {&g.gate, "gate"}}));
    NormView sum;
    if ((dpost && !post) || (dpre && !pre) || (dgate != nullptr) != (gate != nullptr))
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: dpost, dpre and dgate go with their tensors");
    ST_TRY(norm_weight(dpost, "dpost", g.cols, &sum));
    ST_TRY(norm_weight(dpre, "dpre", g.cols, &sum));
    if ((dpost && dpost->dtype != ST_F32) || (dpre && dpre->dtype != ST_F32))
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: dpost and dpre must be ST_F32");
    g.dpost = dpost ? static_cast<float *>(dpost->data) : nullptr;
    g.dpre = dpre ? static_cast<float *>(dpre->data) : nullptr;
    if (dgate) {
        int mode = kGateNone;
        ST_TRY(norm_gate(dgate, g.rows, g.cols, &g.dgate, &mode));
        if (mode != g.gate_mode) return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: dgate must have the gate's shape");
        if (dgate->rank == 2) ST_TRY(check_output(*dgate, "dgate"));
        if (dgate->dtype != ST_F32 && (mode != kGateFull || dgate->dtype != t))
            return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward: dgate must be ST_F32, or the branch's type where "
                                                 "the gate is [rows, cols]");
    }
    const uint64_t need = static_cast<uint64_t>(residual_norm_backward_workspace(g.rows, g.cols));
    const bool sums = dpost || dpre || g.gate_mode == kGateChannel;
    if (sums && g.rows > 0 && (!workspace || workspace_bytes < need))
        return fail(ST_ERR_INVALID_ARGUMENT, "residual_norm_backward needs a workspace of " + std::to_string(need) + " bytes");
    if (sums && g.rows > 0 && !aligned16(workspace)) return fail(ST_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(launch_residual_norm_backward(g, workspace, x.dev->dev_err, kDeviceWaitLimitNs, x.stream));
    return finish(x);
}

int st_check_device_wait(st_ctx *ctx, int32_t kind, uint32_t limit_us, const st_exec *exec) {
    if (kind != 0 && kind != 1 && (kind < 16 || kind > 18))
        return fail(ST_ERR_INVALID_ARGUMENT, "st_check_device_wait: kind must be 0 (mbarrier), 1 (flag), 16 (row ring of the "
                                             "norms), 17 or 18 (scaling warp of the 8-bit product, by rows or by columns)");
    if (limit_us == 0 || limit_us > 10u * 1000 * 1000)
        return fail(ST_ERR_INVALID_ARGUMENT, "st_check_device_wait: limit_us must be in [1, 10^7]");
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    DeviceGuard guard(x.dev->ordinal);
    const uint64_t limit_ns = static_cast<uint64_t>(limit_us) * 1000;
    if (kind < 16) ST_TRY(launch_wait_check(kind, limit_ns, x.dev->dev_err, x.stream));
    else if (kind == 16) ST_TRY(launch_norm_wait_check(limit_ns, x.dev->dev_err, x.stream));
    else ST_TRY(launch_fp8_wait_check(kind == 18, limit_ns, x.dev->dev_err, x.stream));
    return finish(x);
}

int st_cast(st_ctx *ctx, const st_tensor *a, const st_tensor *c, const st_exec *exec) {
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    if (!a || !c) return fail(ST_ERR_INVALID_ARGUMENT, "cast: null tensor");
    if (c->rank != 1 && c->rank != 2) return fail(ST_ERR_INVALID_ARGUMENT, "cast: tensors must be rank 1 or 2");
    ST_TRY(check_view(a, "A", c->rank));
    ST_TRY(check_view(c, "C", c->rank));
    for (const st_tensor *t : {a, c})
        if (t->dtype != ST_F32 && t->dtype != ST_F16 && t->dtype != ST_BF16)
            return fail(ST_ERR_INVALID_ARGUMENT, "cast: tensors must be ST_F32, ST_F16 or ST_BF16");
    for (int i = 0; i < c->rank; ++i)
        if (a->shape[i] != c->shape[i]) return fail(ST_ERR_INVALID_ARGUMENT, "cast: A and C must have the same shape");
    DeviceGuard guard(x.dev->ordinal);
    const int64_t rows = c->rank == 2 ? c->shape[0] : 1;
    const int64_t cols = c->rank == 2 ? c->shape[1] : c->shape[0];
    const int64_t sa[2] = {a->rank == 1 ? cols : a->strides[0], a->rank == 1 ? a->strides[0] : a->strides[1]};
    const int64_t sc[2] = {c->rank == 1 ? cols : c->strides[0], c->rank == 1 ? c->strides[0] : c->strides[1]};
    ST_TRY(launch_cast(a->data, a->dtype, sa, c->data, c->dtype, sc, rows, cols, x.dev->sm_count, x.stream));
    return finish(x);
}

int st_vector_add_host(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *c, const st_exec *exec) {
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x, true));
    ST_TRY(check_vector_add(a, b, c));
    if (x.flags & ST_EXEC_ALL_DEVICES) {
        ST_TRY(check_all_devices(exec));
        return vector_add_host_split(ctx, x, *a, *b, *c);
    }
    DeviceGuard guard(x.dev->ordinal);
    return vector_add_host_one(x, *a, *b, *c, true);
}

int st_matmul_host(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *bias, const st_tensor *c,
                   const st_exec *exec) {
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x, true));
    ST_TRY(check_matmul(a, b, bias, c));
    if (x.flags & ST_EXEC_ALL_DEVICES) {
        ST_TRY(check_all_devices(exec));
        return matmul_host_split(ctx, x, *a, *b, bias, *c);
    }
    DeviceGuard guard(x.dev->ordinal);
    return matmul_host_one(x, *a, *b, bias, *c, true);
}

int st_ipc_handle(st_ctx *ctx, int32_t device, void *ptr, uint8_t handle[64]) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    if (!ptr || !handle) return fail(ST_ERR_INVALID_ARGUMENT, "st_ipc_handle: null pointer");
    static_assert(sizeof(cudaIpcMemHandle_t) == 64, "IPC handle size");
    DeviceGuard guard(d->ordinal);
    cudaIpcMemHandle_t h;
    ST_CUDA_TRY(cudaIpcGetMemHandle(&h, ptr));
    std::memcpy(handle, &h, 64);
    return ST_OK;
}

int st_ipc_open(st_ctx *ctx, int32_t device, const uint8_t handle[64], void **out) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    if (!handle || !out) return fail(ST_ERR_INVALID_ARGUMENT, "st_ipc_open: null pointer");
    DeviceGuard guard(d->ordinal);
    cudaIpcMemHandle_t h;
    std::memcpy(&h, handle, 64);
    ST_CUDA_TRY(cudaIpcOpenMemHandle(out, h, cudaIpcMemLazyEnablePeerAccess));
    return ST_OK;
}

int st_ipc_close(st_ctx *ctx, int32_t device, void *ptr) {
    DeviceState *d;
    ST_TRY(get_dev(ctx, device, &d));
    DeviceGuard guard(d->ordinal);
    if (ptr) ST_CUDA_TRY(cudaIpcCloseMemHandle(ptr));
    return ST_OK;
}

int st_matmul_allgather(st_ctx *ctx, const st_tensor *a, const st_tensor *b, const st_tensor *bias,
                        const st_tensor *c_full, void *const *peer_c_full, int32_t n_peers, int64_t row_offset,
                        const st_exec *exec) {
    ExecCtx x;
    ST_TRY(resolve_exec(ctx, exec, &x));
    if (!a || !c_full) return fail(ST_ERR_INVALID_ARGUMENT, "st_matmul_allgather: null tensor");
    ST_TRY(check_view(c_full, "C", 2));
    if (n_peers < 0 || n_peers > kMaxPeers || (n_peers > 0 && !peer_c_full))
        return fail(ST_ERR_INVALID_ARGUMENT, "st_matmul_allgather: between 0 and 7 peer copies of C");
    if (row_offset < 0 || a->rank != 2 || row_offset + a->shape[0] > c_full->shape[0])
        return fail(ST_ERR_INVALID_ARGUMENT, "st_matmul_allgather: A's rows must fall inside C at row_offset");
    // this rank's rows of C, and the same rows in each peer's copy
    const size_t es = dtype_size(c_full->dtype);
    const size_t byte_off = static_cast<size_t>(row_offset) * static_cast<size_t>(c_full->strides[0]) * es;
    st_tensor c_rows = *c_full;
    c_rows.shape[0] = a->shape[0];
    c_rows.data = static_cast<uint8_t *>(c_full->data) + byte_off;
    ST_TRY(check_matmul(a, b, bias, &c_rows));
    PeerOutputs peers;
    peers.n = n_peers;
    for (int i = 0; i < n_peers; ++i) {
        if (!peer_c_full[i]) return fail(ST_ERR_INVALID_ARGUMENT, "st_matmul_allgather: null peer pointer");
        peers.base[i] = static_cast<uint8_t *>(peer_c_full[i]) + byte_off;
    }
    DeviceGuard guard(x.dev->ordinal);
    ST_TRY(matmul_device(x, *a, *b, bias, c_rows, &peers));
    return finish(x);
}

int st_shard_range(int64_t total, int32_t count, int32_t rank, int64_t align, int64_t *begin, int64_t *end) {
    if (total < 0 || count < 1 || rank < 0 || rank >= count || align < 1 || !begin || !end)
        return fail(ST_ERR_INVALID_ARGUMENT, "st_shard_range: need total >= 0, 0 <= rank < count, align >= 1");
    const int64_t units = cdiv(total, align);
    const int64_t b = units * rank / count, e = units * (rank + 1) / count;
    *begin = std::min(b * align, total);
    *end = std::min(e * align, total);
    return ST_OK;
}

}  // extern "C"
