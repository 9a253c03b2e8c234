"""8-bit blocks and their matrix product on CUDA tensors.

``quantize_fp8`` makes 8-bit blocks of 128 with one float32 scale each,
``matmul_fp8`` multiplies them.  A layer y = x @ W.t(), its gradients among
its calls:

    Wq, Ws = quantize_fp8(W, block=(128, 128))             # W [N, K], once
    xq, xs = quantize_fp8(x)                               # x [M, K], blocks of 1 x 128
    y = matmul_fp8(xq, Wq.t(), xs, Ws.t())

    gq, gs = quantize_fp8(dy, dtype=torch.float8_e5m2)     # dx = dy @ W: W as it is stored
    dx = matmul_fp8(gq, Wq, gs, Ws)
    gq, gs = quantize_fp8(dy, block=(128, 1))              # dW = dy.t() @ x: blocks along the tokens
    xq, xs = quantize_fp8(x, block=(128, 1))
    dW = matmul_fp8(gq.t(), xq, gs.t(), xs, out_dtype=torch.float32)

Neither call takes part in autograd.  Both run on torch's current stream of
the tensors' device, keep nothing between calls and can be captured into a
CUDA graph.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .api import _CODES, _TENSOR_DESC, _exec_desc
from .runtime import context

BLOCK = 128
_BLOCKS = ((1, BLOCK), (BLOCK, 1), (BLOCK, BLOCK))
_FP8 = {torch.float8_e4m3fn: N.ST_E4M3, torch.float8_e5m2: N.ST_E5M2}
_ALL_CODES = {**_CODES, **_FP8}

_vp, _cp, _i32, _u64 = ctypes.c_void_p, ctypes.c_char_p, ctypes.c_int32, ctypes.c_uint64
_pack = _TENSOR_DESC.pack
_fns: dict = {}


def _fn(name: str, *args):
    """`name` from the native library; descriptors are passed as packed bytes."""
    fn = _fns[name] = ctypes.CFUNCTYPE(ctypes.c_int, *args)((name, N.lib()))
    return fn


def _desc(t: torch.Tensor) -> bytes:
    """The st_tensor descriptor of `t`, 8-bit types among them."""
    shape, strides = t.shape, t.stride()
    code = _ALL_CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {t.dtype}")
    if len(shape) == 2:
        r, c = shape
        return _pack(t.data_ptr() if r and c else 0, code, 2, r, c, *strides)
    if len(shape) == 1:
        return _pack(t.data_ptr() if shape[0] else 0, code, 1, shape[0], 0, strides[0], 0)
    raise ValueError("tensors must be rank 1 or 2")


def _device_of(*tensors: torch.Tensor | None) -> int:
    """The one CUDA device of every tensor given."""
    dev = None
    for t in tensors:
        if t is None:
            continue
        d = t.get_device()
        if d != dev:
            if d < 0:
                raise ValueError("Input tensors must be on a CUDA device.")
            if dev is not None:
                raise ValueError("Input tensors must be on the same CUDA device.")
            dev = d
    return dev


# Outputs are made and described at once: their shapes and strides are known,
# and a call's host time is mostly that of its tensors.
def _new(like: torch.Tensor, rows: int, cols: int, s0: int, s1: int, dtype: torch.dtype) -> tuple[torch.Tensor, bytes]:
    t = like.new_empty_strided((rows, cols), (s0, s1), dtype=dtype)
    return t, _pack(t.data_ptr(), _ALL_CODES[dtype], 2, rows, cols, s0, s1)


def _new_codes(like: torch.Tensor, rows: int, cols: int, dtype: torch.dtype) -> tuple[torch.Tensor, bytes]:
    """[rows, cols] 8-bit codes, each row on a 16-byte boundary, where the tensor core's loads can start."""
    return _new(like, rows, cols, (cols + 15) // 16 * 16, 1, dtype)


def _new_scales(like: torch.Tensor, rows: int, cols: int, block_rows: int, block_cols: int) -> tuple[torch.Tensor, bytes]:
    """One scale per block, lying along the rows (columns) that have one each, as the product reads them."""
    r, c = -(-rows // block_rows), -(-cols // block_cols)
    return _new(like, r, c, 1, r, torch.float32) if block_rows == 1 else _new(like, r, c, c, 1, torch.float32)


def quantize_fp8(A: torch.Tensor, *, block: tuple[int, int] = (1, BLOCK), dtype: torch.dtype = torch.float8_e4m3fn,
                 out: torch.Tensor | None = None, scale_out: torch.Tensor | None = None
                 ) -> tuple[torch.Tensor, torch.Tensor]:
    """(Q, scale): A (rank 2; float32, float16 or bfloat16; any strides) as 8-bit blocks.

    For each block, (1, 128), (128, 1) or (128, 128), cut at A's edges:
    scale = max(max|a| / limit, 2^-126), Q = fp8(a * (1 / scale)) rounded to
    nearest even, with limit 448 for float8_e4m3fn and 57344 for float8_e5m2.
    scale is float32 [ceil(rows / block[0]), ceil(cols / block[1])].  Q is
    laid out in A's order (by rows, or by columns for a transposed A) on
    16-byte boundaries, so it need not be contiguous.  A block with a NaN or
    an infinity gets a scale that is one, and a product that reads it is NaN.
    """
    shape = A.shape
    if len(shape) != 2:
        raise ValueError("A must be a 2D tensor.")
    block = tuple(block)
    if block not in _BLOCKS:
        raise ValueError(f"block must be one of {_BLOCKS}, got {block}")
    if dtype not in _FP8:
        raise ValueError(f"dtype must be torch.float8_e4m3fn or torch.float8_e5m2, got {dtype}")
    dev = _device_of(A, out, scale_out)
    rows, cols = shape
    if out is None:
        s0, s1 = A.stride()
        if s0 == 1 and s1 != 1 and cols > 1:
            out, dq = _new(A, rows, cols, 1, (rows + 15) // 16 * 16, dtype)
        else:
            out, dq = _new_codes(A, rows, cols, dtype)
    else:
        if out.dtype != dtype:
            raise ValueError(f"out must have dtype {dtype}, got {out.dtype}")
        dq = _desc(out)
    if scale_out is None:
        scale_out, ds = _new_scales(A, rows, cols, *block)
    else:
        ds = _desc(scale_out)
    fn = _fns.get("st_quantize_fp8") or _fn("st_quantize_fp8", _vp, _cp, _cp, _cp, _i32, _i32, _cp)
    rc = fn(context(dev), _desc(A), dq, ds, block[0], block[1], _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "quantize_fp8")
    return out, scale_out


def matmul_fp8(A: torch.Tensor, B: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
               bias: torch.Tensor | None = None, *, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """C = A @ B (+ bias) for 8-bit A [M, K] and B [K, N] with a scale for each block of 128 along K.

    A, B: float8_e4m3fn or float8_e5m2, each of its own type and any strides
    (rows or columns on 16-byte boundaries, as quantize_fp8 lays them out,
    are read in place; anything else is copied first).  a_scale: float32
    [M, ceil(K/128)], or [ceil(M/128), ceil(K/128)] with one scale for 128
    rows; b_scale: float32 [ceil(K/128), N] or [ceil(K/128), ceil(N/128)];
    any strides.  Products are summed in fp32, block by block, and a block's
    sum is multiplied by a_scale * b_scale in fp32: keep that product within
    2^-126 and 2^128 (a block of zeros gives 0 whatever its scale).  C is
    bfloat16, float16 or float32; bias (length N) is float32 or C's dtype.
    The same inputs give the same bits.
    """
    sa, sb = A.shape, B.shape
    if len(sa) != 2 or len(sb) != 2:
        raise ValueError("A and B must be 2D tensors.")
    if sa[1] != sb[0]:
        raise ValueError(f"Incompatible matrices: K dimension of A ({sa[1]}) "
                         f"must match K dimension of B ({sb[0]})")
    dev = _device_of(A, B, a_scale, b_scale, bias, out)
    if out is None:
        if out_dtype not in _CODES:
            raise ValueError(f"unsupported dtype {out_dtype}")
        out, dc = _new(A, sa[0], sb[1], max(sb[1], 1), 1, out_dtype)
    else:
        dc = _desc(out)
    da, db = _desc(A), _desc(B)
    workspace, need = None, 0
    # operands that the tensor core's loads cannot address in place are copied: ask how much room that takes
    (a0, a1), (b0, b1) = A.stride(), B.stride()
    if not ((a1 == 1 and a0 % 16 == 0 and a0 >= sa[1] or a0 == 1 and a1 % 16 == 0 and a1 >= sa[0]) and
            (b1 == 1 and b0 % 16 == 0 and b0 >= sb[1] or b0 == 1 and b1 % 16 == 0 and b1 >= sb[0]) and
            (A.data_ptr() | B.data_ptr()) % 16 == 0):
        size = ctypes.c_uint64(0)
        fn = _fns.get("st_matmul_fp8_workspace") or _fn("st_matmul_fp8_workspace", _cp, _cp, _vp)
        rc = fn(da, db, ctypes.addressof(size))
        if rc != N.ST_OK:
            N.check(rc, "matmul_fp8")
        need = size.value
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=A.device)
    fn = _fns.get("st_matmul_fp8") or _fn("st_matmul_fp8", _vp, _cp, _cp, _cp, _cp, _cp, _cp, _vp, _u64, _cp)
    rc = fn(context(dev), da, db, _desc(a_scale), _desc(b_scale), None if bias is None else _desc(bias), dc,
            None if workspace is None else workspace.data_ptr(), need, _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "matmul_fp8")
    return out
