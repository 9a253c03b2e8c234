"""4-bit blocks and their matrix product on CUDA tensors.

``quantize_fp4`` makes 4-bit blocks of 16 or 32 elements with one 8-bit scale
each, ``matmul_fp4`` multiplies them on the tensor cores, ``dequantize_fp4``
gives the values back.  A layer y = x @ W.t(), its gradients among its calls:

    W4 = quantize_fp4(W)                                   # W [N, K], once per update
    x4 = quantize_fp4(x)                                   # x [M, K]
    y = matmul_fp4(x4.codes, W4.codes.t(), x4.scale, W4.scale,
                   a_tensor_scale=x4.tensor_scale, b_tensor_scale=W4.tensor_scale)

    g4, V4 = quantize_fp4(dy), quantize_fp4(W.t())         # dx = dy @ W: blocks along N
    g4, u4 = quantize_fp4(dy.t()), quantize_fp4(x.t())     # dW = dy.t() @ x: blocks along the tokens

An element is e2m1: 0, 0.5, 1, 1.5, 2, 3, 4, 6 or one of their negatives, two
of them a byte along a row.  Neither call takes part in autograd.  All run on
torch's current stream of the tensors' device, keep nothing between calls and
can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import functools
from typing import NamedTuple

import torch

from . import _native as N
from .api import _CODES, _exec_desc
from .fp8 import _cp, _desc, _device_of, _fn, _fns, _new, _pack, _u64, _vp
from .runtime import context

_BLOCK = {torch.float8_e4m3fn: 16}
_SCALE_CODES = {torch.float8_e4m3fn: N.ST_E4M3}
# An older torch lacks the two types: codes are uint8 there, and blocks of 32 are not to be had.
if hasattr(torch, "float8_e8m0fnu"):
    _BLOCK[torch.float8_e8m0fnu] = 32
    _SCALE_CODES[torch.float8_e8m0fnu] = N.ST_E8M0
_CODES_TYPE = getattr(torch, "float4_e2m1fn_x2", torch.uint8)


class Quantized4(NamedTuple):
    codes: torch.Tensor                # float4_e2m1fn_x2 [rows, ceil(cols / 2)] (uint8 with a torch that lacks the type)
    scale: torch.Tensor                # [ceil(rows / 128), ceil(blocks / 4), 32, 4, 4], see quantize_fp4
    tensor_scale: torch.Tensor | None  # float32, one element (None for blocks of 32)


def _codes_desc(t: torch.Tensor, name: str) -> bytes:
    if t.dtype != _CODES_TYPE and t.dtype != torch.uint8:
        raise ValueError(f"{name} must have dtype torch.float4_e2m1fn_x2 (or torch.uint8), got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be a 2D tensor.")
    r, c = t.shape
    return _pack(t.data_ptr() if r and c else 0, N.ST_E2M1X2, 2, r, c, *t.stride())


def _scale_shape(rows: int, code_bytes: int, block: int) -> tuple[int, ...]:
    return (-(-rows // 128), -(-(-(-2 * code_bytes // block)) // 4), 32, 4, 4)


def _scale_desc(t: torch.Tensor, name: str, rows: int, code_bytes: int) -> bytes:
    block = _BLOCK.get(t.dtype)
    if block is None:
        raise ValueError(f"{name} must have dtype torch.float8_e4m3fn (blocks of 16) or torch.float8_e8m0fnu (of 32), "
                         f"got {t.dtype}")
    shape = _scale_shape(rows, code_bytes, block)
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous {list(shape)}, got {list(t.shape)} with strides {list(t.stride())}")
    n = t.numel()
    return _pack(t.data_ptr() if n else 0, _SCALE_CODES[t.dtype], 1, n, 0, 1, 0)


def _scalar_desc(t: torch.Tensor | None, name: str) -> bytes | None:
    if t is None:
        return None
    if t.dtype != torch.float32 or t.numel() != 1:
        raise ValueError(f"{name} must be one float32, got {t.dtype} {list(t.shape)}")
    return _pack(t.data_ptr(), N.ST_F32, 1, 1, 0, 1, 0)


@functools.lru_cache(maxsize=1)
def _quantize_workspace() -> int:
    size = ctypes.c_uint64(0)
    N.check(N.lib().st_quantize_fp4_workspace(ctypes.byref(size)), "quantize_fp4")
    return size.value


def quantize_fp4(A: torch.Tensor, *, scale_dtype: torch.dtype = torch.float8_e4m3fn, amax: torch.Tensor | None = None
                 ) -> Quantized4:
    """A (rank 2; float32, float16 or bfloat16; any strides) as 4-bit blocks along its rows.

    scale_dtype float8_e4m3fn, blocks of 16: tensor_scale is the least power
    of two t >= 2^-126 with 2688 t >= amax, a block's scale is
    e4m3(max|a| / (6 t)), its codes e2m1(a / (scale t)).  ``amax`` (one
    float32 on the device) is the largest |a| to provide for, larger elements
    saturate with their sign, however large (0, an infinity or a NaN makes the
    tensor_scale 1); left out, it is taken from A's finite elements in a first pass.
    scale_dtype float8_e8m0fnu, blocks of 32: a block's scale is the least
    power of two >= 2^-127 with 6 scale >= max|a|, its codes e2m1(a / scale).

    Rounding is to nearest even; the codes are the same on any machine that
    rounds the quotients correctly.  A block with a NaN or an infinity gets
    the scale NaN, and a product that reads it is NaN.

    codes [rows, ceil(cols / 2)] holds two elements a byte, the first in the
    low half, rows on 16-byte boundaries (so it need not be contiguous).
    scale[i, j, r, q, b] belongs to row 128 i + 32 q + r and block 4 j + b, the
    order in which the tensor cores take it, and is 0 where that row or block
    does not exist.
    """
    if A.dim() != 2:
        raise ValueError("A must be a 2D tensor.")
    block = _BLOCK.get(scale_dtype)
    if block is None:
        raise ValueError(f"scale_dtype must be torch.float8_e4m3fn or torch.float8_e8m0fnu, got {scale_dtype}")
    if amax is not None and block == 32:
        raise ValueError("amax goes with scale_dtype torch.float8_e4m3fn")
    da = _desc(A)
    dev = _device_of(A, amax)
    rows, cols = A.shape
    width = (cols + 1) // 2
    pitch = (width + 15) // 16 * 16
    codes = A.new_empty_strided((rows, width), (pitch, 1), dtype=_CODES_TYPE)
    scale = A.new_empty(_scale_shape(rows, width, block), dtype=scale_dtype)
    n = scale.numel()
    t = workspace = None
    need = 0
    if block == 16:
        t = A.new_empty_strided((), (), dtype=torch.float32)
        if amax is None:
            need = _quantize_workspace()
            workspace = A.new_empty_strided((need,), (1,), dtype=torch.uint8)
    fn = _fns.get("st_quantize_fp4") or _fn("st_quantize_fp4", _vp, _cp, _cp, _cp, _cp, _cp, _vp, _u64, _cp)
    rc = fn(context(dev), da, _pack(codes.data_ptr() if rows and cols else 0, N.ST_E2M1X2, 2, rows, width, pitch, 1),
            _pack(scale.data_ptr() if n else 0, _SCALE_CODES[scale_dtype], 1, n, 0, 1, 0), _scalar_desc(amax, "amax"),
            _scalar_desc(t, "tensor_scale"), None if workspace is None else workspace.data_ptr(), need, _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "quantize_fp4")
    return Quantized4(codes, scale, t)


def dequantize_fp4(codes: torch.Tensor, scale: torch.Tensor, tensor_scale: torch.Tensor | None = None, *,
                   cols: int | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of 4-bit blocks: code * scale * tensor_scale, rounded to fp32 and that to out_dtype.

    (In fp32 it is exact where tensor_scale is a power of two, as quantize_fp4
    makes it, and the result lies in fp32's normal range.)  codes, scale and
    tensor_scale as quantize_fp4 makes them, or any other tensor scale (codes
    of any strides; uint8 is taken as well); ``cols`` where the last byte of a
    row holds one element only.
    """
    dq = _codes_desc(codes, "codes")
    if out_dtype not in _CODES:
        raise ValueError(f"unsupported dtype {out_dtype}")
    rows, width = codes.shape
    if cols is None:
        cols = 2 * width
    elif (cols + 1) // 2 != width:
        raise ValueError(f"cols must be {2 * width} or one less, got {cols}")
    ds, dt = _scale_desc(scale, "scale", rows, width), _scalar_desc(tensor_scale, "tensor_scale")
    dev = _device_of(codes, scale, tensor_scale)
    out, do = _new(scale, rows, cols, max(cols, 1), 1, out_dtype)
    fn = _fns.get("st_dequantize_fp4") or _fn("st_dequantize_fp4", _vp, _cp, _cp, _cp, _cp, _cp)
    rc = fn(context(dev), dq, ds, dt, do, _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "dequantize_fp4")
    return out


def matmul_fp4(A: torch.Tensor, B: torch.Tensor, a_scale: torch.Tensor, b_scale: torch.Tensor,
               bias: torch.Tensor | None = None, *, a_tensor_scale: torch.Tensor | None = None,
               b_tensor_scale: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """C = A @ B (+ bias) for 4-bit A [M, K] and B [K, N] with scales along K, as quantize_fp4 makes them.

    A [M, K/2] and B [K/2, N] are codes (B the transposed view of what
    quantize_fp4 made of [N, K]); rows of A and columns of B on 16-byte
    boundaries are read in place, anything else is copied first.  a_scale and
    b_scale have one dtype, which says the blocks' length; entries of theirs
    that belong to no block must be 0 (or at least finite).  The sum is fp32;
    it is multiplied by a_tensor_scale * b_tensor_scale (by one after the other
    where that product leaves fp32's normal range), the bias (length N; float32
    or C's dtype) is added, and the result rounded once to C's dtype, bfloat16,
    float16 or float32.  The same inputs give the same bits.
    """
    da, db = _codes_desc(A, "A"), _codes_desc(B, "B")
    (m, ka), (kb, n) = A.shape, B.shape
    if ka != kb:
        raise ValueError(f"Incompatible matrices: K dimension of A ({ka} bytes) must match K dimension of B ({kb})")
    dsa, dsb = _scale_desc(a_scale, "a_scale", m, ka), _scale_desc(b_scale, "b_scale", n, kb)
    dta, dtb = _scalar_desc(a_tensor_scale, "a_tensor_scale"), _scalar_desc(b_tensor_scale, "b_tensor_scale")
    dev = _device_of(A, B, a_scale, b_scale, bias, a_tensor_scale, b_tensor_scale, out)
    if out is None:
        if out_dtype not in _CODES:
            raise ValueError(f"unsupported dtype {out_dtype}")
        out, dc = _new(a_scale, m, n, max(n, 1), 1, out_dtype)
    else:
        dc = _desc(out)
    workspace, need = None, 0
    (a0, a1), (b0, b1) = A.stride(), B.stride()
    if not (a1 == 1 and a0 % 16 == 0 and a0 >= ka and b0 == 1 and b1 % 16 == 0 and b1 >= kb and
            (A.data_ptr() | B.data_ptr()) % 16 == 0):
        size = ctypes.c_uint64(0)
        fn = _fns.get("st_matmul_fp4_workspace") or _fn("st_matmul_fp4_workspace", _cp, _cp, _vp)
        rc = fn(da, db, ctypes.addressof(size))
        if rc != N.ST_OK:
            N.check(rc, "matmul_fp4")
        need = size.value
        if need:
            workspace = torch.empty(need, dtype=torch.uint8, device=A.device)
    fn = _fns.get("st_matmul_fp4") or _fn("st_matmul_fp4", _vp, _cp, _cp, _cp, _cp, _cp, _cp, _cp, _cp, _vp, _u64, _cp)
    rc = fn(context(dev), da, db, dsa, dsb, dta, dtb, None if bias is None else _desc(bias), dc,
            None if workspace is None else workspace.data_ptr(), need, _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "matmul_fp4")
    return out
