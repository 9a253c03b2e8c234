"""The norms after and before a block, fused with its gate and residual scale.

Between two blocks of a network a residual stream takes the last block's
output in and hands a normed copy of itself to the next:

    u        = x * rsqrt(mean(x^2) + eps) * (post_weight + weight_offset)
    residual = residual + alpha * gate * u
    normed   = residual * rsqrt(mean(residual^2) + eps) * (pre_weight + weight_offset)

``residual_norm`` does it in one pass, ``residual_norm_backward`` takes the
gradients back.  Either norm and the gate can be left out: with x None it is
the norm before the first block, without pre_weight the one after the last.
The normed copy can leave as 8-bit blocks for matmul_fp8.  Neither call takes
part in autograd; both run on torch's current stream of the tensors' device,
keep nothing between calls and can be captured into a CUDA graph.
"""
from __future__ import annotations

import ctypes
import functools
import struct
from typing import NamedTuple

import torch

from . import _native as N
from .api import _exec_desc
from .fp8 import (_ALL_CODES, _FP8, BLOCK, _cp, _desc, _device_of, _fn, _fns, _new, _new_codes, _new_scales, _pack, _u64,
                  _vp)
from .runtime import context

_OPTIONS = struct.Struct("@fff")  # alpha, eps, weight_offset
assert _OPTIONS.size == ctypes.sizeof(N.StNormOptions)


class ResidualNorm(NamedTuple):
    residual: torch.Tensor        # the updated stream
    normed: torch.Tensor | None   # for the next block (None without pre_weight)
    scale: torch.Tensor | None    # float32 [rows, ceil(cols / 128)] where normed is 8-bit


class ResidualNormGrads(NamedTuple):
    x: torch.Tensor | None
    residual: torch.Tensor
    post_weight: torch.Tensor | None  # float32 [cols]
    gate: torch.Tensor | None         # the gate's shape; float32, or the gate's dtype where it is [rows, cols]
    pre_weight: torch.Tensor | None   # float32 [cols]


def _new_sums(like: torch.Tensor, cols: int) -> tuple[torch.Tensor, bytes]:
    t = like.new_empty_strided((cols,), (1,), dtype=torch.float32)
    return t, _pack(t.data_ptr(), N.ST_F32, 1, cols, 0, 1, 0)


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(rows: int, cols: int) -> int:
    """What residual_norm_backward needs for its sums over rows: a function of the extents alone."""
    size = ctypes.c_uint64(0)
    N.check(N.lib().st_residual_norm_backward_workspace(rows, cols, ctypes.byref(size)), "residual_norm_backward")
    return size.value


def _opt(t: torch.Tensor | None) -> bytes | None:
    return None if t is None else _desc(t)


def residual_norm(x: torch.Tensor | None, residual: torch.Tensor, post_weight: torch.Tensor | None = None,
                  gate: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None, *, alpha: float = 1.0,
                  eps: float = 1e-6, weight_offset: float = 0.0, quantize: bool | torch.dtype = False,
                  out_dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> ResidualNorm:
    """The updated residual stream and its normed copy (see the module).

    x, residual: [rows, cols] with unit column stride, at most 16384 columns;
    x float32, float16 or bfloat16, residual of x's dtype or float32 (the
    updated stream keeps residual's dtype).  post_weight, pre_weight: [cols];
    gate: [cols] or [1, cols] (a channel's), [rows, 1] (a token's) or
    [rows, cols]; each float32 or x's dtype.  normed has x's dtype (without
    x: out_dtype or residual's dtype) and is computed from the stream before
    its rounding.  quantize: True or an 8-bit dtype for normed as 8-bit
    blocks of 1 x 128, as quantize_fp8 makes them (True: float8_e4m3fn).
    out: where the updated stream goes; ``residual`` itself is allowed.
    """
    shape = residual.shape
    if len(shape) != 2:
        raise ValueError("residual must be a 2D tensor.")
    if residual.dtype not in _ALL_CODES:
        raise ValueError(f"unsupported dtype {residual.dtype}")
    dev = _device_of(residual, x, post_weight, gate, pre_weight, out)
    rows, cols = shape
    d_out = d_normed = d_scale = normed = scale = None
    if x is None:
        if out is not None:
            raise ValueError("out is the updated stream: without x there is none")
    elif out is None:
        out, d_out = _new(residual, rows, cols, max(cols, 1), 1, residual.dtype)
    else:
        d_out = _desc(out)
    if x is not None and out_dtype is not None and out_dtype != x.dtype:
        raise ValueError(f"out_dtype {out_dtype} differs from x's dtype {x.dtype}")
    if pre_weight is not None:
        if quantize:
            kind = torch.float8_e4m3fn if quantize is True else quantize
            if kind not in _FP8:
                raise ValueError(f"quantize must be torch.float8_e4m3fn or torch.float8_e5m2, got {kind}")
            normed, d_normed = _new_codes(residual, rows, cols, kind)
            scale, d_scale = _new_scales(residual, rows, cols, 1, BLOCK)
        else:
            dtype = x.dtype if x is not None else out_dtype or residual.dtype
            if dtype not in _ALL_CODES:
                raise ValueError(f"unsupported dtype {dtype}")
            normed, d_normed = _new(residual, rows, cols, max(cols, 1), 1, dtype)
    elif quantize:
        raise ValueError("quantize is for the normed copy: it needs pre_weight")
    fn = _fns.get("st_residual_norm") or _fn("st_residual_norm", _vp, *[_cp] * 10)
    rc = fn(context(dev), None if x is None else _desc(x), _desc(residual),
            None if post_weight is None else _desc(post_weight), None if gate is None else _desc(gate),
            None if pre_weight is None else _desc(pre_weight), d_out, d_normed, d_scale,
            _OPTIONS.pack(alpha, eps, weight_offset), _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "residual_norm")
    return ResidualNorm(residual if out is None else out, normed, scale)


def residual_norm_backward(d_residual: torch.Tensor | None, d_normed: torch.Tensor | None, x: torch.Tensor | None,
                           residual: torch.Tensor | None, post_weight: torch.Tensor | None = None,
                           gate: torch.Tensor | None = None, pre_weight: torch.Tensor | None = None, *,
                           alpha: float = 1.0, eps: float = 1e-6, weight_offset: float = 0.0) -> ResidualNormGrads:
    """The gradients of residual_norm.

    d_residual, d_normed: gradients of the two outputs (one may be None;
    d_normed is the gradient of the unquantized copy, there exactly if
    pre_weight is).  x, post_weight, gate, pre_weight, alpha, eps and
    weight_offset as in the forward call; ``residual`` is the updated stream
    that it returned (needed with pre_weight).  Gradients of x and residual
    have their dtypes; sums over rows are float32.
    """
    like = d_residual if d_residual is not None else d_normed
    if like is None:
        raise ValueError("one of d_residual and d_normed must be given")
    shape = like.shape
    if len(shape) != 2:
        raise ValueError("gradients must be 2D tensors.")
    dev = _device_of(like, d_normed, x, residual, post_weight, gate, pre_weight)
    rows, cols = shape
    stream = residual if residual is not None else like
    pitch = max(cols, 1)
    for t in (stream, x):
        if t is not None and t.dtype not in _ALL_CODES:
            raise ValueError(f"unsupported dtype {t.dtype}")
    dr, d_dr = _new(like, rows, cols, pitch, 1, stream.dtype)
    dx, d_dx = (None, None) if x is None else _new(like, rows, cols, pitch, 1, x.dtype)
    dpost = dpre = dgate = d_dpost = d_dpre = d_dgate = None
    if post_weight is not None:
        dpost, d_dpost = _new_sums(like, cols)
    if pre_weight is not None:
        dpre, d_dpre = _new_sums(like, cols)
    if gate is not None:
        if gate.dim() == 1:
            dgate, d_dgate = _new_sums(like, gate.shape[0])
        elif gate.dim() == 2:
            g0, g1 = gate.shape
            if gate.dtype not in _ALL_CODES:
                raise ValueError(f"unsupported dtype {gate.dtype}")
            dgate, d_dgate = _new(like, g0, g1, max(g1, 1), 1, gate.dtype if g0 == rows and g1 == cols else torch.float32)
        else:
            raise ValueError("gate must be rank 1 or 2")
    size = _workspace_bytes(rows, cols)
    workspace = like.new_empty_strided((size,), (1,), dtype=torch.uint8)
    fn = _fns.get("st_residual_norm_backward") or _fn("st_residual_norm_backward", _vp, *[_cp] * 12, _vp, _u64, _cp, _cp)
    rc = fn(context(dev), _opt(d_residual), _opt(d_normed), _opt(x), _opt(residual), _opt(post_weight), _opt(gate),
            _opt(pre_weight), d_dx, d_dr, d_dpost, d_dgate, d_dpre, workspace.data_ptr(), size,
            _OPTIONS.pack(alpha, eps, weight_offset), _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "residual_norm_backward")
    return ResidualNormGrads(dx, dr, dpost, dgate, dpre)
