"""Matrix products by groups of rows on CUDA tensors: layers whose tokens meet different weights.

Tokens sorted by the expert that they go to are rows of one matrix; group g is
rows [ends[g - 1], ends[g]), and meets the g-th of a stack of matrices.  A
layer y = x @ W[g].t() of experts W [G, N, K], its gradients among its calls:

    y = matmul_grouped(x, W.transpose(1, 2), ends)          # x [T, K]
    dx = matmul_grouped(dy, W, ends)                        # W as it is stored
    dW = matmul_grouped_weights(dy, x, ends, out_dtype=torch.float32)      # [G, N, K]

The ends stay on the device: no call waits for them, so a router's result can
be used as it comes, and a captured CUDA graph serves any division of the
rows.  Neither call takes part in autograd.  Both run on torch's current
stream of the tensors' device and keep nothing between calls.
"""
from __future__ import annotations

import ctypes

import torch

from . import _native as N
from .api import _CODES, _exec_desc
from .fp8 import _cp, _desc, _device_of, _fn, _fns, _i32, _new, _pack, _u64, _vp
from .runtime import context

_i64 = ctypes.c_int64


def _ends_desc(ends: torch.Tensor) -> bytes:
    if ends.dtype != torch.int32 or ends.dim() != 1:
        raise ValueError(f"ends must be a 1D tensor of int32, got {ends.dtype} of rank {ends.dim()}")
    n = ends.shape[0]
    return _pack(ends.data_ptr() if n else 0, N.ST_I32, 1, n, 0, ends.stride(0), 0)


def _stack_desc(t: torch.Tensor, groups: int, name: str) -> tuple[bytes, int]:
    """The descriptor of a stack's first matrix, and the stride of its groups."""
    if t.dim() != 3:
        raise ValueError(f"{name} must be a 3D tensor.")
    if t.shape[0] != groups:
        raise ValueError(f"{name} must hold one matrix for each of the {groups} groups, got {t.shape[0]}")
    code = _CODES.get(t.dtype)
    if code is None:
        raise ValueError(f"unsupported dtype {t.dtype}")
    _, r, c = t.shape
    sg, s0, s1 = t.stride()
    return _pack(t.data_ptr() if r and c and groups else 0, code, 2, r, c, s0, s1), sg


def _workspace(name: str, like: torch.Tensor, da: bytes, db: bytes, *args: int) -> tuple[torch.Tensor | None, int]:
    size = ctypes.c_uint64(0)
    fn = _fns.get(name) or _fn(name, _cp, _cp, *[_i64] * len(args), _vp)
    rc = fn(da, db, *args, ctypes.addressof(size))
    if rc != N.ST_OK:
        N.check(rc, name[3:].replace("_workspace", ""))
    need = size.value
    return (torch.empty(need, dtype=torch.uint8, device=like.device) if need else None), need


def _on_16(t: torch.Tensor, rows: int, cols: int) -> bool:
    """Whether matrices [..., rows, cols] (dimension numbers) of 16-bit elements are read in place: contiguous rows,
    everything on 16-byte boundaries."""
    s = t.stride()
    return (s[cols] == 1 and s[rows] % 8 == 0 and s[rows] >= t.shape[cols] and t.data_ptr() % 16 == 0 and
            (len(s) == 2 or s[0] % 8 == 0 and s[0] > 0))


def matmul_grouped(A: torch.Tensor, B: torch.Tensor, ends: torch.Tensor, *, out_dtype: torch.dtype | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """C [T, N]: C[r] = A[r] @ B[g] for the rows r of each group g.

    A [T, K] and B [G, K, N], both float16 or both bfloat16, any strides (the
    gradient of A is this call with B's transposed view).  ends [G], int32 on
    the device, at most 1024 of them: group g is rows [ends[g - 1], ends[g]); groups
    may be empty, and an end out of order counts as the nearest one in order.
    Sums are fp32 as the tensor core adds them, truncating: within (K + 4) 2^-23
    of the sum of the terms' magnitudes (for K = 1001 1.2e-6 of the result as a
    whole, where fp32 operations that round have 0.5e-6), then one rounding to
    C's type, out_dtype, by default A's.  Rows behind the last
    group are 0 in a new C, and left as they were in ``out``.  The same inputs
    give the same bits.  Operands off 16-byte boundaries are copied first.
    """
    if A.dim() != 2:
        raise ValueError("A must be a 2D tensor.")
    de = _ends_desc(ends)
    groups = ends.shape[0]
    db, stride = _stack_desc(B, groups, "B")
    da = _desc(A)
    if A.shape[1] != B.shape[1]:
        raise ValueError(f"Incompatible matrices: K dimension of A ({A.shape[1]}) must match K dimension of B ({B.shape[1]})")
    dev = _device_of(A, B, ends, out)
    fresh = out is None
    if fresh:
        out_dtype = out_dtype or A.dtype
        if out_dtype not in _CODES:
            raise ValueError(f"unsupported dtype {out_dtype}")
        rows, cols = A.shape[0], B.shape[2]
        out, dc = _new(A, rows, cols, max(cols, 1), 1, out_dtype)
    else:
        dc = _desc(out)
    workspace, need = None, 0
    if not (_on_16(A, 0, 1) and (_on_16(B, 2, 1) or _on_16(B, 1, 2))):
        workspace, need = _workspace("st_matmul_grouped_workspace", A, da, db, stride, groups)
    fn = _fns.get("st_matmul_grouped") or _fn("st_matmul_grouped", _vp, _cp, _cp, _i64, _cp, _cp, _i32, _vp, _u64, _cp)
    rc = fn(context(dev), da, db, stride, de, dc, fresh, None if workspace is None else workspace.data_ptr(), need,
            _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "matmul_grouped")
    return out


def matmul_grouped_weights(A: torch.Tensor, C: torch.Tensor, ends: torch.Tensor, *, out_dtype: torch.dtype | None = None,
                           out: torch.Tensor | None = None) -> torch.Tensor:
    """D [G, K, N]: D[g] = A[rows of g].t() @ C[rows of g], 0 for an empty group.

    A [T, K] and C [T, N], both float16 or both bfloat16, any strides; ends as
    in matmul_grouped.  With C the gradient of matmul_grouped's result, D is
    that of its B (of B's transposed view with A and C exchanged).  Sums as in
    matmul_grouped, over a group's rows; D is out_dtype, A's type by default,
    and ``out`` a stack of any layout whose columns lie together and whose groups
    do not overlap ([K, G, N] transposed among them).  The same inputs give the
    same bits.  Operands off 16-byte boundaries are copied first.
    """
    if A.dim() != 2 or C.dim() != 2:
        raise ValueError("A and C must be 2D tensors.")
    de = _ends_desc(ends)
    groups = ends.shape[0]
    da, dc = _desc(A), _desc(C)
    if A.shape[0] != C.shape[0]:
        raise ValueError(f"A and C must have the same rows, got {A.shape[0]} and {C.shape[0]}")
    dev = _device_of(A, C, ends, out)
    if out is None:
        out_dtype = out_dtype or A.dtype
        if out_dtype not in _CODES:
            raise ValueError(f"unsupported dtype {out_dtype}")
        out = A.new_empty((groups, A.shape[1], C.shape[1]), dtype=out_dtype)
    dd, stride = _stack_desc(out, groups, "out")
    workspace, need = None, 0
    if not (_on_16(A, 0, 1) and _on_16(C, 0, 1)):
        workspace, need = _workspace("st_matmul_grouped_weights_workspace", A, da, dc, groups)
    fn = _fns.get("st_matmul_grouped_weights") or _fn("st_matmul_grouped_weights", _vp, _cp, _cp, _cp, _cp, _i64, _vp, _u64, _cp)
    rc = fn(context(dev), da, dc, de, dd, stride, None if workspace is None else workspace.data_ptr(), need, _exec_desc(dev))
    if rc != N.ST_OK:
        N.check(rc, "matmul_grouped_weights")
    return out
