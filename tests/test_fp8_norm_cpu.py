"""Refusals of the 8-bit and norm calls, without a GPU: every argument is
checked before the context and the device are looked at."""
import ctypes

import pytest
import torch

import sptiles_b200 as st
from sptiles_b200 import _native as N

E4, E5, F32, F16, BF16, I32 = N.ST_E4M3, N.ST_E5M2, N.ST_F32, N.ST_F16, N.ST_BF16, N.ST_I32
DATA = 0x1000  # a pointer that is never read


def t2(rows, cols, dtype=F32, strides=None, data=DATA):
    v = N.StTensor()
    v.data, v.dtype, v.rank = data, dtype, 2
    v.shape[0], v.shape[1] = rows, cols
    v.strides[0], v.strides[1] = strides if strides else (max(cols, 1), 1)
    return v


def t1(n, dtype=F32, stride=1, data=DATA):
    v = N.StTensor()
    v.data, v.dtype, v.rank = data, dtype, 1
    v.shape[0], v.strides[0] = n, stride
    return v


def ref(v):
    return None if v is None else ctypes.byref(v)


def refused(rc, code, word):
    assert rc == code, (rc, N.last_error())
    assert word in N.last_error(), N.last_error()


BAD, NOT = N.ST_ERR_INVALID_ARGUMENT, N.ST_ERR_UNSUPPORTED


# ------------------------------------------------------------------ quantize
def quantize(a=None, q=None, s=None, block=(1, 128)):
    a = a or t2(10, 300)
    q = q or t2(10, 300, E4)
    s = s or t2(10, 3)
    return N.lib().st_quantize_fp8(None, ref(a), ref(q), ref(s), *block, None)


@pytest.mark.parametrize("kw,word", [
    (dict(block=(1, 64)), "blocks are"), (dict(block=(128, 64)), "blocks are"), (dict(a=t2(10, 300, E4)), "A must be"),
    (dict(a=t2(10, 300, I32)), "A must be"), (dict(q=t2(10, 300, F16)), "Q must be"), (dict(s=t2(10, 3, F16)), "scale must be"),
    (dict(q=t2(10, 301, E4)), "same shape"), (dict(s=t2(10, 2)), "scale must be"), (dict(s=t2(3, 10)), "scale must be"),
    (dict(a=t1(10)), "rank 2"), (dict(a=t2(10, 300, strides=(-300, 1))), "negative stride"), (dict(a=t2(-1, 300)), "negative extent"),
    (dict(a=t2(10, 300, data=None)), "null data"), (dict(q=t2(10, 300, E4, strides=(0, 1))), "overlapping"),
    (dict(q=t2(10, 300, E4, strides=(299, 1))), "overlapping"), (dict(s=t2(10, 3, strides=(1, 9))), "overlapping"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_quantize_refusals(kw, word):
    refused(quantize(**kw), BAD, word)


def test_good_arguments_reach_the_context():
    refused(quantize(), BAD, "null context")
    refused(quantize(s=t2(1, 300), block=(128, 1)), BAD, "null context")
    refused(matmul(), BAD, "null context")
    refused(forward(), BAD, "null context")
    refused(backward(), BAD, "null context")


# ------------------------------------------------------------------ matmul
def matmul(a=None, b=None, sa=None, sb=None, bias=None, c=None, ws=None, ws_bytes=0):
    a = a or t2(16, 256, E4)
    b = b or t2(256, 32, E4, strides=(1, 256))
    sa, sb, c = sa or t2(16, 2), sb or t2(2, 32), c or t2(16, 32, BF16)
    return N.lib().st_matmul_fp8(None, ref(a), ref(b), ref(sa), ref(sb), ref(bias), ref(c), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(a=t2(16, 256, F16)), BAD, "A and B must be"), (dict(b=t2(256, 32, BF16)), BAD, "A and B must be"),
    (dict(b=t2(255, 32, E4, strides=(1, 256))), BAD, "Incompatible matrices"), (dict(sa=t2(16, 3)), BAD, "a_scale"),
    (dict(sa=t2(2, 2)), BAD, "a_scale"), (dict(sb=t2(2, 31)), BAD, "b_scale"), (dict(sb=t2(32, 2)), BAD, "b_scale"),
    (dict(sa=t2(16, 2, F16)), BAD, "a_scale must be"), (dict(c=t2(32, 16, BF16)), BAD, "C must be [M, N]"),
    (dict(c=t2(16, 32, E4)), BAD, "C must be"), (dict(c=t2(16, 32, BF16, strides=(1, 16))), NOT, "unit column stride"),
    (dict(c=t2(16, 32, BF16, strides=(0, 1))), BAD, "overlapping"), (dict(bias=t1(31)), BAD, "N elements"),
    (dict(bias=t1(32, F16)), BAD, "bias must be"), (dict(bias=t1(32, stride=2)), NOT, "contiguous"),
    (dict(bias=t1(32, data=None)), BAD, "null data"), (dict(a=t2(16, 256, E4, strides=(257, 1))), BAD, "workspace"),
    (dict(a=t2(16, 256, E4, data=DATA + 1)), BAD, "workspace"),
    (dict(a=t2(16, 256, E4, data=DATA + 1), ws=0x2008, ws_bytes=1 << 20), BAD, "16-byte aligned"),
    (dict(a=t2(2 ** 31, 256, E4), sa=t2(2 ** 24, 2), c=t2(2 ** 31, 32, BF16)), NOT, "int32"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_matmul_refusals(kw, code, word):
    refused(matmul(**kw), code, word)


def test_matmul_workspace():
    L, n = N.lib(), ctypes.c_uint64(7)

    def need(a, b):
        assert L.st_matmul_fp8_workspace(ref(a), ref(b), ctypes.byref(n)) == N.ST_OK, N.last_error()
        return n.value

    k_major = t2(256, 32, E4, strides=(1, 256))
    assert need(t2(16, 256, E4), k_major) == 0
    assert need(t2(16, 256, E4, strides=(1, 16)), t2(256, 32, E4)) == 0     # both along their outer dimension
    assert need(t2(1, 33, E4), t2(33, 1, E4, strides=(1, 7))) == 0          # one row: its stride is not used
    assert need(t2(16, 250, E4), t2(250, 32, E4, strides=(1, 256))) == 16 * 256
    assert need(t2(16, 256, E4, data=DATA + 8), k_major) == 16 * 256
    assert need(t2(16, 256, E4, strides=(0, 1)), k_major) == 16 * 256       # a broadcast row
    assert need(t2(16, 256, E4, strides=(32, 1)), k_major) == 16 * 256      # overlapping rows
    assert need(t2(16, 256, E4, strides=(512, 2)), t2(256, 30, E4)) == 16 * 256 + 256 * 32
    assert need(t2(0, 256, E4, strides=(3, 1)), k_major) == 0
    refused(L.st_matmul_fp8_workspace(ref(t2(16, 256, F32)), ref(k_major), ctypes.byref(n)), BAD, "A and B must be")
    refused(L.st_matmul_fp8_workspace(ref(t2(16, 256, E4)), ref(k_major), None), BAD, "bytes")


# ------------------------------------------------------------------ norms
def options(alpha=1.0, eps=1e-6, offset=0.0):
    return N.StNormOptions(alpha, eps, offset)


def forward(x=0, r=None, post=None, gate=None, pre=0, out=0, h=0, hs=None, opt=0):
    x = t2(8, 64, BF16) if x == 0 else x
    r = r or t2(8, 64)
    pre = t1(64) if pre == 0 else pre
    out = t2(8, 64) if out == 0 else out
    h = t2(8, 64, BF16) if h == 0 else h
    opt = options() if opt == 0 else opt
    return N.lib().st_residual_norm(None, *map(ref, (x, r, post, gate, pre, out, h, hs, opt)), None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(x=t2(8, 63, BF16)), BAD, "x must be"), (dict(x=t2(8, 64, E4)), BAD, "tensors must be"),
    (dict(r=t2(8, 64, F16), out=t2(8, 64, F16)), BAD, "tensors must be"), (dict(out=t2(8, 64, BF16)), BAD, "same dtype"),
    (dict(h=t2(8, 64, F16)), BAD, "normed must have"), (dict(post=t1(63)), BAD, "one element per column"),
    (dict(post=t1(64, F16)), BAD, "post_weight must be"), (dict(pre=t1(64, stride=2)), NOT, "contiguous"),
    (dict(pre=None), BAD, "come together"), (dict(h=None), BAD, "come together"), (dict(gate=t2(8, 63)), BAD, "gate must be"),
    (dict(gate=t2(2, 64)), BAD, "gate must be"), (dict(gate=t2(8, 64, strides=(128, 2))), NOT, "unit column"),
    (dict(x=None, post=t1(64)), BAD, "need x"), (dict(x=None, pre=None, h=None, out=None), BAD, "nothing"),
    (dict(h=t2(8, 64, E4)), BAD, "scales"), (dict(hs=t2(8, 1)), BAD, "scales"), (dict(h=t2(8, 64, E4), hs=t2(8, 2)), BAD, "normed_scale"),
    (dict(r=t2(8, 64, strides=(64, 2))), NOT, "unit column"), (dict(out=t2(8, 64, strides=(0, 1))), BAD, "overlapping"),
    (dict(opt=None), BAD, "options"), (dict(opt=options(eps=-1.0)), BAD, "eps"), (dict(opt=options(alpha=float("nan"))), BAD, "finite"),
    (dict(x=None, r=t2(8, 0), out=None, pre=t1(0), h=t2(8, 0)), BAD, "at least one element"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_forward_refusals(kw, code, word):
    refused(forward(**kw), code, word)


def backward(dres=0, dh=0, x=0, r=0, post=None, gate=None, pre=0, dx=0, dr=0, dpost=None, dgate=None, dpre=0, ws=0x4000,
             ws_bytes=1 << 30, opt=0):
    pick = lambda v, d: d if v == 0 else v  # noqa: E731
    args = (pick(dres, t2(8, 64)), pick(dh, t2(8, 64, BF16)), pick(x, t2(8, 64, BF16)), pick(r, t2(8, 64)), post, gate,
            pick(pre, t1(64)), pick(dx, t2(8, 64, BF16)), pick(dr, t2(8, 64)), dpost, dgate, pick(dpre, t1(64)))
    return N.lib().st_residual_norm_backward(None, *map(ref, args), ws, ws_bytes, ref(pick(opt, options())), None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(dres=None, dh=None), BAD, "no gradient"), (dict(dh=None), BAD, "come together"), (dict(pre=None, dpre=None), BAD, "come together"),
    (dict(r=None), BAD, "updated residual"), (dict(dx=None), BAD, "come together"), (dict(x=None, dx=None, gate=t1(64), dgate=t1(64)), BAD, "need x"),
    (dict(dpost=t1(64)), BAD, "go with"), (dict(gate=t1(64)), BAD, "go with"), (dict(dpre=t1(64, BF16)), BAD, "ST_F32"),
    (dict(gate=t1(64), dgate=t2(8, 64)), BAD, "gate's shape"), (dict(gate=t1(64), dgate=t1(64, BF16)), BAD, "dgate must be"),
    (dict(gate=t2(8, 64, BF16), dgate=t2(8, 64, F16)), BAD, "dgate must be"), (dict(dr=t2(8, 64, BF16)), BAD, "dtype of its tensor"),
    (dict(dh=t2(8, 64)), BAD, "dtype of its tensor"), (dict(dres=t2(8, 64, F16)), BAD, "dtype of its tensor"),
    (dict(ws=None), BAD, "workspace"), (dict(ws_bytes=64), BAD, "workspace"), (dict(ws=0x4008), BAD, "16-byte aligned"),
    (dict(dx=t2(8, 64, BF16, strides=(32, 1))), BAD, "overlapping"), (dict(opt=options(eps=float("inf"))), BAD, "finite"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_backward_refusals(kw, code, word):
    refused(backward(**kw), code, word)


def test_backward_workspace():
    n = ctypes.c_uint64(0)
    L = N.lib()
    for rows, cols in [(1, 1), (8, 64), (100000, 512), (100000, 513), (3, 16384)]:
        assert L.st_residual_norm_backward_workspace(rows, cols, ctypes.byref(n)) == N.ST_OK
        assert 3 * 4 * cols <= n.value <= 3 * 4 * cols * 2400
    refused(L.st_residual_norm_backward_workspace(-1, 4, ctypes.byref(n)), BAD, "extents")
    refused(L.st_residual_norm_backward_workspace(4, 0, ctypes.byref(n)), BAD, "extents")


# ------------------------------------------------------------------ Python
def test_python_refusals():
    x = torch.randn(4, 128)
    q = torch.zeros(4, 128, dtype=torch.float8_e4m3fn)
    s = torch.ones(4, 1)
    for call in (lambda: st.quantize_fp8(x), lambda: st.matmul_fp8(q, q.t(), s, s.t()), lambda: st.residual_norm(x, x),
                 lambda: st.residual_norm_backward(x, None, x, None)):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    with pytest.raises(ValueError, match="block"):
        st.quantize_fp8(x, block=(2, 128))
    with pytest.raises(ValueError, match="dtype"):
        st.quantize_fp8(x, dtype=torch.float16)
    with pytest.raises(ValueError, match="2D"):
        st.quantize_fp8(x[0])
    with pytest.raises(ValueError, match="Incompatible"):
        st.matmul_fp8(q, q, s, s)
    with pytest.raises(ValueError, match="2D"):
        st.matmul_fp8(q[0], q.t(), s, s.t())
    with pytest.raises(ValueError, match="must be given"):
        st.residual_norm_backward(None, None, x, None)


@pytest.mark.parametrize("dtype", [torch.float64, torch.int32, torch.bool])
def test_python_refuses_a_residual_of_another_type(dtype):
    r = torch.zeros(4, 128, dtype=dtype)
    for x in (None, torch.zeros(4, 128), r):
        with pytest.raises(ValueError, match="unsupported dtype"):
            st.residual_norm(x, r, pre_weight=torch.ones(128))


def test_older_calls_still_refuse_8_bit_types():
    from sptiles_b200 import api

    q = torch.zeros(4, 128, dtype=torch.float8_e4m3fn)
    for f in (api.tensor_view, api._desc):
        with pytest.raises(ValueError, match="unsupported dtype"):
            f(q)
    assert N.lib().st_cast(None, ref(t2(4, 4, E4)), ref(t2(4, 4)), None) == BAD
