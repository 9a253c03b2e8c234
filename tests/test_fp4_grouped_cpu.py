"""Refusals of the 4-bit and grouped calls, without a GPU: every argument is
checked before the context and the device are looked at."""
import ctypes
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import sptiles_b200 as st
from sptiles_b200 import _native as N

E4, E8, Q4, F32, F16, BF16, I32 = N.ST_E4M3, N.ST_E8M0, N.ST_E2M1X2, N.ST_F32, N.ST_F16, N.ST_BF16, N.ST_I32
DATA = 0x1000  # a pointer that is never read
BAD, NOT = N.ST_ERR_INVALID_ARGUMENT, N.ST_ERR_UNSUPPORTED


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


def pick(v, default):
    return default if v == 0 else v


# ------------------------------------------------------------------ quantise
def quantize(a=0, q=0, s=0, amax=None, t=0, ws=0x4000, ws_bytes=1 << 20):
    return N.lib().st_quantize_fp4(None, ref(pick(a, t2(10, 300))), ref(pick(q, t2(10, 150, Q4))), ref(pick(s, t1(5 * 512, E4))), ref(amax),
                                   ref(pick(t, t1(1))), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(a=t2(10, 300, E4)), BAD, "A must be"), (dict(a=t2(10, 300, I32)), BAD, "A must be"), (dict(a=t1(10)), BAD, "rank 2"),
    (dict(a=t2(10, 300, data=None)), BAD, "null data"), (dict(a=t2(10, 300, strides=(-300, 1))), BAD, "negative stride"),
    (dict(q=t2(10, 150, E4)), BAD, "Q must be"), (dict(q=t2(10, 300, Q4)), BAD, "Q must be [rows"), (dict(q=t2(9, 150, Q4)), BAD, "Q must be [rows"),
    (dict(q=t2(10, 150, Q4, strides=(300, 2))), NOT, "unit column"), (dict(q=t2(10, 150, Q4, strides=(149, 1))), BAD, "overlapping"),
    (dict(s=t1(4 * 512, E4)), BAD, "scale must be contiguous"), (dict(s=t1(5 * 512, F32)), BAD, "scale must be"),
    (dict(s=t1(5 * 512, E4, stride=2)), BAD, "contiguous"), (dict(s=t1(5 * 512, E4, data=DATA + 8)), BAD, "16-byte"),
    (dict(s=t1(5 * 512, E4, data=None)), BAD, "null data"), (dict(s=None), BAD, "scale is null"), (dict(s=t1(5 * 512, E8)), BAD, "scales"),
    (dict(s=t1(3 * 512, E8)), BAD, "go with"), (dict(s=t1(3 * 512, E8), amax=t1(1), t=None), BAD, "go with"), (dict(t=None), BAD, "need tensor_scale"),
    (dict(t=t1(2)), BAD, "one ST_F32"), (dict(t=t1(1, BF16)), BAD, "one ST_F32"), (dict(amax=t1(0)), BAD, "one ST_F32"),
    (dict(ws=None), BAD, "workspace"), (dict(ws_bytes=16), BAD, "workspace"), (dict(ws=0x4002), BAD, "4-byte aligned"),
    (dict(a=t2(1, 2 ** 30), q=t2(1, 2 ** 29, Q4)), NOT, "at most"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_quantize_refusals(kw, code, word):
    refused(quantize(**kw), code, word)


def test_good_arguments_reach_the_context():
    refused(quantize(), BAD, "null context")
    refused(quantize(amax=t1(1), ws=None, ws_bytes=0), BAD, "null context")
    refused(quantize(s=t1(3 * 512, E8), t=None, ws=None, ws_bytes=0), BAD, "null context")
    refused(dequantize(), BAD, "null context")
    refused(dequantize(out=t2(10, 299)), BAD, "null context")
    refused(product(), BAD, "null context")
    refused(grouped(), BAD, "null context")
    refused(weights(), BAD, "null context")
    refused(grouped(b=t2(64, 32, F16, data=None), ends=t1(0, I32, data=None)), BAD, "null context")
    refused(weights(d=t2(64, 32, data=None), ends=t1(0, I32, data=None)), BAD, "null context")


def dequantize(q=0, s=0, t=0, out=0):
    return N.lib().st_dequantize_fp4(None, ref(pick(q, t2(10, 150, Q4))), ref(pick(s, t1(5 * 512, E4))), ref(pick(t, t1(1))),
                                     ref(pick(out, t2(10, 300, BF16))), None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(q=t2(10, 150, E4)), BAD, "Q must be"), (dict(s=t1(512, E4)), BAD, "scale must be"), (dict(out=t2(10, 301)), BAD, "out must be"),
    (dict(out=t2(10, 298)), BAD, "out must be"), (dict(out=t2(9, 300)), BAD, "out must be"), (dict(out=t2(10, 300, E4)), BAD, "out must be"),
    (dict(out=t2(10, 300, strides=(0, 1))), BAD, "overlapping"), (dict(s=t1(3 * 512, E8)), BAD, "goes with"), (dict(t=t1(2)), BAD, "one ST_F32"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_dequantize_refusals(kw, code, word):
    refused(dequantize(**kw), code, word)


# ------------------------------------------------------------------ product
def product(a=0, b=0, sa=0, sb=0, ta=None, tb=None, bias=None, c=0, ws=None, ws_bytes=0):
    return N.lib().st_matmul_fp4(None, ref(pick(a, t2(16, 128, Q4))), ref(pick(b, t2(128, 32, Q4, strides=(1, 128)))),
                                 ref(pick(sa, t1(4 * 512, E4))), ref(pick(sb, t1(4 * 512, E4))), ref(ta), ref(tb), ref(bias),
                                 ref(pick(c, t2(16, 32, BF16))), ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(a=t2(16, 128, E4)), BAD, "A must be ST_E2M1X2"), (dict(b=t2(128, 32, F16)), BAD, "B must be ST_E2M1X2"),
    (dict(b=t2(127, 32, Q4, strides=(1, 128))), BAD, "Incompatible matrices"), (dict(sa=t1(3 * 512, E4)), BAD, "a_scale must be contiguous"),
    (dict(sb=t1(512, E4)), BAD, "b_scale must be contiguous"), (dict(sa=t1(2 * 512, E8)), BAD, "one type"), (dict(sb=t1(2048, F32)), BAD, "b_scale must be"),
    (dict(sa=t1(2 * 512, E8), sb=t1(2 * 512, E8), ta=t1(1)), BAD, "tensor scales go with"), (dict(ta=t1(2)), BAD, "a_tensor_scale must be one"),
    (dict(tb=t1(1, F16)), BAD, "b_tensor_scale must be one"), (dict(c=t2(32, 16, BF16)), BAD, "C must be [M, N]"), (dict(c=t2(16, 32, E4)), BAD, "C must be"),
    (dict(c=t2(16, 32, BF16, strides=(1, 16))), NOT, "unit column stride"), (dict(c=t2(16, 32, BF16, strides=(0, 1))), BAD, "overlapping"),
    (dict(bias=t1(31)), BAD, "N elements"), (dict(bias=t1(32, F16)), BAD, "bias must be"), (dict(bias=t1(32, stride=2)), NOT, "contiguous"),
    (dict(bias=t1(32, data=None)), BAD, "null data"), (dict(a=t2(16, 128, Q4, strides=(129, 1))), BAD, "workspace"),
    (dict(b=t2(128, 32, Q4)), BAD, "workspace"), (dict(a=t2(16, 128, Q4, data=DATA + 1), ws=0x2008, ws_bytes=1 << 20), BAD, "16-byte aligned"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_product_refusals(kw, code, word):
    refused(product(**kw), code, word)


def test_product_workspace():
    L, n = N.lib(), ctypes.c_uint64(7)

    def need(a, b):
        assert L.st_matmul_fp4_workspace(ref(a), ref(b), ctypes.byref(n)) == N.ST_OK, N.last_error()
        return n.value

    b = t2(128, 32, Q4, strides=(1, 128))
    assert need(t2(16, 128, Q4), b) == 0
    assert need(t2(1, 33, Q4), t2(33, 1, Q4, strides=(1, 7))) == 0            # one row: its stride is not used
    assert need(t2(16, 125, Q4), t2(125, 32, Q4, strides=(1, 128))) == 16 * 128
    assert need(t2(16, 128, Q4, data=DATA + 8), b) == 16 * 128
    assert need(t2(16, 128, Q4, strides=(0, 1)), b) == 16 * 128               # a broadcast row
    assert need(t2(16, 128, Q4), t2(128, 32, Q4)) == 32 * 128                 # stored across K
    refused(L.st_matmul_fp4_workspace(ref(t2(16, 128, E4)), ref(b), ctypes.byref(n)), BAD, "A must be")
    refused(L.st_matmul_fp4_workspace(ref(t2(16, 128, Q4)), ref(b), None), BAD, "bytes")


# ------------------------------------------------------------------ groups
def grouped(a=0, b=0, stride=2048, ends=0, c=0, ws=None, ws_bytes=0):
    return N.lib().st_matmul_grouped(None, ref(pick(a, t2(16, 64, F16))), ref(pick(b, t2(64, 32, F16))), stride, ref(pick(ends, t1(4, I32))),
                                     ref(pick(c, t2(16, 32))), 0, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(ends=None), BAD, "ends is null"), (dict(ends=t1(4, F32)), BAD, "ST_I32"), (dict(ends=t1(4, I32, stride=2)), BAD, "contiguous"),
    (dict(ends=t1(4, I32, data=None)), BAD, "null data"), (dict(ends=t1(1025, I32)), NOT, "at most 1024"), (dict(ends=t2(2, 2, I32)), BAD, "rank 1"),
    (dict(a=t2(16, 64), b=t2(64, 32)), NOT, "ST_F16 or ST_BF16"), (dict(a=t2(16, 64, BF16)), BAD, "both be"), (dict(a=t2(16, 64, E4)), BAD, "both be"),
    (dict(b=t2(63, 32, F16)), BAD, "Incompatible matrices"), (dict(stride=-1), BAD, "negative group stride"), (dict(b=None), BAD, "B is null"),
    (dict(b=t2(64, 32, F16, data=None)), BAD, "null data"), (dict(c=t2(16, 31)), BAD, "C must be [16, 32]"), (dict(c=t2(16, 32, E4)), BAD, "C must be"),
    (dict(c=t2(16, 32, strides=(64, 2))), NOT, "unit column"), (dict(c=t2(16, 32, strides=(31, 1))), BAD, "overlapping"),
    (dict(a=t2(16, 64, F16, strides=(65, 1))), BAD, "workspace"), (dict(stride=2049), BAD, "workspace"), (dict(stride=4, ws=0x2008, ws_bytes=1 << 24), BAD, "16-byte"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_grouped_refusals(kw, code, word):
    refused(grouped(**kw), code, word)


def weights(a=0, c=0, ends=0, d=0, stride=2048, ws=None, ws_bytes=0):
    return N.lib().st_matmul_grouped_weights(None, ref(pick(a, t2(16, 64, F16))), ref(pick(c, t2(16, 32, F16))), ref(pick(ends, t1(4, I32))),
                                             ref(pick(d, t2(64, 32))), stride, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,code,word", [
    (dict(c=t2(15, 32, F16)), BAD, "same rows"), (dict(c=t2(16, 32, BF16)), BAD, "both be"), (dict(d=t2(32, 64)), BAD, "D must be [64, 32]"),
    (dict(d=t2(64, 32, strides=(0, 1))), BAD, "overlapping"), (dict(stride=2047), BAD, "overlapping groups"), (dict(stride=0), BAD, "overlapping groups"),
    (dict(d=None), BAD, "D is null"), (dict(a=t2(16, 64, F16, strides=(1, 16))), BAD, "workspace"), (dict(ends=t1(2000, I32)), NOT, "at most"),
], ids=lambda v: v if isinstance(v, str) else "")
def test_weights_refusals(kw, code, word):
    refused(weights(**kw), code, word)


def test_grouped_workspace():
    L, n = N.lib(), ctypes.c_uint64(7)

    def need(a, b, stride, groups):
        assert L.st_matmul_grouped_workspace(ref(a), ref(b), stride, groups, ctypes.byref(n)) == N.ST_OK, N.last_error()
        return n.value

    a, b = t2(16, 64, F16), t2(64, 32, F16)
    assert need(a, b, 2048, 4) == 0
    assert need(a, t2(64, 32, F16, strides=(1, 64)), 2048, 4) == 0              # each matrix stored along K
    assert need(a, b, 0, 4) == 0                                                # one matrix for all
    assert need(a, b, 2052, 4) == 4 * 64 * 32 * 2                               # matrices off 16-byte boundaries
    assert need(a, b, 2052, 1) == 0
    assert need(t2(16, 64, F16, strides=(1, 16)), b, 2048, 4) == 16 * 64 * 2    # A stored along its rows
    assert need(t2(16, 63, F16), t2(63, 30, F16), 1890, 4) == 16 * 64 * 2 + 4 * 63 * 32 * 2
    refused(L.st_matmul_grouped_workspace(ref(a), ref(b), 2048, 1025, ctypes.byref(n)), BAD, "groups")
    refused(L.st_matmul_grouped_workspace(ref(a), ref(b), 2048, 4, None), BAD, "bytes")
    assert L.st_matmul_grouped_weights_workspace(ref(a), ref(t2(16, 32, F16)), 4, ctypes.byref(n)) == N.ST_OK and n.value == 0
    assert L.st_matmul_grouped_weights_workspace(ref(a), ref(t2(16, 30, F16)), 4, ctypes.byref(n)) == N.ST_OK and n.value == 16 * 32 * 2


# ------------------------------------------------------------------ Python
def test_python_refusals():
    x = torch.randn(4, 128)
    q = torch.zeros(4, 64, dtype=torch.uint8)
    s = torch.zeros(1, 2, 32, 4, 4, dtype=torch.uint8).view(torch.float8_e4m3fn)
    wide = torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu)
    a, b, ends = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(2, 8, 16, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: st.quantize_fp4(x), lambda: st.dequantize_fp4(q, s), lambda: st.matmul_fp4(q, q.t(), s, s),
                 lambda: st.matmul_grouped(a, b, ends), lambda: st.matmul_grouped_weights(a, a, ends)):
        with pytest.raises(ValueError, match="CUDA device"):
            call()
    for call, word in [
        (lambda: st.quantize_fp4(x[0]), "2D"), (lambda: st.quantize_fp4(x, scale_dtype=torch.float16), "scale_dtype"),
        (lambda: st.quantize_fp4(x.double()), "unsupported dtype"), (lambda: st.quantize_fp4(x, scale_dtype=torch.float8_e8m0fnu, amax=x[0, 0]), "amax goes with"),
        (lambda: st.dequantize_fp4(x, s), "codes must have dtype"), (lambda: st.dequantize_fp4(q, s, cols=126), "cols must be"),
        (lambda: st.dequantize_fp4(q, x), "scale must have dtype"), (lambda: st.dequantize_fp4(q, s[:, :1]), "scale must be contiguous"),
        (lambda: st.dequantize_fp4(q, s, x), "one float32"), (lambda: st.dequantize_fp4(q, s, out_dtype=torch.int32), "unsupported dtype"),
        (lambda: st.matmul_fp4(q, q, s, s), "Incompatible"), (lambda: st.matmul_fp4(q[0], q.t(), s, s), "2D"), (lambda: st.matmul_fp4(x, q.t(), s, s), "A must have dtype"),
        (lambda: st.matmul_fp4(q, q.t(), s, wide[:0]), "b_scale must be contiguous"), (lambda: st.matmul_fp4(q, q.t(), s, s, a_tensor_scale=x), "one float32"),
        (lambda: st.matmul_grouped(a[0], b, ends), "2D"), (lambda: st.matmul_grouped(a, b[0], ends), "3D"), (lambda: st.matmul_grouped(a, b[:1], ends), "one matrix"),
        (lambda: st.matmul_grouped(a, b.transpose(1, 2), ends), "Incompatible"), (lambda: st.matmul_grouped(a, b, ends.long()), "int32"),
        (lambda: st.matmul_grouped(a, b, ends[None]), "int32"), (lambda: st.matmul_grouped_weights(a, a[:3], ends), "same rows"),
        (lambda: st.matmul_grouped_weights(a, b, ends), "2D"), (lambda: st.matmul_grouped_weights(a.int(), a, ends), "unsupported dtype"),
    ]:
        with pytest.raises(ValueError, match=word):
            call()


def test_other_calls_refuse_4_bit_types():
    assert N.lib().st_cast(None, ref(t2(4, 4, Q4)), ref(t2(4, 4)), None) == BAD
    refused(N.lib().st_quantize_fp8(None, ref(t2(10, 300)), ref(t2(10, 300, Q4)), ref(t2(10, 3)), 1, 128, None), BAD, "Q must be")
    refused(N.lib().st_matmul_fp8(None, ref(t2(16, 256, Q4)), ref(t2(256, 32, Q4)), ref(t2(16, 2)), ref(t2(2, 32)), None, ref(t2(16, 32)),
                                  None, 0, None), BAD, "A and B must be")


# ------------------------------------------------------------------ addresses and extents that a kernel could not take
@pytest.mark.parametrize("call,kw,name", [
    (quantize, dict(a=t2(10, 300, data=DATA + 2)), "A"), (quantize, dict(a=t2(10, 300, BF16, data=DATA + 1)), "A"),
    (quantize, dict(amax=t1(1, data=DATA + 1)), "amax"), (quantize, dict(t=t1(1, data=DATA + 2)), "tensor_scale"),
    (dequantize, dict(out=t2(10, 300, BF16, data=DATA + 1)), "out"), (dequantize, dict(t=t1(1, data=DATA + 2)), "tensor_scale"),
    (product, dict(c=t2(16, 32, BF16, data=DATA + 1)), "C"), (product, dict(bias=t1(32, data=DATA + 2)), "bias"),
    (product, dict(tb=t1(1, data=DATA + 1)), "b_tensor_scale"),
    (grouped, dict(a=t2(16, 64, F16, data=DATA + 1)), "A"), (grouped, dict(b=t2(64, 32, F16, data=DATA + 1)), "B"),
    (grouped, dict(ends=t1(4, I32, data=DATA + 2)), "ends"), (grouped, dict(c=t2(16, 32, data=DATA + 2)), "C"),
    (weights, dict(c=t2(16, 32, F16, data=DATA + 1)), "C"), (weights, dict(d=t2(64, 32, data=DATA + 2)), "D"),
])
def test_elements_off_their_boundary(call, kw, name):
    refused(call(**kw), BAD, name + " must start on a boundary of its elements")


@pytest.mark.parametrize("extent", [2**30, 2**31 - 1])
def test_extents_near_int32(extent):
    refused(grouped(a=t2(extent, 64, F16), c=t2(extent, 32)), NOT, "extents of at most")
    refused(grouped(b=t2(64, extent, F16), c=t2(16, extent)), NOT, "extents of at most")
    refused(weights(a=t2(extent, 64, F16), c=t2(extent, 32, F16)), NOT, "extents of at most")


def test_a_torch_without_the_small_types():
    """The package imports and keeps its other calls; 4-bit codes are uint8 and blocks of 32 are refused."""
    code = """
import torch
for name in ("float4_e2m1fn_x2", "float8_e8m0fnu"):
    delattr(torch, name)
import sptiles_b200 as st
x = torch.zeros(2, 32)
for call, word in [(lambda: st.matmul(x, x), "K"), (lambda: st.quantize_fp4(x, scale_dtype=torch.uint8), "scale_dtype"),
                   (lambda: st.quantize_fp4(x), "CUDA"),
                   (lambda: st.dequantize_fp4(x.to(torch.uint8), torch.zeros(1, 1, 32, 4, 4, dtype=torch.uint8)), "scale must have"),
                   (lambda: st.dequantize_fp4(x.to(torch.uint8), torch.zeros(1, 1, 32, 4, 4).to(torch.float8_e4m3fn)), "CUDA"),
                   (lambda: st.dequantize_fp4(x, x), "codes must have")]:
    try:
        call()
    except (ValueError, RuntimeError) as e:
        assert word.lower() in str(e).lower(), (word, e)
    else:
        raise SystemExit("not refused: " + word)
print("kept")
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          cwd=str(Path(__file__).resolve().parents[1]))
    assert done.returncode == 0 and "kept" in done.stdout, done.stdout + done.stderr


def test_weights_of_groups_in_turn():
    """Results [K, groups, N] do not overlap and get past that check, to the workspace's; a row too short for all groups does."""
    for stride, row, word in [(32, 128, "workspace"), (40, 152, "workspace"), (32, 127, "overlapping groups"), (31, 128, "overlapping groups"),
                              (40, 151, "overlapping groups")]:
        refused(weights(a=t2(16, 64, F16, strides=(1, 16)), d=t2(64, 32, strides=(row, 1)), stride=stride), BAD, word)
