"""8-bit blocks and their product on the GPU against plain computations.

The quantiser is compared bit for bit with the same fp32 steps on the CPU.
The product is compared with float64.  Bound for one element: every fp32
addition of a sum of n terms is off by at most 2^-23 of the sum of the terms'
magnitudes (a truncating adder), so a K-term element with its B blocks is
within (K_block + B + 4) 2^-23 sum |a b| of the exact value -- a term passes
at most its block's additions, the blocks' additions and the two scalings --
and the result's rounding adds half a step, eps / 2 relative."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import sptiles_b200 as st

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2
LIMIT = {E4: 448.0, E5: 57344.0}


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ quantiser
def plain_quantize(x, block, dtype):
    """The documented steps, each one IEEE fp32 operation, on the CPU."""
    x = x.float()
    rows, cols = x.shape
    br, bc = block
    pad = torch.zeros(-(-rows // br) * br, -(-cols // bc) * bc)
    pad[:rows, :cols] = x
    tiles = pad.view(pad.shape[0] // br, br, pad.shape[1] // bc, bc)
    limit = torch.tensor(LIMIT[dtype])
    scale = torch.clamp(tiles.abs().amax((1, 3)) / limit, min=2.0 ** -126)
    q = tiles * (torch.tensor(1.0) / scale)[:, None, :, None]
    q = torch.clamp(q, -LIMIT[dtype], LIMIT[dtype]).to(dtype)
    return q.view(pad.shape)[:rows, :cols], scale


def same_codes(got, want):
    """Equal as values and signs; a NaN's code may differ in its sign."""
    g, w = got.cpu().float(), want.float()
    nan = torch.isnan(w)
    assert torch.equal(torch.isnan(g), nan)
    assert torch.equal(g[~nan], w[~nan])
    assert torch.equal(torch.signbit(g[~nan]), torch.signbit(w[~nan]))


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)], ids=["row", "column", "square"])
@pytest.mark.parametrize("src", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 128), (3, 129), (127, 64), (128, 128), (130, 257), (1100, 136), (5, 4096)])
def test_quantize_bits(rows, cols, src, block):
    x = (torch.randn(rows, cols, generator=gen(rows + cols)) * torch.exp(2 * torch.randn(rows, 1, generator=gen(7)))).to(src)
    for dtype in (E4, E5):
        Q, S = st.quantize_fp8(x.to(DEV), block=block, dtype=dtype)
        q, s = plain_quantize(x, block, dtype)
        assert Q.shape == x.shape and Q.dtype == dtype and S.shape == s.shape and S.dtype == torch.float32
        assert torch.equal(S.cpu(), s)
        same_codes(Q, q)


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)], ids=["row", "column", "square"])
@pytest.mark.parametrize("view", ["transposed", "strided", "offset", "broadcast"])
def test_quantize_views(view, block):
    base = torch.randn(301, 405, generator=gen(3))
    cut = {"transposed": lambda t: t.t(), "strided": lambda t: t[::2, ::3], "offset": lambda t: t[1:, 1:],
           "broadcast": lambda t: t[:1].expand(140, -1)}[view]
    Q, S = st.quantize_fp8(cut(base.to(DEV)), block=block)
    q, s = plain_quantize(cut(base), block, E4)
    assert torch.equal(S.cpu(), s)
    same_codes(Q, q)


def test_quantize_extremes():
    """All-zero, subnormal, huge, infinite and NaN blocks; exact ties go to the even code."""
    x = torch.zeros(8, 128)
    x[1, 5], x[2], x[3, 0] = 1e-45, 3e38, float("inf")
    x[4, 100] = float("nan")
    x[5, :4] = torch.tensor([448.0, 17.0, 19.0, -21.0])  # scale 1: between 16, 18, 20 and 22
    x[6] = -0.0
    x[7] = 2.0 ** -130
    Q, S = st.quantize_fp8(x.to(DEV))
    q, s = plain_quantize(x, (1, 128), E4)
    assert torch.equal(torch.nan_to_num(S.cpu(), 1.5), torch.nan_to_num(s, 1.5))
    same_codes(Q, q)
    assert S[5, 0].item() == 1.0 and Q[5, 1:4].float().tolist() == [16.0, 20.0, -20.0]
    assert torch.isnan(S[4, 0]) and torch.isinf(S[3, 0])


def test_quantize_empty_and_given_outputs():
    for shape in [(0, 5), (5, 0), (0, 0)]:
        Q, S = st.quantize_fp8(torch.empty(shape, device=DEV))
        assert Q.shape == shape and S.shape == (shape[0], -(-shape[1] // 128))
    x = torch.randn(70, 200, generator=gen(1))
    room = torch.full((72, 300), 7, dtype=torch.uint8, device=DEV)
    out = room.view(E4)[1:71, 5:205]
    scale = torch.full((2, 72), 5.0, device=DEV)
    Q, S = st.quantize_fp8(x.to(DEV), out=out, scale_out=scale[:, 1:71].t())
    assert Q.data_ptr() == out.data_ptr()
    q, s = plain_quantize(x, (1, 128), E4)
    same_codes(out, q)
    assert torch.equal(S.cpu(), s)
    keep = room.clone()
    keep[1:71, 5:205] = 7
    assert (keep == 7).all() and (scale[:, 0] == 5).all() and (scale[:, 71] == 5).all()  # nothing around them


# ------------------------------------------------------------------ product
def codes(rows, cols, dtype, seed):
    """8-bit codes over the whole range of a quantised block, NaN-free, on the CPU."""
    x = torch.randn(rows, cols, generator=gen(seed)) * LIMIT[dtype] / 4
    return x.clamp(-LIMIT[dtype], LIMIT[dtype]).to(dtype)


def scales(rows, cols, seed):
    return torch.exp(torch.randn(rows, cols, generator=gen(seed))) * 1e-3


def expand(s, rows, k):
    """Scales [rows or blocks of rows, K blocks] for each element of [rows, k]."""
    if s.shape[0] != rows:
        s = s.repeat_interleave(128, 0)[:rows]
    return s.repeat_interleave(128, 1)[:, :k]


def check_product(C, a, b, sa, sb, bias, out_dtype):
    """a [M, K], b [N, K], sa, sb by rows, all on the CPU; see the file's head for the bound."""
    m, k = a.shape
    n = b.shape[0]
    fa = a.double() * expand(sa, m, k).double()
    fb = b.double() * expand(sb, n, k).double()
    fa, fb = fa.to(DEV), fb.to(DEV)
    want, mass = fa @ fb.t(), fa.abs() @ fb.abs().t()
    if bias is not None:
        want = want + bias.double().to(DEV)
        mass = mass + bias.double().abs().to(DEV)
    bound = (min(k, 128) + -(-k // 128) + 4) * 2.0 ** -23 * mass
    half = torch.finfo(out_dtype).eps / 2 * (want.abs() + bound) + torch.finfo(out_dtype).smallest_normal * torch.finfo(out_dtype).eps
    assert C.dtype == out_dtype and C.shape == (m, n)
    worst = ((C.double() - want).abs() - bound - half).max().item() if C.numel() else -1
    assert worst <= 0, worst


def make(m, n, k, ta=E4, tb=E4, a_square=False, b_square=True, seed=0):
    a, b = codes(m, k, ta, seed + 1), codes(n, k, tb, seed + 2)
    kb = -(-k // 128)
    sa = scales(-(-m // 128) if a_square else m, kb, seed + 3)
    sb = scales(-(-n // 128) if b_square else n, kb, seed + 4)
    return a, b, sa, sb


def put(t, by_rows=True, aligned=True):
    """A copy of t [r, c] on the GPU with its rows (columns) contiguous, on 16-byte boundaries or one byte off."""
    src = t if by_rows else t.t()
    ld = -(-src.shape[1] // 16) * 16 + (0 if aligned else 3)
    room = torch.zeros(src.shape[0] * ld + 64, dtype=torch.uint8, device=DEV)
    room[:] = 0x7F  # NaN around the data
    v = room.view(t.dtype)[0 if aligned else 1:].as_strided(src.shape, (ld, 1))
    v.copy_(src.to(DEV))
    return v if by_rows else v.t()


SHAPES = [(1, 1, 1), (1, 16, 128), (1, 130, 129), (7, 129, 300), (16, 256, 1024), (17, 384, 511), (33, 100, 640),
          (64, 200, 4096), (65, 70, 33), (128, 128, 128), (129, 257, 1000), (300, 1, 400), (255, 513, 2048), (1, 640, 8192)]


@pytest.mark.parametrize("b_square", [True, False], ids=["b128", "b1"])
@pytest.mark.parametrize("m,n,k", SHAPES, ids=lambda v: str(v))
def test_matmul_shapes(m, n, k, b_square):
    a, b, sa, sb = make(m, n, k, b_square=b_square)
    C = st.matmul_fp8(put(a), put(b).t(), sa.to(DEV), sb.t().to(DEV), out_dtype=torch.float32)
    check_product(C, a, b, sa, sb, None, torch.float32)


@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("ta,tb", [(E4, E4), (E5, E4), (E4, E5), (E5, E5)], ids=["44", "54", "45", "55"])
@pytest.mark.parametrize("m", [5, 150])
def test_matmul_types_and_bias(m, ta, tb, out):
    a, b, sa, sb = make(m, 200, 700, ta, tb)
    sa, sb = sa * 1e-2, sb * (1e-2 if E5 not in (ta, tb) else 1e-6)  # inside float16's range
    for bias in (None, torch.randn(200, generator=gen(9)), torch.randn(200, generator=gen(9)).to(out)):
        C = st.matmul_fp8(put(a), put(b).t(), sa.to(DEV), sb.t().to(DEV), None if bias is None else bias.to(DEV), out_dtype=out)
        check_product(C, a, b, sa, sb, bias, out)


@pytest.mark.parametrize("aligned", [True, False], ids=["aligned", "off"])
@pytest.mark.parametrize("a_rows", [True, False], ids=["aK", "aM"])
@pytest.mark.parametrize("b_rows", [True, False], ids=["bK", "bN"])
@pytest.mark.parametrize("b_square", [True, False], ids=["b128", "b1"])
@pytest.mark.parametrize("m,n,k", [(3, 150, 260), (40, 130, 500), (200, 300, 333), (130, 20, 129)], ids=lambda v: str(v))
def test_matmul_layouts(m, n, k, b_square, b_rows, a_rows, aligned):
    a, b, sa, sb = make(m, n, k, b_square=b_square)
    C = st.matmul_fp8(put(a, a_rows, aligned), put(b, b_rows, aligned).t(), sa.to(DEV), sb.t().to(DEV), out_dtype=torch.float32)
    check_product(C, a, b, sa, sb, None, torch.float32)


def test_matmul_strided_broadcast_and_square_a():
    a, b, sa, sb = make(140, 150, 300, a_square=True)
    wide_a = torch.zeros(140, 600, dtype=torch.uint8, device=DEV).view(E4)
    wide_a[:, ::2].copy_(a.to(DEV))
    C = st.matmul_fp8(wide_a[:, ::2], put(b).t(), sa.to(DEV), sb.t().to(DEV), out_dtype=torch.float32)
    check_product(C, a, b, sa, sb, None, torch.float32)
    one = a[:1].expand(140, -1)
    s1 = sa[:1].expand(2, -1)
    C = st.matmul_fp8(put(a)[:1].expand(140, -1), put(b).t(), s1.to(DEV), sb.t().to(DEV), out_dtype=torch.float32)
    check_product(C, one, b, s1, sb, None, torch.float32)


def test_matmul_overlapping_rows():
    """Rows of A that overlap (a window moving by 16) are copied, not read as a matrix of separate rows."""
    a, b, sa, sb = make(1, 150, 2400)
    line = put(a)[0]
    _, _, sa, _ = make(100, 150, 800)
    b, sb = b[:, :800], sb[:, :7]
    C = st.matmul_fp8(line.as_strided((100, 800), (16, 1)), put(b).t(), sa.to(DEV), sb.t().to(DEV), out_dtype=torch.float32)
    rows = torch.stack([a[0, 16 * i:16 * i + 800].float() for i in range(100)]).to(E4)
    check_product(C, rows, b, sa, sb, None, torch.float32)


def test_first_call_may_be_captured():
    """In a process of its own: each operator's first call inside a graph capture."""
    code = """
import torch, sptiles_b200 as st
dev = torch.device('cuda:0')
torch.manual_seed(0)
x = torch.randn(300, 1024, device=dev, dtype=torch.bfloat16)
w = torch.randn(256, 1024, device=dev, dtype=torch.bfloat16)
p = torch.ones(1024, device=dev, dtype=torch.bfloat16)
s = torch.cuda.Stream()
torch.cuda.synchronize()
st.runtime.context(0)
def step():
    wq, ws = st.quantize_fp8(w, block=(128, 128))
    f = st.residual_norm(x, x, p, p, p, quantize=True)
    y = st.matmul_fp8(f.normed, wq.t(), f.scale, ws.t())
    return y, *st.residual_norm_backward(x, x, x, f.residual, p, p, p)
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g, stream=s):
    out = step()
g.replay()
torch.cuda.synchronize()
want = step()
assert all(torch.equal(a, b) for a, b in zip(out, want))
print('captured')
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300,
                          cwd=str(Path(__file__).resolve().parents[1]))
    assert done.returncode == 0 and "captured" in done.stdout, done.stdout + done.stderr


def test_matmul_output_view_and_edges():
    """C inside a larger array: nothing around it is written, whatever the tile."""
    for m, n in [(3, 70), (130, 140), (20, 131)]:
        a, b, sa, sb = make(m, n, 200)
        room = torch.full((m + 2, n + 9), 3.0, device=DEV)
        st.matmul_fp8(put(a), put(b).t(), sa.to(DEV), sb.t().to(DEV), out=room[1:m + 1, 4:n + 4])
        check_product(room[1:m + 1, 4:n + 4], a, b, sa, sb, None, torch.float32)
        room[1:m + 1, 4:n + 4] = 3.0
        assert (room == 3.0).all()


@pytest.mark.parametrize("n,k", [(20000, 130), (12000, 4200), (8000, 2100), (300, 4096)], ids=lambda v: str(v))
def test_matmul_one_row_as_a_column(n, k):
    """C [1, N] with unit strides both ways (a column's transpose), with a bias: the weights' rows in one, two, four and
    eight parts."""
    a, b, sa, sb = make(1, n, k)
    bias = torch.randn(n, generator=gen(9))
    room = torch.full((n + 2, 1), 3.0, device=DEV)
    out = room[1:n + 1].t()
    assert out.stride() == (1, 1)
    st.matmul_fp8(put(a), put(b).t(), sa.to(DEV), sb.t().to(DEV), bias.to(DEV), out=out)
    check_product(out, a, b, sa, sb, bias, torch.float32)
    assert room[0] == 3.0 and room[-1] == 3.0


@pytest.mark.parametrize("m", [1, 40, 64])
def test_matmul_one_column(m):
    a, b, sa, sb = make(m, 1, 2000)
    bias = torch.randn(1, generator=gen(9))
    C = st.matmul_fp8(put(a), put(b).t(), sa.to(DEV), sb.t().to(DEV), bias.to(DEV), out_dtype=torch.float32)
    check_product(C, a, b, sa, sb, bias, torch.float32)


def test_matmul_empty():
    z = torch.zeros
    A, B = z(4, 0, dtype=torch.uint8, device=DEV).view(E4), z(0, 6, dtype=torch.uint8, device=DEV).view(E4)
    bias = torch.arange(6.0, device=DEV)
    C = st.matmul_fp8(A, B, z(4, 0, device=DEV), z(0, 6, device=DEV), bias, out_dtype=torch.float32)
    assert torch.equal(C, bias.expand(4, 6))
    assert (st.matmul_fp8(A, B, z(4, 0, device=DEV), z(0, 1, device=DEV)) == 0).all()
    A, B = z(0, 130, dtype=torch.uint8, device=DEV).view(E4), z(130, 6, dtype=torch.uint8, device=DEV).view(E4)
    assert st.matmul_fp8(A, B, z(0, 2, device=DEV), z(2, 6, device=DEV)).shape == (0, 6)


def test_matmul_nan_stays_in_its_row_and_column():
    a, b, sa, sb = make(40, 300, 512)
    A, B = put(a), put(b)
    A[3, 100] = float("nan")
    SB = sb.to(DEV)
    SB[1, 2] = float("inf")  # columns 128 .. 255
    C = st.matmul_fp8(A, B.t(), sa.to(DEV), SB.t(), out_dtype=torch.float32)
    bad = ~torch.isfinite(C)
    assert bad[3].all() and bad[:, 128:256].all()
    bad[3], bad[:, 128:256] = False, False
    assert not bad.any()


@pytest.mark.parametrize("b_square", [True, False], ids=["b128", "b1"])
@pytest.mark.parametrize("m,n", [(3, 300), (150, 200), (2048, 1800)], ids=str)
def test_matmul_scales_at_the_ends_of_their_range(m, n, b_square):
    """Products of two scales down to 2^-126 and up to 2^90, from factors far apart and near each other: as exact as
    any.  (300 products of codes up to 448 sum to less than 2^26, so 2^90 times that stays finite.)"""
    k = 300
    for ea, eb in [(-63, -63), (-126, 0), (0, -126), (-126, 60), (100, -126), (45, 45), (90, 0)]:
        a, b, sa, sb = make(m, n, k, b_square=b_square)
        sa, sb = torch.full_like(sa, 2.0 ** ea), torch.full_like(sb, 2.0 ** eb)
        C = st.matmul_fp8(put(a), put(b).t(), sa.to(DEV), sb.t().to(DEV), out_dtype=torch.float32)
        check_product(C, a, b, sa, sb, None, torch.float32)


@pytest.mark.parametrize("b_square", [True, False], ids=["b128", "b1"])
@pytest.mark.parametrize("m,n", [(3, 300), (150, 200), (2048, 1800)], ids=str)
def test_matmul_blocks_of_zeros(m, n, b_square):
    """Tokens and weights of zeros carry the least scale, 2^-126: their products with any other are 0."""
    x, w = torch.randn(m, 300, generator=gen(1)), torch.randn(n, 300, generator=gen(2)) * 1e-3
    x[m // 2], x[0, :128], w[:128] = 0, 0, 0
    xq, xs = st.quantize_fp8(x.to(DEV))
    wq, ws = st.quantize_fp8(w.to(DEV), block=(128, 128) if b_square else (1, 128))
    assert xs[m // 2, 0] == 2.0 ** -126 and ws[0, 0] == 2.0 ** -126
    C = st.matmul_fp8(xq, wq.t(), xs, ws.t(), out_dtype=torch.float32)
    assert (C[m // 2] == 0).all() and (C[:, :128] == 0).all()
    check_product(C, xq.cpu(), wq.cpu(), xs.cpu(), ws.cpu(), None, torch.float32)


def test_matmul_same_bits_streams_and_graph():
    a, b, sa, sb = make(24, 1000, 4000)
    A, B, SA, SB = put(a, aligned=False), put(b).t(), sa.to(DEV), sb.t().to(DEV)
    first = st.matmul_fp8(A, B, SA, SB)
    assert torch.equal(first, st.matmul_fp8(A, B, SA, SB))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        assert torch.equal(first, st.matmul_fp8(A, B, SA, SB))
        for _ in range(2):  # two graphs with workspaces of their own, replayed side by side
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                C = st.matmul_fp8(A, B, SA, SB)
            graphs.append((g, C))
    torch.cuda.synchronize()
    for g, C in graphs:
        C.zero_()
    torch.cuda.synchronize()
    other = torch.cuda.Stream()
    for _ in range(20):
        for (g, C), s in zip(graphs, (side, other)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for g, C in graphs:
        assert torch.equal(first, C)


def test_layer_forward_and_gradients():
    """quantize_fp8 and matmul_fp8 as a layer uses them, against the product of the dequantised values."""
    m, n, k = 200, 264, 392
    x, w, dy = (torch.randn(*s, generator=gen(i)).to(torch.bfloat16) for i, s in enumerate([(m, k), (n, k), (m, n)]))
    X, W, DY = x.to(DEV), w.to(DEV), dy.to(DEV)
    Wq, Ws = st.quantize_fp8(W, block=(128, 128))
    xq, xs = st.quantize_fp8(X)
    y = st.matmul_fp8(xq, Wq.t(), xs, Ws.t(), out_dtype=torch.float32)
    check_product(y, xq.cpu(), Wq.cpu(), xs.cpu(), Ws.cpu(), None, torch.float32)
    gq, gs = st.quantize_fp8(DY, dtype=E5)
    dx = st.matmul_fp8(gq, Wq, gs, Ws, out_dtype=torch.float32)
    check_product(dx, gq.cpu(), Wq.cpu().t(), gs.cpu(), Ws.cpu().t(), None, torch.float32)
    gq, gs = st.quantize_fp8(DY, block=(128, 1), dtype=E5)
    xq, xs = st.quantize_fp8(X, block=(128, 1))
    dw = st.matmul_fp8(gq.t(), xq, gs.t(), xs, out_dtype=torch.float32)
    check_product(dw, gq.cpu().t(), xq.cpu().t(), gs.cpu().t(), xs.cpu().t(), None, torch.float32)
    # and near the unquantised gradients: two roundings of relative 2^-4 (e4m3) and 2^-3 (e5m2), largest in a block,
    # each term at most 2^-4 + 2^-3 + 2^-7 off
    for got, want, mass in [(dx, dy.double() @ w.double(), dy.double().abs() @ w.double().abs()),
                            (dw, dy.double().t() @ x.double(), dy.double().abs().t() @ x.double().abs())]:
        assert ((got.cpu().double() - want).abs() <= (2 ** -4 + 2 ** -3 + 2 ** -7 + 2 ** -8) * mass).all()


# 256 x 256 tiles of CTA pairs: enough of them, ragged at every edge, one and many blocks of K
LARGE = [(2048, 1800, 100), (1793, 2100, 384), (3000, 1300, 1111), (2047, 2049, 2048)]


@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("b_square", [True, False], ids=["b128", "b1"])
@pytest.mark.parametrize("m,n,k", LARGE, ids=lambda v: str(v))
def test_matmul_large(m, n, k, b_square, out):
    a, b, sa, sb = make(m, n, k, E5, E4, b_square=b_square)
    bias = torch.randn(n, generator=gen(9)) if k < 1000 else None
    A, B, SA, SB = put(a), put(b).t(), sa.to(DEV), sb.t().to(DEV)
    ld = -(-n // 8) * 8
    for room in (torch.full((m, ld), 3.0, dtype=out, device=DEV), torch.full((m, n + 1), 3.0, dtype=out, device=DEV)):
        C = room[:, :n]  # rows on 16-byte boundaries, and (for odd n) not
        st.matmul_fp8(A, B, SA, SB, None if bias is None else bias.to(DEV), out=C)
        check_product(C, a, b, sa, sb, bias, out)
        assert (room[:, n:] == 3.0).all()


@pytest.mark.parametrize("a_rows", [True, False], ids=["aK", "aM"])
@pytest.mark.parametrize("b_rows", [True, False], ids=["bK", "bN"])
@pytest.mark.parametrize("b_square", [True, False], ids=["b128", "b1"])
def test_matmul_large_layouts(b_square, b_rows, a_rows):
    m, n, k = 2050, 1810, 900
    a, b, sa, sb = make(m, n, k, a_square=b_rows, b_square=b_square)
    C = st.matmul_fp8(put(a, a_rows), put(b, b_rows, aligned=a_rows).t(), sa.to(DEV), sb.t().contiguous().to(DEV), out_dtype=torch.float32)
    check_product(C, a, b, sa, sb, None, torch.float32)


# ------------------------------------------------------------------ offsets past 32 bits
def some_codes(rows, cols, seed):
    """Codes below 2 in magnitude (so none is NaN), made on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(0, 256, (rows, cols), generator=g, device=DEV, dtype=torch.uint8).bitwise_and_(0xBF).view(E4)


@pytest.mark.parametrize("block", [(1, 128), (128, 1), (128, 128)], ids=["row", "column", "square"])
def test_quantize_many_elements(block):
    rows, cols, first = 140000, 16384, 139904
    x = torch.randn(rows, cols, device=DEV, dtype=torch.bfloat16)
    Q, S = st.quantize_fp8(x, block=block)
    q, s = plain_quantize(x[first:].cpu(), block, E4)
    same_codes(Q[first:], q)
    assert torch.equal(S[-s.shape[0]:].cpu(), s)


def test_quantize_longest_row():
    cols = 2 ** 31 - 1
    x = torch.zeros(1, cols, device=DEV, dtype=torch.bfloat16)
    tail = torch.randn(1, 127 + 256, generator=gen(3)).to(torch.bfloat16)
    x[:, -tail.shape[1]:] = tail.to(DEV)
    Q, S = st.quantize_fp8(x)
    q, s = plain_quantize(tail, (1, 128), E4)
    same_codes(Q[:, -tail.shape[1]:], q)
    assert torch.equal(S[:, -3:].cpu(), s) and (S[:, :-3] == 2.0 ** -126).all()


@pytest.mark.parametrize("aligned", [True, False], ids=["aligned", "off"])
def test_matmul_many_weights(aligned):
    m, n, k, last = 3, 270000, 8192, 300
    a, _, sa, _ = make(m, 1, k)
    ld = k if aligned else k + 1
    w = some_codes(1, n * ld, 1).as_strided((n, k), (ld, 1))
    sb = torch.rand(n, k // 128, device=DEV)
    C = st.matmul_fp8(put(a), w.t(), sa.to(DEV), sb.t(), out_dtype=torch.float32)
    check_product(C[:, -last:], a, w[-last:].cpu(), sa, sb[-last:].cpu(), None, torch.float32)


def test_matmul_many_results():
    m, n, k, last = 33000, 66000, 128, 300
    a, w = some_codes(m, k, 1), some_codes(n, k, 2)
    sa, sb = torch.rand(m, 1, device=DEV), torch.rand(-(-n // 128), 1, device=DEV)
    C = st.matmul_fp8(a, w.t(), sa, sb.t())
    part = sb.repeat_interleave(128, 0)[:n][-last:]
    check_product(C[-last:, -last:], a[-last:].cpu(), w[-last:].cpu(), sa[-last:].cpu(), part.cpu(), None, torch.bfloat16)
