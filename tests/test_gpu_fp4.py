"""4-bit blocks and their product on the GPU against plain computations.

The quantiser is compared bit for bit with a float64 computation on the CPU:
a tensor scale and an e8m0 scale are powers of two and a code's border times
the scale has at most seven bits, so every comparison below is exact.  Products
of integers whose sums stay below 2^24 of their least step are exact in fp32
and compared for equality.  Other products: each fp32 addition is off by at
most 2^-23 of the sum of the terms' magnitudes (a truncating adder), so a
K-term sum by (K + 4) 2^-23 sum |a b|, the tensor scales' product included; the
result's rounding adds half a step, eps / 2 relative."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import sptiles_b200 as st

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
E4, E8, CODES = torch.float8_e4m3fn, torch.float8_e8m0fnu, torch.float4_e2m1fn_x2
LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
BLOCK = {E4: 16, E8: 32}


def gen(seed):
    return torch.Generator().manual_seed(seed)


# ------------------------------------------------------------------ plain forms
def nearest(y, levels):
    """Index of the level nearest to y >= 0; ties to the even index; above the last, the last."""
    lv = torch.tensor(levels, dtype=torch.float64)
    hi = torch.searchsorted(lv, y.contiguous()).clamp(max=len(levels) - 1)
    lo = (hi - 1).clamp(min=0)
    up, down = lv[hi] - y, y - lv[lo]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)


E4M3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1]


def least_power(top, limit, least):
    e = least
    while limit * 2.0 ** e < top:
        e += 1
    return e


def plain_quantize(x, scale_dtype, amax=None):
    """(codes 0..15 [rows, cols], scale bytes [rows, blocks], tensor scale) in float64."""
    x = x.double()
    rows, cols = x.shape
    b = BLOCK[scale_dtype]
    parts = torch.nn.functional.pad(x, (0, -cols % b)).view(rows, -1, b)
    top = parts.abs().amax(2)
    bad = ~torch.isfinite(top)
    if b == 16:
        m = x[torch.isfinite(x)].abs().max().item() if amax is None else amax
        t = 2.0 ** least_power(m, 2688.0, -126) if m > 0 else 1.0
        byte = nearest(torch.where(bad, 0.0, top) / (6 * t), E4M3)
        unit = torch.tensor(E4M3, dtype=torch.float64)[byte] * t
        byte = torch.where(bad, 0x7f, byte)
    else:
        t = None
        e = torch.tensor([[least_power(0.0 if not torch.isfinite(v) else v.item(), 6.0, -127) for v in row] for row in top])
        byte, unit = torch.where(bad, 255, e + 127), torch.pow(torch.tensor(2.0, dtype=torch.float64), e.double())
    live = unit > 0
    q = torch.where(bad[:, :, None], 0.0, parts) / torch.where(live, unit, 1.0)[:, :, None]
    code = nearest(q.abs(), LEVELS) + 8 * torch.signbit(parts)
    code = torch.where(live[:, :, None], code, code & 8)
    return code.view(rows, -1)[:, :cols], byte, t, bad.repeat_interleave(b, 1)[:, :cols]


def tiled(byte):
    rows, blocks = byte.shape
    byte = torch.nn.functional.pad(byte.to(torch.uint8), (0, -blocks % 4, 0, -rows % 128))
    return byte.view(-(-rows // 128), 4, 32, -(-blocks // 4), 4).permute(0, 3, 2, 1, 4).contiguous()


def untiled(scale, rows, blocks):
    byte = scale.view(torch.uint8).cpu()
    i, j = byte.shape[:2]
    return byte.permute(0, 3, 2, 1, 4).reshape(128 * i, 4 * j)[:rows, :blocks]


def split(codes, cols):
    byte = codes.view(torch.uint8).cpu()
    return torch.stack((byte & 15, byte >> 4), 2).flatten(1), cols


def check_quantize(x, scale_dtype, amax=None, where=None):
    got = st.quantize_fp4(x.to(DEV) if where is None else where, scale_dtype=scale_dtype,
                          amax=None if amax is None else torch.tensor(amax, device=DEV))
    code, byte, t, bad = plain_quantize(x, scale_dtype, amax)
    rows, cols = x.shape
    assert got.codes.dtype == CODES and got.codes.shape == (rows, (cols + 1) // 2) and got.scale.dtype == scale_dtype
    assert (got.tensor_scale is None) == (t is None)
    if t is not None:
        assert got.tensor_scale.item() == t
    assert torch.equal(got.scale.view(torch.uint8).cpu(), tiled(byte))  # zeros where no row or block is
    halves, _ = split(got.codes, cols)
    assert (halves[:, cols:] == 0).all()
    assert torch.equal(torch.where(bad, 0, halves[:, :cols].long()), torch.where(bad, 0, code.long()))
    return got


SRC = [torch.float32, torch.float16, torch.bfloat16]


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
@pytest.mark.parametrize("src", SRC, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 16), (3, 33), (127, 64), (128, 128), (130, 257), (301, 136), (5, 4096)])
def test_quantize_bits(rows, cols, src, scale_dtype):
    x = (torch.randn(rows, cols, generator=gen(rows + cols)) * torch.exp(2 * torch.randn(rows, 1, generator=gen(7)))).to(src)
    check_quantize(x, scale_dtype)


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
@pytest.mark.parametrize("src", SRC, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("view", ["transposed", "transposed offset", "strided", "offset", "broadcast", "broadcast column"])
def test_quantize_views(view, src, scale_dtype):
    base = torch.randn(301, 406, generator=gen(3)).to(src)
    cut = {"transposed": lambda t: t.t(), "transposed offset": lambda t: t[1:, 1:].t(), "strided": lambda t: t[::2, ::3],
           "offset": lambda t: t[1:, 1:], "broadcast": lambda t: t[:1].expand(140, -1),
           "broadcast column": lambda t: t[:, :1].expand(-1, 50)}[view]
    check_quantize(cut(base), scale_dtype, where=cut(base.to(DEV)))


@pytest.mark.parametrize("src", SRC, ids=["f32", "f16", "bf16"])
def test_quantize_borders(src):
    """Every border between two codes times every scale mantissa, and the elements next to it."""
    borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    rows = []
    for m in range(8, 16):
        s = torch.tensor(m / 8, dtype=src)
        at = torch.tensor(borders, dtype=src) * s
        inf, zero = torch.tensor(float("inf"), dtype=src), torch.tensor(0.0, dtype=src)
        if src == torch.bfloat16:  # no nextafter: one step of its bits
            near = (at.view(torch.int16) + 1).view(src), (at.view(torch.int16) - 1).view(src)
        else:
            near = torch.nextafter(at.float(), inf.float()).to(src) if src == torch.float32 else (at.view(torch.int16) + 1).view(src), \
                torch.nextafter(at.float(), zero.float()) if src == torch.float32 else (at.view(torch.int16) - 1).view(src)
        for v in (at, *near):
            for sign in (1, -1):
                row = torch.zeros(16, dtype=src)
                row[:7], row[15] = sign * v, 6 * s
                rows.append(row)
    x = torch.stack(rows)
    x = torch.cat((x, 448 * x / 1.75), 1) if src == torch.float32 else x
    check_quantize(x, E4, amax=2688.0)
    check_quantize(x, E4, amax=2688.0, where=x.t().contiguous().to(DEV).t())
    check_quantize(x.repeat(1, 2), E8)


def test_quantize_extremes():
    """Zero, subnormal, huge, infinite and NaN blocks; saturation at a known maximum; tensors near the ends of fp32."""
    x = torch.zeros(8, 64)
    x[1, 5], x[2], x[3, 0], x[4, 40] = 1e-45, 3e38, float("inf"), float("nan")
    x[5, :4], x[6], x[7] = torch.tensor([448.0, 17.0, 19.0, -21.0]), -0.0, 2.0 ** -130
    for dtype in (E4, E8):
        check_quantize(x, dtype)
        check_quantize(x[[0, 1, 5, 6, 7]] * 2.0 ** -100, dtype)
        check_quantize(x[[0, 6]], dtype)
        check_quantize(torch.randn(40, 100, generator=gen(5)) * 2.0 ** -120, dtype)
        check_quantize(torch.randn(40, 100, generator=gen(5)) * 2.0 ** 124, dtype)
    got = check_quantize(torch.tensor([[100.0] * 16 + [1.0] * 16]), E4, amax=8.0)
    back = st.dequantize_fp4(got.codes, got.scale, got.tensor_scale, out_dtype=torch.float32)
    assert back[0, 0].item() == 6 * 448 * got.tensor_scale.item() < 100.0
    bad = st.dequantize_fp4(*check_quantize(x, E4))
    assert torch.isnan(bad[3, :16]).all() and torch.isnan(bad[4, 32:48]).all() and not torch.isnan(bad[4, 48:]).any()


def test_quantize_empty():
    for shape in [(0, 5), (5, 0), (0, 0)]:
        for dtype in (E4, E8):
            q = st.quantize_fp4(torch.empty(shape, device=DEV), scale_dtype=dtype)
            assert q.codes.shape == (shape[0], (shape[1] + 1) // 2)
            assert q.scale.shape == (-(-shape[0] // 128), -(-(-(-shape[1] // BLOCK[dtype])) // 4), 32, 4, 4)
            assert q.tensor_scale is None or q.tensor_scale.item() == 1.0
            assert st.dequantize_fp4(*q, cols=shape[1]).shape == shape


def test_quantize_large():
    """A tensor whose second pass walks many units a thread, and whose maximum lies in its last element."""
    x = torch.randn(4096, 2050, generator=gen(1)).to(torch.bfloat16)
    x[-1, -1] = 300.0
    got = st.quantize_fp4(x.to(DEV))
    assert got.tensor_scale.item() == 0.125
    take = [0, 1, 127, 128, 2047, 4095]
    code, byte, t, _ = plain_quantize(x[take], E4, amax=300.0)
    assert torch.equal(split(got.codes, 2050)[0][take][:, :2050].long(), code.long())
    assert torch.equal(untiled(got.scale, 4096, 129)[take].long(), byte.long())


# ------------------------------------------------------------------ back to values
def values(code, byte, t, scale_dtype):
    level = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64)[code.long()]
    scale = byte.to(torch.uint8).view(scale_dtype).double().repeat_interleave(BLOCK[scale_dtype], 1)[:, : code.shape[1]]
    return level * scale * (1.0 if t is None else t)


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
@pytest.mark.parametrize("cols", [1, 15, 31, 64, 333])
def test_dequantize(cols, scale_dtype):
    x = torch.randn(140, cols, generator=gen(cols))
    q = st.quantize_fp4(x.to(DEV), scale_dtype=scale_dtype)
    code, byte, t, _ = plain_quantize(x, scale_dtype)
    want = values(code, byte, t, scale_dtype)
    for dtype in (torch.float32, torch.bfloat16, torch.float16):  # one rounding; exact in the first two
        assert torch.equal(st.dequantize_fp4(*q, cols=cols, out_dtype=dtype).cpu(), want.float().to(dtype))
    wide = st.dequantize_fp4(*q, out_dtype=torch.float32)
    assert wide.shape == (140, cols + cols % 2) and (cols % 2 == 0 or (wide[:, -1] == 0).all())
    for turned in (q.codes.view(torch.uint8).t().contiguous().t(), q.codes.contiguous()):
        assert torch.equal(st.dequantize_fp4(turned, *q[1:], cols=cols, out_dtype=torch.float32).cpu(), want.float())


def test_dequantize_any_tensor_scale():
    q = st.quantize_fp4(torch.randn(3, 48, generator=gen(1)).to(DEV))
    t = torch.tensor([0.3], device=DEV)
    code = split(q.codes, 48)[0]
    want = values(code, untiled(q.scale, 3, 3), None, E4)
    unit = (want.float() != 0)
    got = st.dequantize_fp4(q.codes, q.scale, t, out_dtype=torch.float32).cpu()
    # scale * t and its product with the code: two roundings of half a step
    assert ((got.double() - want * t.cpu().double()).abs() <= 2.0 ** -23 * (want * 0.3).abs() * 1.0001)[unit].all()


# ------------------------------------------------------------------ the product
def random_operand(rows, cols, scale_dtype, seed):
    """Codes and scales at random, with the values they stand for; scales 0.5, 1 or 2."""
    g = gen(seed)
    b = BLOCK[scale_dtype]
    code = torch.randint(0, 16, (rows, cols), generator=g)
    power = torch.randint(-1, 2, (rows, -(-cols // b)), generator=g)
    byte = torch.pow(2.0, power).to(scale_dtype).view(torch.uint8)
    padded = torch.nn.functional.pad(code, (0, cols % 2)).to(torch.uint8)
    return padded[:, 0::2] | (padded[:, 1::2] << 4), tiled(byte).view(scale_dtype), values(code, byte, None, scale_dtype)


def aligned(codes):
    """Rows on 16-byte boundaries, as quantize_fp4 lays them out."""
    room = torch.full((codes.shape[0], (codes.shape[1] + 15) // 16 * 16), 0x77, dtype=torch.uint8, device=DEV)
    room[:, : codes.shape[1]] = codes.to(DEV)
    return room[:, : codes.shape[1]].view(CODES)


SHAPES = [(1, 1, 1), (1, 128, 64), (1, 500, 2048), (2, 129, 33), (16, 256, 256), (17, 100, 130), (33, 515, 512), (64, 128, 4096),
          (65, 127, 63), (128, 128, 1000), (200, 300, 255), (257, 129, 257), (300, 513, 96), (1000, 520, 1111), (1, 4100, 6000)]


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product_exact(m, n, k, scale_dtype):
    qa, sa, va = random_operand(m, k, scale_dtype, 1)
    qb, sb, vb = random_operand(n, k, scale_dtype, 2)
    want = (va @ vb.t()).float()
    a, b, sa, sb = aligned(qa), aligned(qb).t(), sa.to(DEV), sb.to(DEV)
    assert torch.equal(st.matmul_fp4(a, b, sa, sb, out_dtype=torch.float32).cpu(), want)
    # operands off every boundary, and stored across K: copied first
    off = torch.zeros(qa.shape[0], qa.shape[1] + 1, dtype=torch.uint8, device=DEV)[:, 1:]
    off.copy_(qa)
    assert torch.equal(st.matmul_fp4(off, qb.t().contiguous().to(DEV), sa, sb, out_dtype=torch.float32).cpu(), want)
    bias = torch.randint(-8, 8, (n,), generator=gen(3)).float()
    got = st.matmul_fp4(a, b, sa, sb, bias.to(DEV), out_dtype=torch.float32)
    assert torch.equal(got.cpu(), want + bias)
    for dtype in (torch.bfloat16, torch.float16):
        got = st.matmul_fp4(a, b, sa, sb, bias.to(dtype).to(DEV), out_dtype=dtype)
        assert torch.equal(got.cpu(), (want + bias).to(dtype))
    if scale_dtype == E4:
        t = torch.tensor(0.25, device=DEV), torch.tensor([4.0], device=DEV)
        got = st.matmul_fp4(a, b, sa, sb, bias.to(DEV), a_tensor_scale=t[0], out_dtype=torch.float32)
        assert torch.equal(got.cpu(), 0.25 * want + bias)
        got = st.matmul_fp4(a, b, sa, sb, a_tensor_scale=t[0], b_tensor_scale=t[1], out_dtype=torch.float32)
        assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
@pytest.mark.parametrize("m,n,k", [(3, 700, 900), (130, 257, 1025), (1024, 512, 2048)])
def test_product_of_quantised(m, n, k, scale_dtype):
    """What quantize_fp4 makes, multiplied, against float64 on the values it stands for."""
    x = torch.randn(m, k, generator=gen(1)) * torch.exp(torch.randn(m, 1, generator=gen(2)))
    w = torch.randn(n, k, generator=gen(3))
    xq, wq = (st.quantize_fp4(t.to(torch.bfloat16).to(DEV), scale_dtype=scale_dtype) for t in (x, w))
    vx, vw = (st.dequantize_fp4(*q, cols=k, out_dtype=torch.float32).double() for q in (xq, wq))
    want, size = vx @ vw.t(), vx.abs() @ vw.abs().t()
    ts = {} if scale_dtype == E8 else dict(a_tensor_scale=xq.tensor_scale, b_tensor_scale=wq.tensor_scale)
    for dtype in (torch.float32, torch.bfloat16):
        got = st.matmul_fp4(xq.codes, wq.codes.t(), xq.scale, wq.scale, out_dtype=dtype, **ts).double()
        slack = (k + 4) * 2.0 ** -23 * size
        assert ((got - want).abs() <= slack + torch.finfo(dtype).eps / 2 * (want.abs() + slack)).all()


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
@pytest.mark.parametrize("m,n,k", [(1500, 1700, 64), (2311, 1025, 700), (1024, 2560, 1601), (300, 5000, 33), (4100, 258, 2048),
                                   (2560, 4096, 512)])
def test_product_exact_large(m, n, k, scale_dtype):
    """Many tiles: each CTA pair has several, cut at C's edges in both directions."""
    qa, sa, va = random_operand(m, k, scale_dtype, 1)
    qb, sb, vb = random_operand(n, k, scale_dtype, 2)
    want = (va.to(DEV) @ vb.to(DEV).t()).float()
    a, b, sa, sb = aligned(qa), aligned(qb).t(), sa.to(DEV), sb.to(DEV)
    bias = torch.randint(-8, 8, (n,), generator=gen(3)).float().to(DEV)
    assert torch.equal(st.matmul_fp4(a, b, sa, sb, out_dtype=torch.float32), want)
    assert torch.equal(st.matmul_fp4(a, b, sa, sb, bias), (want + bias).to(torch.bfloat16))
    room = torch.full((m + 2, n + 5), 7.0, dtype=torch.float16, device=DEV)
    st.matmul_fp4(a, b, sa, sb, bias, out=room[1 : m + 1, 2 : n + 2])
    assert torch.equal(room[1 : m + 1, 2 : n + 2], (want + bias).to(torch.float16))
    room[1 : m + 1, 2 : n + 2] = 7.0
    assert (room == 7).all()


@pytest.mark.parametrize("m", [127, 300])
@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
def test_product_every_scale(scale_dtype, m):
    """Each finite scale, subnormal ones among them, against a block of ones: a row's sum is its scale times the block's length."""
    b = BLOCK[scale_dtype]
    byte = torch.arange(m) % 127 if scale_dtype == E4 else 40 + torch.arange(m) % 170
    scale = byte.to(torch.uint8).view(scale_dtype).double()
    ones = torch.full((m, b // 2), 0x22, dtype=torch.uint8, device=DEV)
    one = torch.full((1, 1), 0x38 if scale_dtype == E4 else 127)
    sa, sb = tiled(byte[:, None]).view(scale_dtype).to(DEV), tiled(one.expand(40, 1)).view(scale_dtype).to(DEV)
    want = (scale * b).float()[:, None].expand(m, 40)
    assert torch.equal(st.matmul_fp4(ones, ones[:40].t(), sa, sb, out_dtype=torch.float32).cpu(), want)
    assert torch.equal(st.matmul_fp4(ones[:40], ones.t(), sb, sa, out_dtype=torch.float32).cpu(), want.t())


def test_product_nan_stays_in_its_row_and_column():
    x, w = torch.randn(40, 128, generator=gen(1)), torch.randn(300, 128, generator=gen(2))
    x[7, 100], w[129, 3] = float("nan"), float("inf")
    for dtype in (E4, E8):
        a, b = st.quantize_fp4(x.to(DEV), scale_dtype=dtype), st.quantize_fp4(w.to(DEV), scale_dtype=dtype)
        c = st.matmul_fp4(a.codes, b.codes.t(), a.scale, b.scale, out_dtype=torch.float32)
        nan = torch.isnan(c)
        assert nan[7].all() and nan[:, 129].all()
        nan[7] = nan[:, 129] = False
        assert not nan.any()


def test_product_empty_and_given_output():
    for m, n, k in [(0, 5, 64), (5, 0, 64), (5, 7, 0)]:
        qa, sa, _ = random_operand(m, k, E4, 1)
        qb, sb, _ = random_operand(n, k, E4, 2)
        bias = torch.arange(n, dtype=torch.float32, device=DEV)
        c = st.matmul_fp4(qa.to(DEV), qb.to(DEV).t(), sa.to(DEV), sb.to(DEV), bias)
        assert c.shape == (m, n) and torch.equal(c.float(), bias.expand(m, n))
    for m, n in [(70, 200), (1, 333), (300, 260)]:
        qa, sa, va = random_operand(m, 320, E4, 1)
        qb, sb, vb = random_operand(n, 320, E4, 2)
        for dtype in (torch.float32, torch.bfloat16):
            room = torch.full((m + 2, n + 9), 7.0, dtype=dtype, device=DEV)
            out = room[1 : m + 1, 3 : n + 3]
            assert st.matmul_fp4(aligned(qa), aligned(qb).t(), sa.to(DEV), sb.to(DEV), out=out) is out
            assert torch.equal(out.cpu(), (va @ vb.t()).to(dtype))
            out.fill_(7.0)
            assert (room == 7).all()


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
def test_layer_forward_and_gradients(scale_dtype):
    """y = x W^T and its gradients, each operand quantised along what is summed over, transposed views as they are
    stored; each product against float64 on the values that its operands' codes stand for."""
    tokens, n, k = 200, 136, 260
    x, w, dy = (torch.randn(*s, generator=gen(i)).to(torch.bfloat16).to(DEV) for i, s in enumerate([(tokens, k), (n, k), (tokens, n)]))

    def product(a, b):
        qa, qb = st.quantize_fp4(a, scale_dtype=scale_dtype), st.quantize_fp4(b, scale_dtype=scale_dtype)
        got = st.matmul_fp4(qa.codes, qb.codes.t(), qa.scale, qb.scale, a_tensor_scale=qa.tensor_scale, b_tensor_scale=qb.tensor_scale,
                            out_dtype=torch.float32).double()
        va, vb = (st.dequantize_fp4(*q, cols=t.shape[1], out_dtype=torch.float32).double() for q, t in ((qa, a), (qb, b)))
        # a code is at most half a step off, a step at most a third of the block's largest value; e8m0 scales up to twice
        assert ((va - a.double()).abs().amax() <= a.double().abs().amax() / 3).item()
        slack = (a.shape[1] + 4) * 2.0 ** -23 * (va.abs() @ vb.abs().t())
        assert ((got - va @ vb.t()).abs() <= slack * (1 + 2.0 ** -24) + 2.0 ** -24 * (va @ vb.t()).abs()).all()
        return got

    assert product(x, w).shape == (tokens, n)          # y
    assert product(dy, w.t()).shape == (tokens, k)     # dx
    assert product(dy.t(), x.t()).shape == (n, k)      # dW


# ------------------------------------------------------------------ streams, graphs, long tensors
def test_same_bits_streams_and_graphs():
    """Quantisers of both kinds into a product: two graphs with workspaces of their own, side by side."""
    x, w = torch.randn(300, 1000, generator=gen(1)).to(DEV), torch.randn(700, 1000, generator=gen(2)).to(DEV)

    def step():
        out = []
        for dtype in (E4, E8):
            a, b = st.quantize_fp4(x[:, 1:], scale_dtype=dtype), st.quantize_fp4(w.t()[1:].t(), scale_dtype=dtype)
            out += [a.scale.view(torch.uint8), st.matmul_fp4(a.codes[1:], b.codes.t(), st.quantize_fp4(x[1:, 1:], scale_dtype=dtype).scale, b.scale),
                    st.dequantize_fp4(*b, cols=999)]
        return out

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side, other = torch.cuda.Stream(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs = []
    with torch.cuda.stream(side):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                out = step()
            graphs.append((g, out))
    torch.cuda.synchronize()
    for _ in range(10):
        for (g, _), s in zip(graphs, (side, other)):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out in graphs:
        assert all(torch.equal(a, b) for a, b in zip(first, out))


def test_first_call_may_be_captured():
    """In a process of its own: each operator's first call inside a graph capture."""
    code = """
import torch, sptiles_b200 as st
dev = torch.device('cuda:0')
torch.manual_seed(0)
x = torch.randn(300, 1024, device=dev, dtype=torch.bfloat16)
w = torch.randn(4, 256, 1024, device=dev, dtype=torch.bfloat16)
ends = torch.tensor([10, 10, 250, 290], device=dev, dtype=torch.int32)
s = torch.cuda.Stream()
torch.cuda.synchronize()
st.runtime.context(0)
def step():
    xq, wq = st.quantize_fp4(x), st.quantize_fp4(w[0])
    y = st.matmul_fp4(xq.codes, wq.codes.t(), xq.scale, wq.scale, a_tensor_scale=xq.tensor_scale, b_tensor_scale=wq.tensor_scale)
    z = st.matmul_grouped(x, w.transpose(1, 2), ends)
    return y, z, st.dequantize_fp4(*xq), st.matmul_grouped_weights(z, x, ends)
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


def some_codes(rows, cols, seed):
    return torch.randint(0, 256, (rows, cols), generator=torch.Generator(DEV).manual_seed(seed), device=DEV, dtype=torch.uint8)


@pytest.mark.parametrize("scale_dtype", [E4, E8], ids=["16", "32"])
@pytest.mark.parametrize("stored", ["rows", "columns", "off"])
def test_quantize_many_elements(stored, scale_dtype):
    """More than 2^31 elements; the last rows against the plain form."""
    rows, cols, first = 140000, 16384, 139904
    if stored == "columns":
        x = torch.randn(cols, rows, device=DEV, dtype=torch.bfloat16).t()
    else:
        x = torch.randn(rows, cols + (stored == "off"), device=DEV, dtype=torch.bfloat16)[:, -cols:]
    amax = torch.tensor(8.0, device=DEV) if scale_dtype == E4 else None
    got = st.quantize_fp4(x, scale_dtype=scale_dtype, amax=amax)
    code, byte, t, _ = plain_quantize(x[first:].cpu(), scale_dtype, 8.0)
    assert torch.equal(split(got.codes[first:], cols)[0].long(), code.long())
    assert torch.equal(untiled(got.scale[first // 128 :], rows - first, byte.shape[1]).long(), byte.long())
    back = st.dequantize_fp4(*got)
    assert torch.equal(back[first:].cpu(), values(code, byte, t, scale_dtype).to(torch.bfloat16))


def test_maximum_of_many_elements():
    x = torch.zeros(140000, 16384, device=DEV, dtype=torch.bfloat16)
    x[139999, 16383], x[0, 0] = 2689.0 * 4, float("inf")
    # 10756 lies 4 above 10752, bf16's numbers there 64 apart: it is 10752 = 2688 * 4 that is stored
    assert x[139999, 16383].item() == 2688 * 4
    assert st.quantize_fp4(x).tensor_scale.item() == 4.0


@pytest.mark.parametrize("aligned", [True, False], ids=["aligned", "off"])
def test_product_many_weights(aligned):
    m, n, kb, last = 3, 270000, 16384, 300
    ld = kb if aligned else kb + 1
    w = some_codes(1, n * ld, 1).as_strided((n, kb), (ld, 1))
    qa, sa, va = random_operand(m, 2 * kb, E4, 2)
    sb = torch.full((-(-n // 128), kb // 32, 32, 4, 4), 1.0, device=DEV).to(E4)
    c = st.matmul_fp4(qa.to(DEV), w.t(), sa.to(DEV), sb, out_dtype=torch.float32)
    vb = values(split(w[-last:].cpu(), 2 * kb)[0], torch.full((last, kb // 8), 0x38), None, E4)
    assert torch.equal(c[:, -last:].cpu(), (va @ vb.t()).float())


def test_product_many_results():
    m, n, k, last = 33000, 66000, 128, 300
    a, b = some_codes(m, k // 2, 1), some_codes(n, k // 2, 2)
    one = lambda rows: torch.ones(-(-rows // 128), 2, 32, 4, 4, device=DEV).to(E4)  # noqa: E731
    c = st.matmul_fp4(a, b.t(), one(m), one(n))
    ones = torch.full((last, k // 16), 0x38)
    va, vb = (values(split(t[-last:].cpu(), k)[0], ones, None, E4) for t in (a, b))
    assert torch.equal(c[-last:, -last:].cpu(), (va @ vb.t()).float().to(torch.bfloat16))


@pytest.mark.parametrize("src", SRC, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["rows", "columns behind the last word", "transposed", "strided"])
def test_maximum_beside_infinities(layout, src):
    """The largest finite element counts wherever it lies, also among the elements that a CTA takes together with an infinity."""
    rows, cols = 2050, 4096
    base = torch.empty(rows, cols + 8, dtype=src, device=DEV).uniform_(-1, 1)
    x = {"rows": base[:, :cols], "columns behind the last word": base[:, : cols + 3], "transposed": base[:, :cols].t(),
         "strided": base[:, ::2]}[layout]
    odd = base.shape[1] // 2 - 1 if layout == "strided" else x.shape[1] - 1
    last = (x.shape[0] - 1, odd)
    # 2000 and 1500: a CTA's first 16-byte words hold the first 1024 elements of f32, or 2048 of 16 bits
    first = [(j, 0) if layout == "transposed" else (0, j) for j in (1, 255, 256, 300, 777, 1023, 1500, 2000)]
    for at in [*first, (1, 1), (3, odd), (odd % x.shape[0], 7), last]:
        for bad in (float("inf"), float("-inf")):
            kept = x[at].clone(), x[0, 0].clone()
            x[at], x[0, 0] = 1000.0, bad
            assert st.quantize_fp4(x).tensor_scale.item() == 0.5, at  # 2688 / 2 >= 1000 > 2688 / 4
            x[at], x[0, 0] = kept
    x[::7, ::5] = float("inf")
    x[last] = 1000.0
    assert st.quantize_fp4(x).tensor_scale.item() == 0.5


@pytest.mark.parametrize("src", SRC, ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("layout", ["whole rows", "rows", "columns", "columns off", "strided"])
@pytest.mark.parametrize("amax", [0.0, 1e-38, 1e-30, 1e-20, 1.0, 8.0])
def test_quantize_far_above_the_maximum(amax, layout, src):
    """Elements however far above a known maximum saturate with their sign; those beside them are as they are without."""
    most = torch.finfo(src).max
    x = torch.randn(40, 96 if layout == "whole rows" else 91, generator=gen(11)) * max(amax, 2.0 ** -126)
    for i, v in enumerate([4.0, -4.0, 1e9, -1e9, most, -most, 2.0 ** 28, -3.0 * 2.0 ** 60]):
        x[i, 3 * i], x[i, 40], x[8 + i, 50] = v, -v, v
    x[20, :16], x[21, 16:32] = most, -most
    x[22, 5], x[22, 6] = float("inf"), most
    x[23, 33], x[23, 34] = float("nan"), -most
    x = x.clamp(-most, most).where(torch.isfinite(x), x).to(src)
    turned = x.t().contiguous()
    off = torch.zeros(turned.shape[0], 41, dtype=src)
    off[:, 1:] = turned
    wide = torch.zeros(40, 2 * x.shape[1], dtype=src)
    wide[:, ::2] = x
    where = {"whole rows": lambda: x.to(DEV), "rows": lambda: x.to(DEV), "columns": lambda: turned.to(DEV).t(),
             "columns off": lambda: off.to(DEV)[:, 1:].t(), "strided": lambda: wide.to(DEV)[:, ::2]}[layout]()
    got = check_quantize(x, E4, amax=torch.tensor(amax).item(), where=where)
    back = st.dequantize_fp4(got.codes, got.scale, got.tensor_scale, cols=x.shape[1], out_dtype=torch.float32).cpu()
    fine = torch.isfinite(x.float())
    assert torch.isfinite(back[fine.view(40, -1).all(1)]).all()
    assert (back[20, :16] > 0).all() and (back[21, 16:32] < 0).all()


@pytest.mark.parametrize("layout", ["rows", "columns", "strided"])
def test_scales_beyond_32_bits(layout):
    """A row of 2^29 elements, padded to 128, has 2^32 bytes of scales: both ends of longer ones against the same columns alone."""
    rows, cols, cut = 2, 2 ** 29 + 4096, 4096
    shape = {"rows": (rows, cols), "columns": (cols, rows), "strided": (rows, 2 * cols)}[layout]
    x = torch.empty(shape, dtype=torch.bfloat16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(1))
    x = {"rows": x, "columns": x.t(), "strided": x[:, ::2]}[layout]
    amax = torch.tensor(8.0, device=DEV)
    got = st.quantize_fp4(x, amax=amax)
    assert got.scale.numel() > 2 ** 32
    back = st.dequantize_fp4(*got)
    quads, half = cut // 64, cut // 2  # groups of four scales, bytes of codes
    for first, quad in [(0, 0), (cols - cut, got.scale.shape[1] - quads)]:
        alone = st.quantize_fp4(x[:, first : first + cut], amax=amax)
        assert torch.equal(got.scale[:, quad : quad + quads].view(torch.uint8), alone.scale.view(torch.uint8))
        assert torch.equal(got.codes[:, first // 2 : first // 2 + half].view(torch.uint8), alone.codes.view(torch.uint8))
        assert torch.equal(back[:, first : first + cut], st.dequantize_fp4(*alone))
    del back
    # ones at both ends and zeros between them, the last columns' scales 2: the product is exact
    codes, scale = got.codes.view(torch.uint8), got.scale.view(torch.uint8)
    codes.zero_()
    codes[:, :half], codes[:, -half:] = 0x22, 0x22
    scale.fill_(0x38)
    scale[:, -quads:] = 0x40
    c = st.matmul_fp4(codes, codes.t(), got.scale, got.scale, out_dtype=torch.float32)
    assert torch.equal(c, torch.full((rows, rows), cut * 1.0 + cut * 4.0, device=DEV))


@pytest.mark.parametrize("m,n", [(1, 300), (40, 300), (200, 130), (2048, 2560)])
@pytest.mark.parametrize("ta,tb", [(-70, -70), (-80, -76), (-126, -30), (-30, -126), (65, 65), (117, 15), (15, 117), (117, 20), (20, 117),
                                   (-126, 117)])
def test_product_of_far_tensor_scales(ta, tb, m, n):
    """Tensor scales whose product leaves fp32's range, where the result does not; a sum of nothing stays 0.

    Sums and scales are powers of two, or those times 49, so a result is exact, or, of 117 and 20, 2^-7 2^137: infinite in fp32."""
    k, up = 2048, ta + tb < 0
    qa, qb = torch.zeros(m, k, dtype=torch.uint8), torch.zeros(n, k, dtype=torch.uint8)
    qa[::2], qb[::3] = 2, 2  # rows of ones and of zeros
    byte = 0x7e if up else 1  # 448 and 2^-9: sums of 2048 * 448^2, about 2^28.6, or of 2^11 * 2^-18
    sa, sb = (tiled(torch.full((r, k // 16), byte)).view(E4).to(DEV) for r in (m, n))
    scale = [torch.tensor(2.0 ** e, device=DEV) for e in (ta, tb)]
    a, b = ((q[:, 0::2] | q[:, 1::2] << 4).to(DEV) for q in (qa, qb))
    one = k * (448.0 ** 2 if up else 2.0 ** -18)
    want = torch.outer((qa[:, 0] == 2).double(), (qb[:, 0] == 2).double()) * one * 2.0 ** ta * 2.0 ** tb
    step = 2.0 ** -149 if 0 < abs(one * 2.0 ** ta * 2.0 ** tb) < 2.0 ** -126 else 0.0  # below that fp32 is a grid of its own
    got = st.matmul_fp4(a, b.t(), sa, sb, a_tensor_scale=scale[0], b_tensor_scale=scale[1], out_dtype=torch.float32).cpu().double()
    want = want.float().double()
    assert ((got == want) | ((got - want).abs() <= step)).all()
    bias = torch.full((n,), 0.0, device=DEV)
    assert torch.equal(st.matmul_fp4(a, b.t(), sa, sb, bias, a_tensor_scale=scale[0], b_tensor_scale=scale[1],
                                     out_dtype=torch.float32).cpu().double(), got)


@pytest.mark.parametrize("m,n", [(128, 40), (1280, 1536)])
@pytest.mark.parametrize("high", [False, True], ids=["low", "high"])
def test_product_every_e8m0_scale(high, m, n):
    """All 255 powers of two, 2^-127 (a subnormal of fp32) and 2^127 among them, against 2^64 or 2^-64 in the other operand."""
    byte = torch.arange(m) % 128 + (127 if high else 0)
    other = 127 - 64 if high else 127 + 64
    ones = torch.full((max(m, n), 16), 0x22, dtype=torch.uint8, device=DEV)
    sa, sb = tiled(byte[:, None]).view(E8).to(DEV), tiled(torch.full((n, 1), other)).view(E8).to(DEV)
    want = (32 * torch.pow(torch.tensor(2.0, dtype=torch.float64), byte - 127.0 + other - 127.0)).float()[:, None].expand(m, n)
    assert torch.equal(st.matmul_fp4(ones[:m], ones[:n].t(), sa, sb, out_dtype=torch.float32).cpu(), want)
    assert torch.equal(st.matmul_fp4(ones[:n], ones[:m].t(), sb, sa, out_dtype=torch.float32).cpu(), want.t())


@pytest.mark.parametrize("layout", ["words", "columns"])
@pytest.mark.parametrize("t", [0.3, 1 / 3, 3e-42, 2.0 ** 120, 2.0 ** 122])
def test_dequantize_rounds_once(t, layout):
    """Each finite scale times each code times a tensor scale of any size, to fp32: the exact product of 30 bits, rounded once."""
    byte = torch.arange(127)[:, None]
    code = torch.arange(16).repeat(127, 1)
    packed = (code[:, 0::2] | code[:, 1::2] << 4).to(torch.uint8).to(DEV)
    packed = packed if layout == "words" else packed.t().contiguous().t()
    ts = torch.tensor(t, dtype=torch.float32)
    got = st.dequantize_fp4(packed, tiled(byte).view(E4).to(DEV), ts.to(DEV), out_dtype=torch.float32).cpu()
    want = values(code, byte, None, E4) * ts.double()
    assert torch.equal(got, want.float())
    assert torch.equal(torch.signbit(got), torch.signbit(want))


@pytest.mark.parametrize("amax", [0.0, float("inf"), float("-inf"), float("nan")])
def test_quantize_a_maximum_that_says_nothing(amax):
    """The tensor's scale is 1."""
    x = torch.randn(5, 100, generator=gen(1)) * 1000
    got = st.quantize_fp4(x.to(DEV), amax=torch.tensor(amax, device=DEV))
    want = st.quantize_fp4(x.to(DEV), amax=torch.tensor(2688.0, device=DEV))
    assert got.tensor_scale.item() == 1.0
    for a, b in zip(got, want):
        assert torch.equal(a.view(torch.uint8) if a.dim() else a, b.view(torch.uint8) if b.dim() else b)
