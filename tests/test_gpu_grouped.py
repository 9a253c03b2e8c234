"""Products by groups of rows on the GPU against plain computations.

Products of small integers are exact in fp32 (their sums stay below 2^24) and
compared for equality.  Others: each fp32 addition is off by at most 2^-23 of
the sum of the terms' magnitudes (a truncating adder), so a K-term sum by
(K + 4) 2^-23 sum |a b|, and the result's rounding adds half a step, eps / 2
relative."""
import pytest
import torch

import sptiles_b200 as st

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(seed, *shape):
    return torch.randint(-4, 5, shape, generator=gen(seed)).float()


def device_ends(ends):
    return torch.tensor(ends, dtype=torch.int32, device=DEV)


def parts(ends, rows):
    """Rows of each group, bounds in disorder taken as documented."""
    first, out = 0, []
    for end in ends:
        end = min(max(end, first), rows)
        out.append((first, end))
        first = end
    return out


def plain(a, b, ends):
    c = torch.zeros(a.shape[0], b.shape[2], dtype=torch.float64)
    for g, (i, j) in enumerate(parts(ends, a.shape[0])):
        c[i:j] = a[i:j].double() @ b[g].double()
    return c


def plain_weights(a, c, ends):
    return torch.stack([a[i:j].double().t() @ c[i:j].double() for i, j in parts(ends, a.shape[0])])


# rows, k, n, ends
CASES = [
    (1, 8, 8, [1]), (1, 1, 1, [1]), (5, 64, 128, [0, 5]), (64, 64, 64, [64]), (130, 72, 136, [1, 1, 129, 130]),
    (300, 128, 256, [0, 0, 300]), (300, 200, 120, [17, 150, 299]), (257, 65, 33, [100, 257]), (1000, 264, 520, [3, 250, 250, 700, 960]),
    (129, 1001, 515, [64, 129]), (513, 40, 1000, [128, 256, 384, 512, 513]), (40, 512, 384, list(range(1, 41))),
    (70, 96, 80, [100]), (70, 96, 80, [30, 10, 200, 5]), (70, 96, 80, [-5, 40]), (2000, 136, 264, [1000, 1000, 1999]),
]
# a long contraction and few tiles: clusters split it; and groups of several tiles of CTA pairs
CASES += [(40, 4096, 200, [7, 40]), (3, 8192, 64, [3]), (200, 2049, 130, [150, 200]), (3000, 64, 72, [3000]), (5000, 40, 136, [4000, 4001]),
          (1300, 320, 1032, [700, 700, 1299]), (2600, 72, 776, [2113, 2600])]
IDS = [f"{r}x{k}x{n}-{len(e)}" for r, k, n, e in CASES]


@pytest.mark.parametrize("layout", ["n", "k", "k padded", "n off"])
@pytest.mark.parametrize("rows,k,n,ends", CASES, ids=IDS)
def test_rows_exact(rows, k, n, ends, layout):
    a, b = ints(1, rows, k), ints(2, len(ends), k, n)
    want = plain(a, b, ends)
    for dtype in (F16, BF16):
        bd = b.to(dtype).to(DEV)
        if layout == "k":
            bd = bd.transpose(1, 2).contiguous().transpose(1, 2)
        elif layout == "k padded":
            room = torch.full((len(ends), n + 3, (k + 7) // 8 * 8 + 8), 9.0, dtype=dtype, device=DEV)
            room[:, :n, :k] = bd.transpose(1, 2)
            bd = room[:, :n, :k].transpose(1, 2)
        elif layout == "n off":
            room = torch.full((len(ends), k, n + 3), 9.0, dtype=dtype, device=DEV)
            room[:, :, 1 : n + 1] = bd
            bd = room[:, :, 1 : n + 1]
        got = st.matmul_grouped(a.to(dtype).to(DEV), bd, device_ends(ends), out_dtype=F32)
        assert torch.equal(got.cpu(), want.float())
    got = st.matmul_grouped(a.to(dtype).to(DEV), bd, device_ends(ends))
    assert got.dtype == dtype and torch.equal(got.cpu(), want.float().to(dtype))


@pytest.mark.parametrize("rows,k,n,ends", CASES, ids=IDS)
def test_weights_exact(rows, k, n, ends):
    a, c = ints(1, rows, k), ints(2, rows, n)
    want = plain_weights(a, c, ends)
    for dtype in (F16, BF16):
        got = st.matmul_grouped_weights(a.to(dtype).to(DEV), c.to(dtype).to(DEV), device_ends(ends), out_dtype=F32)
        assert torch.equal(got.cpu(), want.float())
    got = st.matmul_grouped_weights(a.to(dtype).to(DEV), c.to(dtype).to(DEV), device_ends(ends))
    assert got.dtype == dtype and torch.equal(got.cpu(), want.float().to(dtype))
    turned = [t.to(dtype).to(DEV).t().contiguous().t() for t in (a, c)]  # stored along the rows: copied first
    assert torch.equal(st.matmul_grouped_weights(*turned, device_ends(ends), out_dtype=F32).cpu(), want.float())


def test_other_groups_do_not_matter():
    """NaN and infinities in one group's rows, in its matrix and behind the last group stay there."""
    ends = [70, 133, 200, 260]
    a, b, c = ints(1, 300, 96), ints(2, 4, 96, 136), ints(3, 300, 136)
    want, want_w = plain(a, b, ends).float(), plain_weights(a, c, ends).float()
    bad_a, bad_b, bad_c = a.clone(), b.clone(), c.clone()
    for t in (bad_a, bad_c):
        t[70:133:2], t[71:133:2], t[260:] = float("nan"), float("inf"), float("nan")
    bad_b[1] = float("nan")
    dev = [t.to(BF16).to(DEV) for t in (bad_a, bad_b, bad_c)]
    got = st.matmul_grouped(dev[0], dev[1], device_ends(ends), out_dtype=F32).cpu()
    assert torch.isnan(got[70:133]).all() and (got[260:] == 0).all()
    got[70:133] = want[70:133]
    assert torch.equal(got, want)
    got = st.matmul_grouped_weights(dev[0], dev[2], device_ends(ends), out_dtype=F32).cpu()
    assert torch.isnan(got[1]).all()
    got[1] = want_w[1]
    assert torch.equal(got, want_w)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("n", [64, 65, 200])
def test_given_outputs(n, dtype):
    """Nothing around the output is written, nor its rows behind the last group."""
    ends = [33, 100]
    a, b, c = ints(1, 140, 72), ints(2, 2, 72, n), ints(3, 140, n)
    dev = [t.to(F16).to(DEV) for t in (a, b, c)]
    for left in (0, 3):
        room = torch.full((142, n + 8), 7.0, dtype=dtype, device=DEV)
        out = room[1:141, left : n + left]
        assert st.matmul_grouped(dev[0], dev[1], device_ends(ends), out=out) is out
        assert torch.equal(out[:100].cpu(), plain(a, b, ends)[:100].to(dtype))
        out[:100] = 7.0
        assert (room == 7).all()
        room = torch.full((2, 74, n + 8), 7.0, dtype=dtype, device=DEV)
        out = room[:, 1:73, left : n + left]
        assert st.matmul_grouped_weights(dev[0], dev[2], device_ends(ends), out=out) is out
        assert torch.equal(out.cpu(), plain_weights(a, c, ends).to(dtype))
        out.fill_(7.0)
        assert (room == 7).all()


def test_empty():
    for rows, k, n, ends in [(0, 8, 8, [0, 0]), (5, 0, 8, [5]), (5, 8, 0, [5]), (5, 8, 8, []), (0, 8, 8, [])]:
        a, c = torch.ones(rows, k, dtype=F16, device=DEV), torch.ones(rows, n, dtype=F16, device=DEV)
        b = torch.ones(len(ends), k, n, dtype=F16, device=DEV)
        got = st.matmul_grouped(a, b, device_ends(ends))
        assert got.shape == (rows, n) and (got == 0).all() if k == 0 or not ends else got.shape == (rows, n)
        got = st.matmul_grouped_weights(a, c, device_ends(ends))
        assert got.shape == (len(ends), k, n) and (rows > 0 or (got == 0).all())
    out = torch.full((5, 8), 7.0, device=DEV)
    st.matmul_grouped(torch.ones(5, 0, dtype=F16, device=DEV), torch.ones(2, 0, 8, dtype=F16, device=DEV), device_ends([1, 3]), out=out)
    assert (out[:3] == 0).all() and (out[3:] == 7).all()


def test_views():
    """Rows of a wider matrix, rows stored across, one matrix for every group, every second group."""
    ends = [50, 120, 150]
    a, b = ints(1, 150, 80), ints(2, 3, 80, 48)
    ad, bd, e = a.to(BF16).to(DEV), b.to(BF16).to(DEV), device_ends(ends)
    want = plain(a, b, ends).float()
    wide = torch.full((150, 96), 9.0, dtype=BF16, device=DEV)
    wide[:, 8:88] = ad
    assert torch.equal(st.matmul_grouped(wide[:, 8:88], bd, e, out_dtype=F32).cpu(), want)
    assert torch.equal(st.matmul_grouped(ad.t().contiguous().t(), bd, e, out_dtype=F32).cpu(), want)
    one = bd[:1].expand(3, -1, -1)
    assert torch.equal(st.matmul_grouped(ad, one, e, out_dtype=F32).cpu(), (a @ b[0]).float())
    two = torch.full((6, 80, 48), 9.0, dtype=BF16, device=DEV)
    two[::2] = bd
    assert torch.equal(st.matmul_grouped(ad, two[::2], e, out_dtype=F32).cpu(), want)
    assert torch.equal(st.matmul_grouped(ad[:1].expand(150, -1), bd, e, out_dtype=F32).cpu(),
                       plain(a[:1].expand(150, -1), b, ends).float())


@pytest.mark.parametrize("groups", [33, 1000, 1024])
def test_many_groups(groups):
    sizes = torch.randint(0, 6, (groups,), generator=gen(groups))
    ends = torch.cumsum(sizes, 0).tolist()
    rows = ends[-1]
    a, b, c = ints(1, rows, 64), ints(2, groups, 64, 72), ints(3, rows, 72)
    dev = [t.to(F16).to(DEV) for t in (a, b, c)]
    assert torch.equal(st.matmul_grouped(dev[0], dev[1], device_ends(ends), out_dtype=F32).cpu(), plain(a, b, ends).float())
    assert torch.equal(st.matmul_grouped_weights(dev[0], dev[2], device_ends(ends), out_dtype=F32).cpu(),
                       plain_weights(a, c, ends).float())


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_random_values(dtype):
    ends = [100, 400, 400, 1100]
    a, b, c = (torch.randn(*s, generator=gen(i)).to(dtype) for i, s in enumerate([(1200, 520), (4, 520, 392), (1200, 392)]))
    got = st.matmul_grouped(a.to(DEV), b.to(DEV), device_ends(ends)).cpu().double()
    want, size = plain(a, b, ends), plain(a.abs(), b.abs(), ends)
    slack = 524 * 2.0 ** -23 * size
    assert ((got - want).abs() <= slack + torch.finfo(dtype).eps / 2 * (want.abs() + slack)).all()
    got = st.matmul_grouped_weights(a.to(DEV), c.to(DEV), device_ends(ends), out_dtype=F32).cpu().double()
    want, size = plain_weights(a, c, ends), plain_weights(a.abs(), c.abs(), ends)
    slack = 704 * 2.0 ** -23 * size
    assert ((got - want).abs() <= slack + 2.0 ** -24 * (want.abs() + slack)).all()


def test_gradients_against_autograd():
    """The calls as a layer's forward and backward pass, against float64 autograd of the plain layer."""
    ends = [40, 40, 170, 200]
    x, w, dy = torch.randn(200, 96, generator=gen(1)), torch.randn(4, 64, 96, generator=gen(2)), torch.randn(200, 64, generator=gen(3))
    x, w, dy = x.to(BF16), w.to(BF16), dy.to(BF16)
    lx, lw = x.double().requires_grad_(), w.double().requires_grad_()
    y = torch.cat([lx[i:j] @ lw[g].t() for g, (i, j) in enumerate(parts(ends, 200))])
    gx, gw = torch.autograd.grad(y, [lx, lw], dy.double())
    xd, wd, dyd, e = x.to(DEV), w.to(DEV), dy.to(DEV), device_ends(ends)

    def near(got, want, terms, size):
        slack = (terms + 4) * 2.0 ** -23 * size
        assert ((got.cpu().double() - want).abs() <= slack + 2.0 ** -24 * (want.abs() + slack)).all()

    near(st.matmul_grouped(xd, wd.transpose(1, 2), e, out_dtype=F32), y.detach(), 96, plain(x.abs(), w.abs().transpose(1, 2), ends))
    near(st.matmul_grouped(dyd, wd, e, out_dtype=F32), gx, 64, plain(dy.abs(), w.abs(), ends))
    near(st.matmul_grouped_weights(dyd, xd, e, out_dtype=F32), gw, 130, plain_weights(dy.abs(), x.abs(), ends))
