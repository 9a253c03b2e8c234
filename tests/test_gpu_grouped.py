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
          (1300, 320, 1032, [700, 700, 1299]), (2600, 72, 776, [2113, 2600]), (2700, 136, 4104, [1, 18, 18, 340, 2641])]
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


@pytest.mark.parametrize("order", ["n", "k"])
def test_tiles_of_every_size(order):
    """Groups on both sides of each step of a tile's columns, for one CTA and for pairs."""
    sizes = [1, 15, 16, 17, 31, 32, 33, 48, 49, 63, 64, 65, 95, 97, 127, 128, 129, 145, 160, 161, 191, 193, 224, 225, 240, 241, 255, 256,
             257, 273, 300, 511]
    ends = [sum(sizes[: i + 1]) for i in range(len(sizes))]
    a = ints(3, ends[-1], 264)
    for n in (72, 2056):
        b = ints(4, len(ends), 264, n)
        bd = b.to(BF16).to(DEV)
        bd = bd if order == "n" else bd.transpose(1, 2).contiguous().transpose(1, 2)
        got = st.matmul_grouped(a.to(BF16).to(DEV), bd, device_ends(ends), out_dtype=F32)
        assert torch.equal(got.cpu(), plain(a, b, ends).float())


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


@pytest.mark.parametrize("k,n", [(72, 136), (264, 520), (1032, 2056)])
def test_weights_last_steps(k, n):
    """Last steps of 1 to 64 rows, beside rows of other groups that hold NaN and infinities."""
    sizes = [s for i in range(1, 65) for s in (i if i % 2 else 64 + i, 1 + i % 5)]
    ends = [sum(sizes[: i + 1]) for i in range(len(sizes))]
    a, c = ints(5, ends[-1] + 9, k), ints(6, ends[-1] + 9, n)
    want = plain_weights(a, c, ends)
    for i, (x, y) in enumerate(parts(ends, a.shape[0])):
        if i % 2:
            a[x:y], c[x:y] = float("nan"), float("inf")
    a[ends[-1]:], c[ends[-1]:] = float("inf"), float("nan")
    got = st.matmul_grouped_weights(a.to(BF16).to(DEV), c.to(BF16).to(DEV), device_ends(ends), out_dtype=F32).cpu()
    assert torch.equal(got[::2], want[::2].float()) and got[1::2].isnan().all()


def test_weights_last_steps_on_pairs():
    sizes = [7, 900, 17, 880, 33, 850, 48, 840, 63, 830, 500, 517, 530, 547, 575, 600]
    ends = [sum(sizes[: i + 1]) for i in range(len(sizes))]
    a, c = ints(7, ends[-1], 520), ints(8, ends[-1], 1032)
    want = plain_weights(a, c, ends)
    for i, (x, y) in enumerate(parts(ends, a.shape[0])):
        if i % 2:
            a[x:y], c[x:y] = float("inf"), float("nan")
    got = st.matmul_grouped_weights(a.to(F16).to(DEV), c.to(F16).to(DEV), device_ends(ends), out_dtype=F32).cpu()
    assert torch.equal(got[::2], want[::2].float()) and got[1::2].isnan().all()


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


# ------------------------------------------------------------------ streams, graphs, long tensors
def test_one_graph_serves_any_ends():
    """The ends are read by the kernels: a captured step follows them when they change between replays."""
    rows, groups = 700, 9
    x, w = ints(1, rows, 128), ints(2, groups, 192, 128)
    xd, wd, e = x.to(BF16).to(DEV), w.to(BF16).to(DEV), device_ends([0] * groups)
    dy = ints(3, rows, 192).to(BF16).to(DEV)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y = st.matmul_grouped(xd, wd.transpose(1, 2), e, out_dtype=F32)
        dw = st.matmul_grouped_weights(dy, xd, e, out_dtype=F32)
    for seed in range(6):
        cut = sorted(torch.randint(0, rows + 1, (groups - 1,), generator=gen(seed)).tolist()) + [rows - 50 * (seed % 2)]
        ends = [min(c, cut[-1]) for c in cut]
        e.copy_(device_ends(ends))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), plain(x, w.transpose(1, 2), ends).float())
        assert torch.equal(dw.cpu(), plain_weights(dy.cpu().float(), x, ends).float())


def test_two_streams_at_once():
    ends = [100, 101, 330, 400]
    sets = [[torch.randn(*s, generator=gen(10 * i + j)).to(BF16).to(DEV) for j, s in enumerate([(400, 264), (4, 200, 264), (400, 200)])]
            for i in range(2)]
    e = device_ends(ends)

    def step(d):
        return [st.matmul_grouped(d[0], d[1].transpose(1, 2), e), st.matmul_grouped(d[2], d[1], e),
                st.matmul_grouped(d[0][:, 1:], d[1].transpose(1, 2)[:, 1:], e), st.matmul_grouped_weights(d[2], d[0][:, 1:], e)]

    want = [step(d) for d in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(sets[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


@pytest.mark.parametrize("order", ["n", "k"])
def test_many_weights(order):
    """A stack of more than 2^31 elements; the last groups against the plain form."""
    groups, k, n, rows = 34, 8192, 8192, 40
    b = torch.randint(-4, 5, (groups, k, n), device=DEV, dtype=torch.int8, generator=torch.Generator(DEV).manual_seed(1)).to(BF16)
    if order == "k":
        b = b.transpose(1, 2)
    ends = [0] * (groups - 2) + [17, rows]
    a = ints(2, rows, k)
    got = st.matmul_grouped(a.to(BF16).to(DEV), b, device_ends(ends), out_dtype=F32)
    for g, (i, j) in list(enumerate(parts(ends, rows)))[-2:]:
        assert torch.equal(got[i:j, -300:].cpu(), (a[i:j].double() @ b[g][:, -300:].cpu().double()).float())


def test_many_results():
    rows, n, k = 140000, 16384, 16
    a, b = ints(1, rows, k), ints(2, 3, k, n)
    ends = [5, 139000, 139900]
    got = st.matmul_grouped(a.to(F16).to(DEV), b.to(F16).to(DEV), device_ends(ends))
    assert torch.equal(got[138000:139000].cpu(), (a[138000:139000] @ b[1]).to(F16))
    assert torch.equal(got[139000:139900].cpu(), (a[139000:139900] @ b[2]).to(F16)) and (got[139900:] == 0).all()
    c = ints(3, 40, 8192)
    a = ints(4, 40, 8192)
    got = st.matmul_grouped_weights(a.to(F16).to(DEV), c.to(F16).to(DEV), device_ends([0] * 32 + [40, 40]))
    assert (got[33] == 0).all() and torch.equal(got[32, -100:].cpu(), (a.t()[-100:] @ c).to(F16))


# ------------------------------------------------------------------ together
def test_experts_layer_forward_and_backward():
    """A block of a network: norm, routed experts, a shared 4-bit expert, their sum back into the stream; and the
    experts' gradients.  Each stage is compared with float64 on what the stage before it gave."""
    tokens, hidden, inner, experts = 300, 256, 384, 6
    g = gen(7)
    r = torch.randn(tokens, hidden, generator=g)
    pre = torch.rand(hidden, generator=g) + 0.5
    w1, w2 = (torch.randn(experts, o, i, generator=g).to(BF16) / i ** 0.5 for o, i in ((inner, hidden), (hidden, inner)))
    shared = torch.randn(hidden, hidden, generator=g).to(BF16) / hidden ** 0.5
    choice = torch.randint(0, experts, (tokens,), generator=g)
    choice[choice == 2] = 3  # an expert without a token
    order = torch.argsort(choice, stable=True).to(DEV)
    ends_host = torch.cumsum(torch.bincount(choice, minlength=experts), 0).tolist()
    e = device_ends(ends_host)
    w1d, w2d = w1.to(DEV), w2.to(DEV)
    s4 = st.quantize_fp4(shared.to(DEV))

    f = st.residual_norm(None, r.to(BF16).to(DEV), pre_weight=pre.to(BF16).to(DEV), eps=1e-6)
    h = f.normed[order]
    u = st.matmul_grouped(h, w1d.transpose(1, 2), e, out_dtype=F32)
    v = torch.relu(u).square().to(BF16)
    y = st.matmul_grouped(v, w2d.transpose(1, 2), e, out_dtype=F32)
    h4 = st.quantize_fp4(f.normed)
    z = st.matmul_fp4(h4.codes, s4.codes.t(), h4.scale, s4.scale, a_tensor_scale=h4.tensor_scale, b_tensor_scale=s4.tensor_scale, out_dtype=F32)
    out = torch.empty_like(y)
    out[order] = y
    stream = st.residual_norm((out + z).to(BF16), f.residual).residual

    dy = torch.randn(tokens, hidden, generator=g).to(BF16).to(DEV)[order]
    dv = st.matmul_grouped(dy, w2d, e, out_dtype=F32)
    dw2 = st.matmul_grouped_weights(dy, v, e, out_dtype=F32)
    du = (dv * 2 * torch.relu(u)).to(BF16)
    dh = st.matmul_grouped(du, w1d, e, out_dtype=F32)
    dw1 = st.matmul_grouped_weights(du, h, e, out_dtype=F32)

    def near(got, want, size, terms):
        slack = (terms + 4) * 2.0 ** -23 * size
        assert ((got.cpu().double() - want).abs() <= slack + 2.0 ** -24 * (want.abs() + slack)).all()

    def rows(got, a, b):
        a, b = a.cpu(), b.cpu()
        near(got, plain(a, b, ends_host), plain(a.abs(), b.abs(), ends_host), a.shape[1])

    def sums(got, a, c):
        a, c = a.cpu(), c.cpu()
        near(got, plain_weights(a, c, ends_host), plain_weights(a.abs(), c.abs(), ends_host), tokens)

    rows(u, h, w1d.transpose(1, 2))
    rows(y, v, w2d.transpose(1, 2))
    rows(dv, dy, w2d)
    rows(dh, du, w1d)
    sums(dw2, dy, v)
    sums(dw1, du, h)
    assert (dw1[2] == 0).all() and (dw2[2] == 0).all()
    vh, vs = (st.dequantize_fp4(*q, out_dtype=F32).cpu().double() for q in (h4, s4))
    near(z, vh @ vs.t(), vh.abs() @ vs.abs().t(), hidden)
    want = f.residual.cpu().float() + (out + z).to(BF16).cpu().float()
    assert torch.equal(stream.cpu(), want.to(BF16))
    # a weight's gradient against differences of the layer's output, in float64
    step, at = 2.0 ** -6, (0, 3, 5)
    moved = []
    for sign in (1, -1):
        w = w2.double()
        w[at] += sign * step
        moved.append((plain(v.cpu(), w.transpose(1, 2), ends_host) * dy.cpu().double()).sum())
    slope, size = (moved[0] - moved[1]) / (2 * step), plain_weights(dy.cpu().abs(), v.cpu().abs(), ends_host)[at]
    assert abs(slope - dw2[at].item()) <= (tokens + 4) * 2.0 ** -23 * size + 2.0 ** -24 * abs(slope) + 1e-9 * abs(moved[0])


@pytest.mark.parametrize("rows,k,n,ends", [(130, 72, 136, [1, 1, 129, 130]), (1300, 320, 1032, [700, 700, 1299])])
@pytest.mark.parametrize("pad", [0, 5])
def test_weights_of_groups_in_turn(pad, rows, k, n, ends):
    """Results laid out [K, groups, N]: each where it belongs, what lies between them as it was."""
    a, c = ints(1, rows, k), ints(2, rows, n)
    room = torch.full((k, len(ends), n + pad), 7.0, device=DEV)
    out = room[:, :, :n].transpose(0, 1)
    st.matmul_grouped_weights(a.to(BF16).to(DEV), c.to(BF16).to(DEV), device_ends(ends), out=out)
    assert torch.equal(out.cpu(), plain_weights(a, c, ends).float())
    assert (room[:, :, n:] == 7).all()
