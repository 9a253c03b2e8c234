"""residual_norm and its backward on the GPU against float64.

Bounds.  A row's sum of n squares is added in a tree of depth below 64 (8
elements a lane at most four times, 5 shuffles, 5 more over warps), so it is
within 64 * 2^-24 relative, its root half of that; with the handful of fp32
products around it a value u, h, t or dx before its rounding is within
2^-16 of the sum of the magnitudes it is made of.  A rounding to type T adds
eps(T) / 2 relative.  A sum over rows adds at most rows + 64 fp32 additions,
each 2^-24 of the sum of magnitudes."""
import pytest
import torch

import sptiles_b200 as st

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
REL = 2.0 ** -16
EPS = 1e-5


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half(t):
    return torch.finfo(t).eps / 2


def close(got, want, mass, dtype, rel=REL):
    assert got is not None and got.dtype == dtype and got.shape == want.shape, (got.dtype, got.shape, want.shape)
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    off = (got.double().cpu() - want).abs() - rel * mass - half(dtype) * (want.abs() + rel * mass) - tiny
    assert not torch.isnan(off).any()
    assert off.numel() == 0 or off.max().item() <= 0, off.max().item()


def rms(v, w):
    return v / torch.sqrt(v.square().mean(1, keepdim=True) + EPS) * w


def inputs(rows, cols, tx, tr, gate, post, pre, seed=0, with_x=True):
    g = gen(seed)
    r = {"x": (torch.randn(rows, cols, generator=g) * 2).to(tx) if with_x else None,
         "r": torch.randn(rows, cols, generator=g).to(tr),
         "post": (1 + 0.3 * torch.randn(cols, generator=g)).to(tx) if post else None,
         "pre": (1 + 0.3 * torch.randn(cols, generator=g)).to(F32 if seed % 2 else tx) if pre else None}
    shape = {"none": None, "channel": (cols,), "row": (1, cols), "token": (rows, 1), "full": (rows, cols)}[gate]
    r["gate"] = torch.randn(*shape, generator=g).to(tx) if shape else None
    return r


def dev(d):
    return {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def dbl(d):
    return {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in d.items()}


def forward64(d, alpha, offset):
    r, mass = d["r"], d["r"].abs()
    if d["x"] is not None:
        u = d["x"] if d["post"] is None else rms(d["x"], d["post"] + offset)
        u = u * alpha * (1 if d["gate"] is None else d["gate"])
        r, mass = r + u, mass + u.abs()
    h = None if d["pre"] is None else rms(r, d["pre"] + offset)
    return r, mass, h


def check_forward(d, alpha=0.7, offset=0.0, **kw):
    g = dev(d)
    got = st.residual_norm(g["x"], g["r"], g["post"], g["gate"], g["pre"], alpha=alpha, eps=EPS, weight_offset=offset, **kw)
    r, mass, h = forward64(dbl(d), alpha, offset)
    if d["x"] is not None:
        close(got.residual, r, mass, d["r"].dtype)
    else:
        assert got.residual is g["r"]
    if h is None:
        assert got.normed is None
        return got
    w = (d["pre"].double() + offset).abs()
    hmass = mass / torch.sqrt(r.square().mean(1, keepdim=True) + EPS) * w + h.abs()
    tx = d["x"].dtype if d["x"] is not None else d["r"].dtype
    if got.scale is None:
        close(got.normed, h, hmass, tx)
        return got
    # 8-bit blocks: the scale within the bound of the block's largest value; the codes within half a step of the
    # value, or of the smallest one (2^-9 for e4m3, 2^-16 for e5m2)
    rows, cols = h.shape
    e5 = got.normed.dtype == torch.float8_e5m2
    pad = -cols % 128
    blocks = torch.nn.functional.pad(h, (0, pad)).view(rows, -1, 128)
    mblocks = torch.nn.functional.pad(hmass, (0, pad)).view(rows, -1, 128)
    limit = 57344.0 if e5 else 448.0
    assert got.scale.shape == (rows, blocks.shape[1]) and got.scale.dtype == F32
    want = blocks.abs().amax(2) / limit
    s = got.scale.cpu().double()
    assert ((s - want).abs() <= REL * mblocks.amax(2) / limit + 2.0 ** -23 * want + 2.0 ** -125).all()
    back = got.normed.cpu().double() * s.repeat_interleave(128, 1)[:, :cols]
    step = 2.0 ** -3 if e5 else 2.0 ** -4
    least = (2.0 ** -17 if e5 else 2.0 ** -10) * s.repeat_interleave(128, 1)[:, :cols]
    assert ((back - h).abs() <= step * h.abs() + least + 4 * REL * hmass).all()
    return got


SHAPES = [(1, 1), (1, 4096), (2, 5), (3, 32), (5, 255), (7, 256), (6, 300), (9, 512), (4, 513), (3, 2049), (130, 1024),
          (2, 8192), (2, 8200), (1, 16384), (3, 12001)]


@pytest.mark.parametrize("quantize", [False, True], ids=["plain", "fp8"])
@pytest.mark.parametrize("tx,tr", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)],
                         ids=["f32", "f16", "bf16", "f16_f32", "bf16_f32"])
@pytest.mark.parametrize("rows,cols", SHAPES, ids=lambda v: str(v))
def test_forward(rows, cols, tx, tr, quantize):
    check_forward(inputs(rows, cols, tx, tr, "channel", True, True, seed=rows + cols), quantize=quantize)


@pytest.mark.parametrize("gate", ["none", "channel", "row", "token", "full"])
@pytest.mark.parametrize("post", [True, False], ids=["post", "nopost"])
@pytest.mark.parametrize("pre", [True, False], ids=["pre", "nopre"])
@pytest.mark.parametrize("rows,cols", [(5, 96), (4, 1100)], ids=lambda v: str(v))
def test_forward_parts(rows, cols, pre, post, gate):
    check_forward(inputs(rows, cols, BF16, F32, gate, post, pre, seed=2), offset=1.0)


def test_forward_first_norm():
    for tr, out in [(F32, None), (F32, BF16), (BF16, None)]:
        d = inputs(6, 700, tr if out is None else out, tr, "none", False, True, with_x=False)
        d["pre"] = d["pre"].to(F32)
        g = dev(d)
        got = st.residual_norm(None, g["r"], pre_weight=g["pre"], eps=EPS, out_dtype=out)
        want = rms(d["r"].double(), d["pre"].double())
        close(got.normed, want, 2 * want.abs(), out or tr)
        assert got.residual is g["r"]
    check_forward(inputs(6, 700, BF16, BF16, "none", False, True, with_x=False), quantize=torch.float8_e5m2)


def test_forward_in_place_strided_and_zero_rows():
    d = inputs(20, 640, BF16, BF16, "token", True, True)
    d["x"][3], d["r"][3] = 0, 0  # a row of zeros: normed to zeros
    want = check_forward(d)
    room = torch.full((22, 700), 9.0, dtype=BF16, device=DEV)
    for shift in (8, 3):  # 16-byte rows, and not
        v = room[1:21, shift:shift + 640]
        v.copy_(d["r"])
        g = dev(d)
        got = st.residual_norm(g["x"], v, g["post"], g["gate"], g["pre"], alpha=0.7, eps=EPS, out=v)
        assert got.residual.data_ptr() == v.data_ptr()
        close(v, want.residual.cpu().double(), 2 * want.residual.cpu().double().abs(), BF16, rel=2.0 ** -8)
        keep = room.clone()
        keep[1:21, shift:shift + 640] = 9.0
        assert (keep == 9.0).all()
        room.fill_(9.0)
    empty = st.residual_norm(torch.empty(0, 64, device=DEV), torch.empty(0, 64, device=DEV), pre_weight=torch.ones(64, device=DEV))
    assert empty.residual.shape == (0, 64) and empty.normed.shape == (0, 64)


def test_forward_nan_stays_in_its_row():
    d = inputs(5, 300, F32, F32, "none", True, True)
    d["x"][2, 7] = float("nan")
    g = dev(d)
    got = st.residual_norm(g["x"], g["r"], g["post"], None, g["pre"], eps=EPS, quantize=True)
    assert torch.isnan(got.residual[2]).all() and torch.isnan(got.scale[2]).all()
    for r in (0, 1, 3, 4):
        assert torch.isfinite(got.residual[r]).all() and torch.isfinite(got.scale[r]).all()


# ------------------------------------------------------------------ backward
def backward64(d, dr, dh, alpha, offset):
    """Gradients and, for each, the sum of the magnitudes it is made of."""
    out, mass = {}, {}
    total = dr if dr is not None else torch.zeros_like(dh)
    tmass = total.abs()
    if d["pre"] is not None:
        r, w = d["r"], d["pre"] + offset
        inv = 1 / torch.sqrt(r.square().mean(1, keepdim=True) + EPS)
        hat, t = r * inv, dh * w
        out["pre"], mass["pre"] = (dh * hat).sum(0), (dh * hat).abs().sum(0)
        total = total + inv * (t - hat * (t * hat).mean(1, keepdim=True))
        tmass = tmass + inv * (t.abs() + hat.abs() * (t * hat).abs().mean(1, keepdim=True))
    out["residual"], mass["residual"] = total, tmass
    if d["x"] is None:
        return out, mass
    gate = 1 if d["gate"] is None else d["gate"]
    agate = 1 if d["gate"] is None else d["gate"].abs()
    x, w = d["x"], 1.0 if d["post"] is None else d["post"] + offset
    aw = 1.0 if d["post"] is None else w.abs()
    inv = 1.0 if d["post"] is None else 1 / torch.sqrt(x.square().mean(1, keepdim=True) + EPS)
    hat = x * inv
    du, dumass = alpha * gate * total, alpha * agate * tmass
    if d["post"] is None:
        out["x"], mass["x"] = du, dumass
    else:
        t, tm = du * w, dumass * aw
        out["x"] = inv * (t - hat * (t * hat).mean(1, keepdim=True))
        mass["x"] = inv * (tm + hat.abs() * (tm * hat.abs()).mean(1, keepdim=True))
        out["post"], mass["post"] = (du * hat).sum(0), (dumass * hat.abs()).sum(0)
    if d["gate"] is not None:
        g, gm = alpha * total * hat * w, alpha * tmass * hat.abs() * aw
        if d["gate"].dim() == 1 or (d["gate"].shape[0] == 1 and g.shape[0] != 1):
            g, gm = (v.sum(0).view(d["gate"].shape) for v in (g, gm))
        elif d["gate"].shape[1] == 1 and g.shape[1] != 1:
            g, gm = (v.sum(1, keepdim=True) for v in (g, gm))
        out["gate"], mass["gate"] = g, gm
    return out, mass


def check_backward(d, rows, cols, tx, tr, alpha=0.7, offset=0.0, d_residual=True):
    g = gen(99)
    dr = torch.randn(rows, cols, generator=g).to(tr) if d_residual else None
    dh = torch.randn(rows, cols, generator=g).to(tx) if d["pre"] is not None else None
    c = dev(d)
    args = [None if t is None else t.to(DEV) for t in (dr, dh)]
    got = st.residual_norm_backward(*args, c["x"], c["r"] if d["pre"] is not None else None, c["post"], c["gate"], c["pre"],
                                    alpha=alpha, eps=EPS, weight_offset=offset)
    want, mass = backward64(dbl(d), *[None if t is None else t.double() for t in (dr, dh)], alpha, offset)
    over_rows = REL + (rows + 64) * 2.0 ** -24
    close(got.residual, want["residual"], mass["residual"], tr)
    for name, dtype, value in [("x", tx, got.x), ("post", F32, got.post_weight), ("pre", F32, got.pre_weight),
                               ("gate", None, got.gate)]:
        if name not in want:
            assert value is None
            continue
        if name == "gate":
            full = d["gate"].dim() == 2 and d["gate"].shape == (rows, cols)
            dtype = tx if full else F32
        close(value, want[name], mass[name], dtype, rel=REL if name == "x" else over_rows)
    return got


@pytest.mark.parametrize("tx,tr", [(F32, F32), (F16, F16), (BF16, BF16), (F16, F32), (BF16, F32)],
                         ids=["f32", "f16", "bf16", "f16_f32", "bf16_f32"])
@pytest.mark.parametrize("rows,cols", SHAPES + [(700, 512), (1300, 96), (333, 2048)], ids=lambda v: str(v))
def test_backward(rows, cols, tx, tr):
    check_backward(inputs(rows, cols, tx, tr, "channel", True, True, seed=rows), rows, cols, tx, tr)


@pytest.mark.parametrize("gate", ["none", "channel", "row", "token", "full"])
@pytest.mark.parametrize("post", [True, False], ids=["post", "nopost"])
@pytest.mark.parametrize("pre", [True, False], ids=["pre", "nopre"])
@pytest.mark.parametrize("rows,cols", [(5, 96), (40, 1100), (1, 64)], ids=lambda v: str(v))
def test_backward_parts(rows, cols, pre, post, gate):
    check_backward(inputs(rows, cols, BF16, F32, gate, post, pre, seed=2), rows, cols, BF16, F32, offset=1.0)


def test_backward_first_norm_and_missing_gradients():
    check_backward(inputs(33, 600, F32, F32, "none", False, True, with_x=False), 33, 600, F32, F32, d_residual=False)
    check_backward(inputs(33, 600, BF16, BF16, "none", True, True), 33, 600, BF16, BF16, d_residual=False)
    e = torch.empty(0, 64, device=DEV)
    w = torch.ones(64, device=DEV)
    got = st.residual_norm_backward(e, e, e, e, w, w, w)
    for s in (got.post_weight, got.gate, got.pre_weight):
        assert s.shape == (64,) and (s == 0).all()


def test_backward_against_differences():
    """The gradients times a direction against the forward call's own differences, in float32 with float64 quotients."""
    rows, cols = 6, 80
    d = dbl(inputs(rows, cols, F32, F32, "channel", True, True, seed=4))
    g = gen(5)
    dr, dh = torch.randn(rows, cols, generator=g).double(), torch.randn(rows, cols, generator=g).double()

    def loss(v):
        r, _, h = forward64(v, 0.7, 0.0)
        return (r * dr).sum() + (h * dh).sum()

    r_out = forward64(d, 0.7, 0.0)[0]
    f = {k: v.float().to(DEV) for k, v in d.items()}
    got = st.residual_norm_backward(dr.float().to(DEV), dh.float().to(DEV), f["x"], r_out.float().to(DEV), f["post"], f["gate"],
                                    f["pre"], alpha=0.7, eps=EPS)
    for name, grad in [("x", got.x), ("r", got.residual), ("post", got.post_weight), ("gate", got.gate), ("pre", got.pre_weight)]:
        way = torch.randn(d[name].shape, generator=g).double()
        step = 1e-5  # central differences in float64: off by about step^2 and 1e-16 / step, both below 1e-9
        up, down = ({**d, name: d[name] + s * step * way} for s in (1, -1))
        slope = (loss(up) - loss(down)) / (2 * step)
        mine = grad.double().cpu()
        assert abs((mine * way).sum() - slope) <= 2.0 ** -14 * (mine.abs() * way.abs()).sum() + 1e-6, name


def test_backward_same_bits_and_graph():
    rows, cols = 500, 1024
    d = dev(inputs(rows, cols, BF16, BF16, "channel", True, True))
    dr = torch.randn(rows, cols, generator=gen(1)).to(BF16).to(DEV)
    dh = torch.randn(rows, cols, generator=gen(2)).to(BF16).to(DEV)

    def step():
        f = st.residual_norm(d["x"], d["r"], d["post"], d["gate"], d["pre"])
        return [f.normed, *st.residual_norm_backward(dr, dh, d["x"], f.residual, d["post"], d["gate"], d["pre"])]

    first = step()
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            again = step()
    torch.cuda.synchronize()
    for t in again:
        t.zero_()
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, again):
        assert torch.equal(a, b)


def test_norm_into_product():
    """The 8-bit copy between two blocks goes straight into matmul_fp8."""
    rows, cols, n = 70, 512, 200
    d = dev(inputs(rows, cols, BF16, F32, "none", True, True))
    W = torch.randn(n, cols, generator=gen(8)).to(BF16).to(DEV)
    Wq, Ws = st.quantize_fp8(W, block=(128, 128))
    f = st.residual_norm(d["x"], d["r"], d["post"], None, d["pre"], eps=EPS, quantize=True)
    y = st.matmul_fp8(f.normed, Wq.t(), f.scale, Ws.t(), out_dtype=F32)
    a = f.normed.double() * f.scale.double().repeat_interleave(128, 1)[:, :cols]
    b = Wq.double() * Ws.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :cols]
    want, mass = a @ b.t(), a.abs() @ b.abs().t()
    assert ((y.double() - want).abs() <= (128 + 4 + 5) * 2.0 ** -23 * mass).all()
    z = st.residual_norm(y[:, :n].to(BF16), torch.zeros(rows, n, device=DEV), torch.ones(n, device=DEV))
    assert torch.isfinite(z.residual).all() and z.normed is None


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("tx,tr", [(F32, F32), (F16, F16), (BF16, F32)], ids=["f32", "f16", "bf16_f32"])
@pytest.mark.parametrize("rows,cols", [(700, 1024), (1601, 520), (500, 5000), (333, 8192)], ids=lambda v: str(v))
def test_forward_many_rows(rows, cols, tx, tr, gate):
    """Enough rows for every persistent CTA to take several, on 16-byte boundaries."""
    d = inputs(rows, cols, tx, tr, gate, True, True, seed=3)
    check_forward(d, quantize=True)
    check_forward(d, offset=1.0)


@pytest.mark.parametrize("post,pre", [(True, False), (False, True)])
def test_forward_many_rows_parts(post, pre):
    check_forward(inputs(900, 768, BF16, BF16, "channel", post, pre, seed=4))
    d = inputs(900, 768, BF16, BF16, "channel", post, pre, seed=4)
    g = dev(d)
    want = st.residual_norm(g["x"], g["r"], g["post"], g["gate"], g["pre"])
    got = st.residual_norm(g["x"], g["r"], g["post"], g["gate"], g["pre"], out=g["r"])  # in place
    assert torch.equal(got.residual, want.residual) and got.residual is g["r"]


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("tx,tr", [(F32, F32), (F16, F16), (BF16, F32)], ids=["f32", "f16", "bf16_f32"])
@pytest.mark.parametrize("rows,cols", [(700, 1024), (1601, 520), (500, 5000), (333, 8192), (2500, 264)], ids=lambda v: str(v))
def test_backward_many_rows(rows, cols, tx, tr, gate):
    check_backward(inputs(rows, cols, tx, tr, gate, True, True, seed=3), rows, cols, tx, tr, offset=0.5)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post", [True, False], ids=["post", "nopost"])
@pytest.mark.parametrize("pre", [True, False], ids=["pre", "nopre"])
def test_backward_many_rows_parts(pre, post, gate):
    check_backward(inputs(900, 768, BF16, BF16, gate, post, pre, seed=4), 900, 768, BF16, BF16)
    if pre:
        check_backward(inputs(900, 768, BF16, F32, gate, post, pre, seed=4), 900, 768, BF16, F32, d_residual=False)


def test_backward_zero_token_gate():
    """A token whose gate is 0 still gets the gate's gradient; its x gets none."""
    for rows in (10, 700):
        d = inputs(rows, 640, F32, F32, "token", True, True)
        d["gate"][::2] = 0
        got = check_backward(d, rows, 640, F32, F32)
        assert (got.x[::2] == 0).all() and (got.gate[::2] != 0).all()


def test_many_elements():
    """Offsets past 32 bits: the last rows of 2^31 and more elements."""
    g = torch.Generator(device=DEV).manual_seed(1)
    for rows, cols in [(140000, 16384), (270000, 8192)]:
        x, r, dr, dh = (torch.randn(rows, cols, generator=g, device=DEV, dtype=BF16) for _ in range(4))
        w = torch.rand(cols, generator=g, device=DEV).to(BF16)
        f = st.residual_norm(x, r, w, None, w, eps=EPS, quantize=True)
        b = st.residual_norm_backward(dr, dh, x, r, w, None, w, eps=EPS)
        last = {"x": x[-5:].cpu(), "r": r[-5:].cpu(), "post": w.cpu(), "pre": w.cpu(), "gate": None}
        want, mass, h = forward64(dbl(last), 1.0, 0.0)
        close(f.residual[-5:], want, mass, BF16)
        same = st.residual_norm(x[-5:].clone(), r[-5:].clone(), w, None, w, eps=EPS, quantize=True)
        back = [(v.normed[-5:].double() * v.scale[-5:].double().repeat_interleave(128, 1)).cpu() for v in (f, same)]
        for v in back:  # half a step of e4m3, or of the block's smallest code, and the fp32 sums' REL
            least = 2.0 ** -10 * f.scale[-5:].double().cpu().repeat_interleave(128, 1)
            assert ((v - h).abs() <= 2.0 ** -4 * h.abs() + least + 8 * REL * (mass + h.abs())).all()
        want, mass = backward64(dbl(last), dr[-5:].double().cpu(), dh[-5:].double().cpu(), 1.0, 0.0)
        close(b.residual[-5:], want["residual"], mass["residual"], BF16)
        close(b.x[-5:], want["x"], mass["x"], BF16)
        del x, r, dr, dh, f, b


def test_two_streams_at_once():
    """Two training steps under way on two streams, each with tensors of its own, as one after the other."""
    rows, cols = 900, 2048
    sets = [dev(inputs(rows, cols, BF16, F32, "channel", True, True, seed=s)) for s in (0, 2)]
    grads = [torch.randn(rows, cols, generator=gen(3 + s)).to(DEV) for s in (0, 1)]

    def step(d, dr):
        f = st.residual_norm(d["x"], d["r"], d["post"], d["gate"], d["pre"])
        b = st.residual_norm_backward(dr, dr.to(BF16), d["x"], f.residual, d["post"], d["gate"], d["pre"])
        return [f.residual, f.normed, *b]

    want = [step(d, g) for d, g in zip(sets, grads)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream(), torch.cuda.Stream()], [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(step(sets[i], grads[i]))
    torch.cuda.synchronize()
    for i in (0, 1):
        for run in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(run, want[i]))


def test_widest_rows():
    """16384 columns in every type, where a row fills one stage of the ring."""
    for tx, tr in [(F32, F32), (BF16, F32), (F16, F16)]:
        check_forward(inputs(400, 16384, tx, tr, "channel", True, True, seed=1), quantize=True)
        check_backward(inputs(320, 16384, tx, tr, "token", True, True, seed=1), 320, 16384, tx, tr)


@pytest.mark.parametrize("rows", [3, 700])
def test_outputs_left_out_in_c(rows):
    """The C calls without an updated stream, without dr and without the sums (then with no workspace)."""
    from sptiles_b200.fp8 import _desc, _fn, _vp, _cp, _u64
    from sptiles_b200.norm import _OPTIONS
    from sptiles_b200.api import _exec_desc

    cols = 1024
    d = dev(inputs(rows, cols, BF16, F32, "token", True, True))
    dr, dh = torch.randn(rows, cols, generator=gen(1)).to(DEV), torch.randn(rows, cols, generator=gen(2)).to(BF16).to(DEV)
    want = st.residual_norm(d["x"], d["r"], d["post"], d["gate"], d["pre"], eps=EPS)
    back = st.residual_norm_backward(dr, dh, d["x"], want.residual, d["post"], d["gate"], d["pre"], eps=EPS)
    ctx, opt, ex = st.runtime.context(0), _OPTIONS.pack(1.0, EPS, 0.0), _exec_desc(0)
    normed = torch.empty(rows, cols, dtype=BF16, device=DEV)
    forward = _fn("st_residual_norm", _vp, *[_cp] * 10)
    x, r, post, gate, pre = (_desc(d[k]) for k in ("x", "r", "post", "gate", "pre"))
    assert forward(ctx, x, r, post, gate, pre, None, _desc(normed), None, opt, ex) == 0
    dx, dgate = torch.empty_like(d["x"]), torch.empty(rows, 1, device=DEV)
    backward = _fn("st_residual_norm_backward", _vp, *[_cp] * 12, _vp, _u64, _cp, _cp)
    assert backward(ctx, _desc(dr), _desc(dh), x, _desc(want.residual), post, gate, pre, _desc(dx), None, None, _desc(dgate),
                    None, None, 0, opt, ex) == 0
    torch.cuda.synchronize()
    # the same arithmetic in another instance of the kernel: one step of the type and the sums' bound apart at most
    for got, ref, dtype in [(normed, want.normed, BF16), (dx, back.x, BF16), (dgate, back.gate, F32)]:
        mass = ref.double().abs().cpu() + ref.double().abs().max().cpu()
        close(got, ref.double().cpu(), mass, dtype, rel=REL + torch.finfo(dtype).eps / 2)


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows,cols", [(7, 96), (5, 301), (700, 1024), (3, 12001)], ids=lambda v: str(v))
def test_backward_of_the_stream_alone(rows, cols, dtype):
    """d_residual and nothing else: the stream's gradient as it is, read and written in its own type.  d_residual is a
    row block among others, so that a read in a wider type would bring in its neighbours; the updated stream, given or
    not, does not matter without pre_weight."""
    room = torch.randn(3 * rows, cols, generator=gen(rows)).to(dtype).to(DEV)
    d = room[rows:2 * rows]
    for residual in (None, torch.zeros(rows, cols, dtype=dtype, device=DEV)):
        got = st.residual_norm_backward(d, None, None, residual)
        assert got.residual.dtype == dtype and torch.equal(got.residual, d)
        assert got.x is None and got.post_weight is None and got.gate is None and got.pre_weight is None


@pytest.mark.parametrize("dtype", [F32, F16, BF16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("rows", [5, 700])
def test_backward_of_the_stream_alone_writes_dr_only(rows, dtype):
    """The same call in C with dr inside a larger array: nothing around it is written."""
    from sptiles_b200.api import _exec_desc
    from sptiles_b200.fp8 import _cp, _desc, _fn, _u64, _vp
    from sptiles_b200.norm import _OPTIONS

    cols = 1024
    d = torch.randn(rows, cols, generator=gen(2)).to(dtype).to(DEV)
    room = torch.full((3 * rows, cols), 3.0, dtype=dtype, device=DEV)
    dr = room[rows:2 * rows]
    backward = _fn("st_residual_norm_backward", _vp, *[_cp] * 12, _vp, _u64, _cp, _cp)
    assert backward(st.runtime.context(0), _desc(d), *[None] * 7, _desc(dr), None, None, None, None, 0,
                    _OPTIONS.pack(1.0, EPS, 0.0), _exec_desc(0)) == 0
    assert torch.equal(dr, d)
    assert (room[:rows] == 3.0).all() and (room[2 * rows:] == 3.0).all()


# ------------------------------------------------------------------ weights and gates of another type than x
def float32_sides(d, names):
    return {k: v.float() if k in names and v is not None else v for k, v in d.items()}


@pytest.mark.parametrize("names", [("gate",), ("post",), ("gate", "post", "pre")], ids="+".join)
@pytest.mark.parametrize("gate", ["none", "channel", "row", "token", "full"])
@pytest.mark.parametrize("tx,tr", [(F16, F16), (BF16, BF16), (BF16, F32)], ids=["f16", "bf16", "bf16_f32"])
@pytest.mark.parametrize("rows,cols", [(5, 96), (4, 1101), (700, 1024), (333, 2056), (300, 4104)], ids=lambda v: str(v))
def test_float32_gate_and_weights_beside_16_bits(rows, cols, tx, tr, gate, names):
    """float32 gates and weights beside a 16-bit x, forward to both kinds of copies and backward, on the generic
    kernels and on the rings; a gate's gradient comes in the gate's type."""
    d = inputs(rows, cols, tx, tr, gate, True, True, seed=6)
    g = gen(7)
    d = float32_sides(d, names)
    for k in names:  # values that 16 bits do not hold
        if d[k] is not None:
            d[k] = d[k] + 1e-4 * torch.randn(d[k].shape, generator=g)
    check_forward(d)
    check_forward(d, quantize=True, offset=0.5)
    full = gate == "full" and d["gate"].dtype == F32
    if not full:
        check_backward(d, rows, cols, tx, tr, offset=0.5)
        return
    dr, dh = torch.randn(rows, cols, generator=g).to(tr), torch.randn(rows, cols, generator=g).to(tx)
    c = dev(d)
    got = st.residual_norm_backward(dr.to(DEV), dh.to(DEV), c["x"], c["r"], c["post"], c["gate"], c["pre"], alpha=0.7, eps=EPS)
    want, mass = backward64(dbl(d), dr.double(), dh.double(), 0.7, 0.0)
    close(got.gate, want["gate"], mass["gate"], F32)
    close(got.x, want["x"], mass["x"], tx)
    close(got.residual, want["residual"], mass["residual"], tr)
    for value, name in ((got.post_weight, "post"), (got.pre_weight, "pre")):
        close(value, want[name], mass[name], F32, rel=REL + (rows + 64) * 2.0 ** -24)


# ------------------------------------------------------------------ NaN and infinities through the rings
BAD_ROWS = {5: float("nan"), 297: float("inf"), 640: float("-inf")}


def test_forward_ring_keeps_bad_rows_apart():
    """Rows of NaN and infinity among rows that the same CTAs take before and after them: every other row has the bits
    that it has without them, its 8-bit codes and scales too."""
    for gate in ("none", "channel", "token", "full"):
        d = inputs(900, 1024, BF16, F32, gate, True, True, seed=5)
        for quantize in (False, True):
            run = lambda v: st.residual_norm(v["x"], v["r"], v["post"], v["gate"], v["pre"], eps=EPS, quantize=quantize)  # noqa: E731
            want = run(dev(d))
            bad = dict(d, x=d["x"].clone(), r=d["r"].clone())
            for i, (row, v) in enumerate(BAD_ROWS.items()):
                bad["x" if i % 2 == 0 else "r"][row, 100 * i + 7] = v
            got = run(dev(bad))
            fine = torch.ones(900, dtype=torch.bool)
            fine[list(BAD_ROWS)] = False
            for a, b in zip(got, want):
                if a is None:
                    continue
                a, b = (v.cpu().view(torch.uint8) if v.element_size() == 1 else v.cpu() for v in (a, b))
                assert torch.equal(a[fine], b[fine])
            assert torch.isnan(got.residual[5]).all()  # x's NaN is in its row's norm
            assert not torch.isfinite(got.residual[297, 107]) and not torch.isfinite(got.residual[640, 207])
            if quantize:  # what reads the blocks' codes and scales gets NaN where the row is bad
                assert torch.isnan(got.scale[5]).all()


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
def test_backward_ring_keeps_bad_rows_apart(gate):
    """The same backward: dx, dr and a row's own gate gradient of every other row keep their bits; sums over rows
    are not finite in the columns that a bad row reaches."""
    rows, cols = 900, 1024
    d = inputs(rows, cols, BF16, F32, gate, True, True, seed=5)
    dr, dh = torch.randn(rows, cols, generator=gen(1)), torch.randn(rows, cols, generator=gen(2)).to(BF16)
    run = lambda v, p, q: st.residual_norm_backward(p.to(DEV), q.to(DEV), v["x"], v["r"], v["post"], v["gate"], v["pre"],  # noqa: E731
                                                    eps=EPS)
    want = run(dev(d), dr, dh)
    x, p, q = d["x"].clone(), dr.clone(), dh.clone()
    x[5, 7], p[297, 107], q[640, 207] = float("nan"), float("inf"), float("nan")
    got = run(dev(dict(d, x=x)), p, q)
    fine = torch.ones(rows, dtype=torch.bool)
    fine[list(BAD_ROWS)] = False
    own = [(got.x, want.x), (got.residual, want.residual)] + ([(got.gate, want.gate)] if gate in ("token", "full") else [])
    for a, b in own:
        assert torch.equal(a.cpu()[fine], b.cpu()[fine])
    assert torch.isnan(got.x[5]).all() and torch.isfinite(got.residual[5]).all()
    assert torch.isinf(got.residual[297, 107]) and torch.isnan(got.residual[640]).all()
    assert torch.isnan(got.post_weight).all() and torch.isnan(got.pre_weight[207])
    if gate == "channel":
        assert torch.isnan(got.gate).all()


@pytest.mark.parametrize("rows", [6, 700])
@pytest.mark.parametrize("eps,alpha,offset", [(0.0, -1.5, 0.0), (1e-12, 0.0, 1.0), (1e-2, 3.0, -0.25), (10.0, 1.0, 2.0)])
def test_other_options(rows, eps, alpha, offset, monkeypatch):
    """eps, alpha and weight_offset over their range, none of them the defaults, on the generic kernels and on the rings."""
    monkeypatch.setitem(globals(), "EPS", eps)
    # backward64's masses of what alpha scales carry alpha's sign: alpha * (a sum of magnitudes), so that sum of magnitudes
    # is their absolute value
    plain = backward64
    monkeypatch.setitem(globals(), "backward64", lambda *a: (lambda v, m: (v, {k: t.abs() for k, t in m.items()}))(*plain(*a)))
    for gate in ("channel", "token"):
        d = inputs(rows, 1024, F32, F32, gate, True, True, seed=8)
        check_forward(d, alpha=alpha, offset=offset)
        check_backward(d, rows, 1024, F32, F32, alpha=alpha, offset=offset)
