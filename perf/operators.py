"""Timed cases of the 8-bit block-scaled matmul, the quantiser that feeds it and the norms around a block.

Each operator in two forms: elementary torch operations in 32 bits, and the
package's own call.  With s a block's scale (one float32 for 128 elements
along the contraction, or for a 128 x 128 block of weights):

  quantize  s = max(max|x| / 448, 2^-126) (57344 for e5m2);  q = fp8(x * (1 / s))
  matmul    C[m, n] = sum_b sa[m, b] sb[b, n] sum_{k in block b} A[m, k] B[k, n]  (+ bias[n])
  norm      r' = r + alpha * gate * rms(x) * (post + offset);   h = rms(r') * (pre + offset)
            with rms(v) = v / sqrt(mean(v^2) + eps), h also as 8-bit blocks;
            backward: from dr' and dh to dx, dr, dgate, dpost and dpre
"""
import math

import torch

own = False

BLOCK = 128
EPS = 1e-6
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16,
         "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1, "e5m2": 1}
BLOCKS = {"1x128": (1, 128), "128x1": (128, 1), "128x128": (128, 128)}


def listed():
    return [
        # one token's hidden state before a projection: latency
        dict(name="quantize token", op="quantize", rows=1, cols=4096, block="1x128", x="bf16", q="e4m3"),
        # the activations of a long prompt, row blocks for the forward product
        dict(name="quantize activations", op="quantize", rows=8192, cols=8192, block="1x128", x="bf16", q="e4m3"),
        # master weights in fp32 at odd sizes, square blocks
        dict(name="quantize weights odd", op="quantize", rows=4111, cols=2049, block="128x128", x="f32", q="e4m3"),
        # decoding one sequence: the weights are read once
        dict(name="matmul token", op="matmul", m=1, n=8192, k=8192, a="e4m3", b="e4m3", a_rows=True, b_rows=False,
             b_scale="block", out="bf16", bias=False),
        # decoding a batch of odd size at odd widths, with a bias
        dict(name="matmul batch odd", op="matmul", m=57, n=4109, k=4001, a="e4m3", b="e4m3", a_rows=True, b_rows=False,
             b_scale="block", out="bf16", bias=True),
        # a short prompt through a square layer
        dict(name="matmul prompt 1024", op="matmul", m=1024, n=1024, k=1024, a="e4m3", b="e4m3", a_rows=True,
             b_rows=False, b_scale="block", out="f32", bias=False),
        # the package's own large square product
        dict(name="matmul 8192", op="matmul", m=8192, n=8192, k=8192, a="e4m3", b="e4m3", a_rows=True, b_rows=False,
             b_scale="block", out="bf16", bias=False),
        # gradient of a layer's weights: both operands stored along the output, contraction over the tokens
        dict(name="matmul weight gradient", op="matmul", m=4096, n=4096, k=16384, a="e5m2", b="e4m3", a_rows=False,
             b_rows=True, b_scale="column", out="f32", bias=False),
        # one token between two blocks: latency
        dict(name="norm token", op="norm", direction="forward", rows=1, cols=4096, x="bf16", r="bf16", post=True,
             gate="channel", pre=True, quantize=True),
        # a prompt between two blocks, handed to the 8-bit product
        dict(name="norm prompt", op="norm", direction="forward", rows=16384, cols=4096, x="bf16", r="bf16", post=True,
             gate="channel", pre=True, quantize=True),
        # odd sizes, a gate for each element, residual stream in fp32
        dict(name="norm odd", op="norm", direction="forward", rows=1025, cols=2049, x="f16", r="f32", post=True,
             gate="full", pre=True, quantize=False),
        # a training step's way back
        dict(name="norm backward", op="norm", direction="backward", rows=8192, cols=4096, x="bf16", r="bf16", post=True,
             gate="channel", pre=True, quantize=False),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "matmul", "matmul", "norm", "norm"])
    if op == "quantize":
        rows, cols = _spread(rng, 1, 16384), _spread(rng, 1, 16384)
        cols = max(1, min(cols, 8192 * 8192 // rows))
        return dict(op=op, rows=rows, cols=cols, block=rng.choice(sorted(BLOCKS)), x=rng.choice(["f32", "f16", "bf16"]),
                    q=rng.choice(["e4m3", "e4m3", "e5m2"]))
    if op == "matmul":
        m, n, k = _spread(rng, 1, 16384), _spread(rng, 16, 16384), _spread(rng, 1, 16384)
        while m * n * k > 8192 ** 3:
            m = (m + 1) // 2
        return dict(op=op, m=m, n=n, k=k, a=rng.choice(["e4m3", "e4m3", "e5m2"]), b=rng.choice(["e4m3", "e4m3", "e5m2"]),
                    a_rows=rng.random() < 0.7, b_rows=rng.random() < 0.4, b_scale=rng.choice(["block", "column"]),
                    out=rng.choice(["bf16", "f16", "f32"]), bias=rng.random() < 0.3)
    # hidden sizes from 32: on a few elements a norm's gradient is the difference of nearly equal numbers
    rows, cols = _spread(rng, 1, 16384), _spread(rng, 32, 16384)
    cols = max(32, min(cols, 16384 * 4096 // rows))
    direction = rng.choice(["forward", "backward"])
    x = rng.choice(["f32", "f16", "bf16"])
    post, gate = rng.random() < 0.7, rng.choice(["none", "channel", "token", "full"])
    return dict(op=op, direction=direction, rows=rows, cols=cols, x=x, r=rng.choice([x, "f32"]), post=post, gate=gate,
                pre=rng.random() < 0.8, quantize=direction == "forward" and rng.random() < 0.4)


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _store(t, dtype):
    """t in dtype, its rows starting on 16-byte boundaries (as the package's quantiser lays them out)."""
    pad = -t.shape[1] % 16
    room = torch.zeros(t.shape[0], t.shape[1] + pad, dtype=dtype, device="cuda")
    room[:, : t.shape[1]] = t.to(dtype)
    return room[:, : t.shape[1]]


def _limit(q):
    return torch.finfo(TYPES[q]).max


def _operand(g, rows, cols, q, square):
    """8-bit rows x cols (blocks along cols) and its scales [rows or its blocks, blocks of cols]: normal values
    whose size differs from row to row and in a few columns, as activations and weights have it."""
    x = _randn(g, rows, cols) * torch.exp(0.5 * _randn(g, rows, 1)) * torch.exp(0.3 * _randn(g, 1, cols))
    br = BLOCK if square else 1
    pr, pc = -rows % br, -cols % BLOCK
    top = torch.nn.functional.pad(x.abs(), (0, pc, 0, pr)).view((rows + pr) // br, br, (cols + pc) // BLOCK, BLOCK)
    s = top.amax((1, 3)).clamp(min=1e-20) / _limit(q)
    wide = s.repeat_interleave(br, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :cols]
    return (x / wide).clamp(-_limit(q), _limit(q)), s


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    if c["op"] == "quantize":
        x = _randn(g, c["rows"], c["cols"]) * torch.exp(_randn(g, c["rows"], 1))
        return {"case": c, "x": x.to(TYPES[c["x"]])}
    if c["op"] == "matmul":
        qa, sa = _operand(g, c["m"], c["k"], c["a"], False)
        qb, sb = _operand(g, c["n"], c["k"], c["b"], c["b_scale"] == "block")
        # scales lie with the rows (of A) and columns (of B) contiguous, as the package's quantiser writes them
        a = _store(qa, TYPES[c["a"]]) if c["a_rows"] else _store(qa.t(), TYPES[c["a"]]).t()
        b = _store(qb.t(), TYPES[c["b"]]) if c["b_rows"] else _store(qb, TYPES[c["b"]]).t()
        bias = _randn(g, c["n"]) if c["bias"] else None
        return {"case": c, "a": a, "b": b, "sa": sa.t().contiguous().t(), "sb": sb.t().contiguous(), "bias": bias}
    t, n = c["rows"], c["cols"]
    tx, tr = TYPES[c["x"]], TYPES[c["r"]]
    s = {"case": c, "x": (_randn(g, t, n) * torch.exp(0.5 * _randn(g, t, 1))).to(tx), "r": (2.0 * _randn(g, t, n)).to(tr)}
    s["post"] = (0.2 + 0.05 * _randn(g, n)).to(tx) if c["post"] else None
    s["pre"] = (1.0 + 0.2 * _randn(g, n)).to(tx) if c["pre"] else None
    shape = {"none": None, "channel": (n,), "token": (t, 1), "full": (t, n)}[c["gate"]]
    s["gate"] = (0.5 + 0.5 * _randn(g, *shape)).to(tx) if shape else None
    if c["direction"] == "backward":
        s["dr"] = (0.01 * _randn(g, t, n)).to(tr)
        s["dh"] = (0.01 * _randn(g, t, n)).to(tx) if c["pre"] else None
    return s


ALPHA = 0.5


# ------------------------------------------------------------------ the calls
def run(state):
    op = state["case"]["op"]
    if op == "quantize":
        return _run_quantize(state)
    if op == "matmul":
        return _run_matmul(state)
    return _run_forward(state) if state["case"]["direction"] == "forward" else _run_backward(state)


def _run_quantize(s):
    c = s["case"]
    if own:
        import sptiles_b200 as st

        q, scale = st.quantize_fp8(s["x"], block=BLOCKS[c["block"]], dtype=TYPES[c["q"]])
        return {"q": q, "scale": scale}
    return dict(zip(("q", "scale"), _plain_blocks(s["x"].float(), BLOCKS[c["block"]], c["q"])))


def _plain_blocks(x, block, q):
    rows, cols = x.shape
    br, bc = block
    pr, pc = -rows % br, -cols % bc
    wide = torch.nn.functional.pad(x, (0, pc, 0, pr)).view((rows + pr) // br, br, (cols + pc) // bc, bc)
    limit = torch.full((), _limit(q), device=x.device)
    scale = (wide.abs().amax((1, 3)) / limit).clamp(min=2.0 ** -126)
    inverse = (torch.ones((), device=x.device) / scale)[:, None, :, None]
    codes = (wide * inverse).clamp(-limit, limit).to(TYPES[q])
    return codes.view(rows + pr, cols + pc)[:rows, :cols], scale


def _run_matmul(s):
    c = s["case"]
    if own:
        import sptiles_b200 as st

        return st.matmul_fp8(s["a"], s["b"], s["sa"], s["sb"], s["bias"], out_dtype=TYPES[c["out"]])
    kb = torch.arange(c["k"], device="cuda") // BLOCK
    nb = torch.arange(c["n"], device="cuda") // (BLOCK if c["b_scale"] == "block" else 1)
    a = s["a"].float() * s["sa"][:, kb]
    b = s["b"].float() * s["sb"][kb][:, nb]
    out = a @ b
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(TYPES[c["out"]])


def _run_forward(s):
    c = s["case"]
    if own:
        import sptiles_b200 as st

        got = st.residual_norm(s["x"], s["r"], s["post"], s["gate"], s["pre"], alpha=ALPHA, eps=EPS,
                               quantize=c["quantize"] and c["pre"])
        return {"residual": got.residual, "normed": got.normed, "scale": got.scale}
    u = s["x"].float()
    if s["post"] is not None:
        u = u * torch.rsqrt(u.square().mean(1, keepdim=True) + EPS) * s["post"].float()
    if s["gate"] is not None:
        u = u * s["gate"].float()
    r = s["r"].float() + ALPHA * u
    h = scale = None
    if s["pre"] is not None:
        h = r * torch.rsqrt(r.square().mean(1, keepdim=True) + EPS) * s["pre"].float()
        if c["quantize"]:
            h, scale = _plain_blocks(h, (1, BLOCK), "e4m3")
        else:
            h = h.to(TYPES[c["x"]])
    return {"residual": r.to(TYPES[c["r"]]), "normed": h, "scale": scale}


def _run_backward(s):
    """s["r"] is the residual stream that the forward call returned."""
    c = s["case"]
    if own:
        import sptiles_b200 as st

        got = st.residual_norm_backward(s["dr"], s["dh"], s["x"], s["r"], s["post"], s["gate"], s["pre"], alpha=ALPHA,
                                        eps=EPS)
        return {"x": got.x, "residual": got.residual, "post": got.post_weight, "gate": got.gate, "pre": got.pre_weight}
    dr, dpre, dpost, dgate = s["dr"].float(), None, None, None
    if s["pre"] is not None:
        r, dh = s["r"].float(), s["dh"].float()
        inv = torch.rsqrt(r.square().mean(1, keepdim=True) + EPS)
        rhat = r * inv
        dpre = (dh * rhat).sum(0)
        t = dh * s["pre"].float()
        dr = dr + inv * (t - rhat * (t * rhat).mean(1, keepdim=True))
    x = s["x"].float()
    gate = s["gate"].float() if s["gate"] is not None else torch.ones((), device="cuda")
    if s["post"] is not None:
        inv = torch.rsqrt(x.square().mean(1, keepdim=True) + EPS)
        xhat = x * inv
        w = s["post"].float()
    else:
        xhat, w = x, torch.ones((), device="cuda")
    du = ALPHA * gate * dr
    if s["post"] is not None:
        dpost = (du * xhat).sum(0)
        t = du * w
        dx = inv * (t - xhat * (t * xhat).mean(1, keepdim=True))
    else:
        dx = du
    if s["gate"] is not None:
        dgate = ALPHA * dr * xhat * w
        if c["gate"] == "channel":
            dgate = dgate.sum(0)
        elif c["gate"] == "token":
            dgate = dgate.sum(1, keepdim=True)
        else:
            dgate = dgate.to(TYPES[c["x"]])
    return {"x": dx.to(TYPES[c["x"]]), "residual": dr.to(TYPES[c["r"]]), "post": dpost, "gate": dgate, "pre": dpre}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "quantize":
        br, bc = BLOCKS[c["block"]]
        n = c["rows"] * c["cols"]
        return {"bytes": n * (SIZE[c["x"]] + 1) + 4 * -(-c["rows"] // br) * -(-c["cols"] // bc), "flops": 3 * n}
    if c["op"] == "matmul":
        m, n, k = c["m"], c["n"], c["k"]
        kb = -(-k // BLOCK)
        scales = m * kb + kb * (-(-n // BLOCK) if c["b_scale"] == "block" else n)
        return {"bytes": m * k + n * k + 4 * scales + m * n * SIZE[c["out"]] + (4 * n if c["bias"] else 0),
                "flops": 2 * m * n * k}
    n, sx, sr = c["rows"] * c["cols"], SIZE[c["x"]], SIZE[c["r"]]
    gate = {"none": 0, "channel": c["cols"], "token": c["rows"], "full": n}[c["gate"]]
    if c["direction"] == "forward":
        h = 0 if not c["pre"] else n * 1 + 4 * c["rows"] * -(-c["cols"] // BLOCK) if c["quantize"] else n * sx
        return {"bytes": n * (sx + 2 * sr) + h + gate * sx + 2 * c["cols"] * sx, "flops": 10 * n}
    dgate = gate * (sx if c["gate"] == "full" else 4)
    return {"bytes": n * (2 * sx + 2 * sr) + (n * (sx + sr) if c["pre"] else 0) + gate * sx + dgate + 2 * c["cols"] * (sx + 4),
            "flops": 24 * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "quantize":
        return dict(zip(("q", "scale"), _exact_blocks(s["x"].double(), BLOCKS[c["block"]], c["q"])))
    if c["op"] == "matmul":
        return _exact_matmul(s)
    d = {k: v.double() if isinstance(v, torch.Tensor) else v for k, v in s.items()}
    if c["direction"] == "forward":
        r = d["r"] + _exact_branch(d["x"], d["post"], d["gate"])
        h, scale = (None, None) if d["pre"] is None else (_exact_rms(r, d["pre"]), None)
        if c["quantize"] and h is not None:
            h, scale = _exact_blocks(h, (1, BLOCK), "e4m3")
        return {"residual": r, "normed": h, "scale": scale}
    return _exact_backward(d)


def _exact_blocks(x, block, q):
    """The values before their rounding to 8 bits, and the scales."""
    br, bc = block
    i = torch.arange(x.shape[0], device="cuda")[:, None] // br
    j = torch.arange(x.shape[1], device="cuda")[None, :] // bc
    nb = -(-x.shape[1] // bc)
    top = torch.zeros(-(-x.shape[0] // br) * nb, dtype=torch.float64, device="cuda")
    at = i * nb + j
    top.scatter_reduce_(0, at.reshape(-1), x.abs().reshape(-1), "amax")
    scale = torch.maximum(top / _limit(q), torch.full_like(top, 2.0 ** -126))
    return x / scale[at], scale.view(-1, nb)


def _exact_matmul(s):
    c = s["case"]
    pad = -c["k"] % BLOCK
    a, b = (torch.nn.functional.pad(t.double(), p) for t, p in ((s["a"], (0, pad)), (s["b"], (0, 0, 0, pad))))
    a = (a.unflatten(1, (-1, BLOCK)) * s["sa"].double()[:, :, None]).flatten(1)
    sb = s["sb"].double()
    if c["b_scale"] == "block":
        sb = sb.repeat_interleave(BLOCK, 1)[:, : c["n"]]
    b = (b.unflatten(0, (-1, BLOCK)) * sb[:, None, :]).flatten(0, 1)
    out = torch.mm(a, b)
    return out if s["bias"] is None else torch.add(out, s["bias"].double())


def _exact_rms(v, w):
    return w * v / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + EPS)


def _exact_branch(x, post, gate):
    u = x if post is None else _exact_rms(x, post)
    return ALPHA * u if gate is None else ALPHA * gate * u


def _exact_backward(d):
    """By differentiating the forward definition."""
    leaf = {k: d[k].requires_grad_() for k in ("x", "r", "post", "gate", "pre") if d[k] is not None}
    out = {k: None for k in ("x", "residual", "post", "gate", "pre")}
    total = d["dr"]
    if "pre" in leaf:
        g = torch.autograd.grad(_exact_rms(leaf["r"], leaf["pre"]), [leaf["r"], leaf["pre"]], d["dh"])
        total, out["pre"] = total + g[0], g[1]
    names = [k for k in ("x", "post", "gate") if k in leaf]
    grads = torch.autograd.grad(_exact_branch(leaf["x"], leaf.get("post"), leaf.get("gate")), [leaf[k] for k in names], total)
    out.update(zip(names, grads))
    out["residual"] = total
    return out
