"""Timed cases of 4-bit blocks (quantiser and matrix product) and of matrix products by groups of rows.

Each operator in two forms: elementary torch operations in 32 bits, and the
package's own call.  4-bit elements are e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and
their negatives), a block lies along the contraction:

  quantize  16 elements:  t = least power of two with 2688 t >= max|x| of the tensor (or of a known maximum),
                          s = e4m3(max|x| of the block / (6 t)),  q = e2m1(x / (s t))
            32 elements:  s = least power of two with 6 s >= max|x| of the block,  q = e2m1(x / s)
  product   C[m, n] = ta tb sum_k (sa A)[m, k] (sb B)[k, n]  (+ bias[n])
  grouped   rows [ends[g-1], ends[g]) of A belong to group g and meet its matrix:  C[r, n] = sum_k A[r, k] B[g, k, n];
            the gradient of the matrices:  D[g, k, n] = sum_{r in group g} A[r, k] dC[r, n]
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one token's hidden state before a 4-bit projection, its largest value known from calibration: latency
        dict(name="quantize token", op="quantize", rows=1, cols=4096, block=16, x="bf16", known=True, by_rows=True),
        # the activations of a long prompt
        dict(name="quantize activations", op="quantize", rows=8192, cols=8192, block=16, x="bf16", known=False, by_rows=True),
        # master weights in fp32 at odd sizes, blocks of 32 along their columns: the operand of the input gradient
        dict(name="quantize weights odd", op="quantize", rows=4111, cols=2049, block=32, x="f32", known=False, by_rows=False),
        # decoding one sequence: the weights are read once
        dict(name="product token", op="product", m=1, n=8192, k=8192, block=16, out="bf16", bias=False),
        # decoding a batch of odd size at odd widths, with a bias
        dict(name="product batch odd", op="product", m=57, n=4109, k=4001, block=16, out="bf16", bias=True),
        # the package's own large square product
        dict(name="product 8192", op="product", m=8192, n=8192, k=8192, block=16, out="bf16", bias=False),
        # gradient of a layer's weights, contraction over the tokens
        dict(name="product weight gradient", op="product", m=4096, n=4096, k=16384, block=32, out="f32", bias=False),
        # decoding 8 sequences with 8 experts each: the weights of the experts that are met are read once
        dict(name="grouped decode", op="grouped", direction="forward", rows=64, groups=64, k=2048, n=4096, x="bf16",
             b_rows=False, out="bf16", split=1),
        # a prompt through the experts' layer, W [g, n, k] as a layer stores it
        dict(name="grouped prompt", op="grouped", direction="forward", rows=16384, groups=32, k=4096, n=4096, x="bf16",
             b_rows=False, out="bf16", split=2),
        # few groups of odd sizes at widths off every boundary
        dict(name="grouped odd", op="grouped", direction="forward", rows=1003, groups=7, k=1001, n=515, x="f16",
             b_rows=True, out="f32", split=3),
        # the gradient of a layer's input: dy meets W as it is stored
        dict(name="grouped input gradient", op="grouped", direction="forward", rows=8192, groups=16, k=4096, n=2048,
             x="bf16", b_rows=True, out="bf16", split=4),
        # the gradient of the experts' weights, summed in fp32 for the optimiser
        dict(name="grouped weight gradient", op="grouped", direction="weights", rows=16384, groups=32, k=2048, n=4096,
             x="bf16", b_rows=True, out="f32", split=5),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["quantize", "product", "product", "grouped", "grouped"])
    if op == "quantize":
        rows, cols = _spread(rng, 1, 16384), _spread(rng, 1, 16384)
        cols = max(1, min(cols, 8192 * 8192 // rows))
        return dict(op=op, rows=rows, cols=cols, block=rng.choice([16, 32]), x=rng.choice(["f32", "f16", "bf16"]),
                    known=rng.random() < 0.4, by_rows=rng.random() < 0.6)
    if op == "product":
        m, n, k = _spread(rng, 1, 16384), _spread(rng, 16, 16384), _spread(rng, 1, 16384)
        while m * n * k > 8192 ** 3:
            m = (m + 1) // 2
        return dict(op=op, m=m, n=n, k=k, block=rng.choice([16, 16, 32]), out=rng.choice(["bf16", "f16", "f32"]),
                    bias=rng.random() < 0.3)
    # widths are multiples of 8, as layers have them, and now and then any number
    wide = rng.random() < 0.8
    rows, groups = _spread(rng, 1, 32768), _spread(rng, 1, 128)
    k, n = _spread(rng, 16, 8192), _spread(rng, 16, 8192)
    if wide:
        k, n = k // 8 * 8, n // 8 * 8
    while groups * k * n > 2 ** 29:
        groups = (groups + 1) // 2
    while rows * k * n > 16384 * 4096 * 4096:
        rows = (rows + 1) // 2
    return dict(op=op, direction=rng.choice(["forward", "forward", "weights"]), rows=rows, groups=groups, k=k, n=n,
                x=rng.choice(["bf16", "bf16", "f16"]), b_rows=rng.random() < 0.5, out=rng.choice(["bf16", "f32"])
                if rng.random() < 0.5 else "bf16", split=rng.randrange(1 << 30))


def _sizes(c):
    """Rows of each group: as a router spreads them, some experts in favour and some without a token."""
    rng = random.Random(c["split"])
    weight = [math.exp(rng.gauss(0.0, 0.8)) if rng.random() < 0.95 else 0.0 for _ in range(c["groups"])]
    if not any(weight):
        weight[0] = 1.0
    if c["rows"] <= 4096:
        sizes = [0] * c["groups"]
        for g in rng.choices(range(c["groups"]), weights=weight, k=c["rows"]):
            sizes[g] += 1
        return sizes
    total, sizes = sum(weight), []
    for w in weight:
        sizes.append(int(c["rows"] * w / total))
    sizes[max(range(len(weight)), key=weight.__getitem__)] += c["rows"] - sum(sizes)
    return sizes


# ------------------------------------------------------------------ inputs
def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _pack(index, negative):
    """Two elements a byte, the first in the low half; a row starts on a 16-byte boundary."""
    rows, cols = index.shape
    code = index.to(torch.uint8) + 8 * negative.to(torch.uint8)
    room = torch.zeros(rows, (cols + 31) // 32 * 32, dtype=torch.uint8, device="cuda")
    room[:, :cols] = code
    return (room[:, 0::2] + 16 * room[:, 1::2])[:, : (cols + 1) // 2]


def _tile(scale):
    """Scales [rows, blocks] in the product's order: [row // 128, block // 4, row % 32, row // 32 % 4, block % 4]."""
    rows, blocks = scale.shape
    byte = scale.view(torch.uint8)
    byte = torch.nn.functional.pad(byte, (0, -blocks % 4, 0, -rows % 128))
    byte = byte.view((rows + 127) // 128, 4, 32, (blocks + 3) // 4, 4).permute(0, 3, 2, 1, 4).contiguous()
    return byte.view(scale.dtype)


def _unpack(code, cols):
    half = torch.stack((code & 15, code >> 4), 2).flatten(1)[:, :cols].long()
    level = torch.tensor(LEVELS, device="cuda")[half & 7]
    return torch.where(half > 7, -level, level)


def _operand(g, rows, cols, block):
    """Codes, scales [rows, blocks] and tensor scale of normal values whose size differs from row to row."""
    x = _randn(g, rows, cols) * torch.exp(0.5 * _randn(g, rows, 1)) * torch.exp(0.3 * _randn(g, 1, cols))
    index, negative, scale, t = _plain_blocks(x, block, x.abs().amax())
    scale = scale.to(torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu)
    return _pack(index, negative), scale, t


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    c = dict(case)
    if c["op"] == "quantize":
        shape = (c["rows"], c["cols"]) if c["by_rows"] else (c["cols"], c["rows"])
        x = (_randn(g, *shape) * torch.exp(_randn(g, shape[0], 1))).to(TYPES[c["x"]])
        x = x if c["by_rows"] else x.t()
        return {"case": c, "x": x, "amax": 1.25 * x.float().abs().amax() if c["known"] and c["block"] == 16 else None}
    if c["op"] == "product":
        a, sa, ta = _operand(g, c["m"], c["k"], c["block"])
        b, sb, tb = _operand(g, c["n"], c["k"], c["block"])
        return {"case": c, "a": a, "b": b, "sa": sa, "sb": sb, "ta": ta, "tb": tb, "sa_tiled": _tile(sa), "sb_tiled": _tile(sb),
                "bias": _randn(g, c["n"]) if c["bias"] else None}
    t, e, k, n, x = c["rows"], c["groups"], c["k"], c["n"], TYPES[c["x"]]
    sizes = _sizes(c)
    ends = [sum(sizes[: i + 1]) for i in range(e)]
    s = {"case": c, "host_ends": ends, "ends": torch.tensor(ends, dtype=torch.int32, device="cuda")}
    s["a"] = (_randn(g, t, k) * torch.exp(0.3 * _randn(g, t, 1))).to(x)
    if c["direction"] == "weights":
        s["dc"] = (0.05 * _randn(g, t, n)).to(x)
        return s
    shape = (k, n) if c["b_rows"] else (n, k)
    s["b"] = torch.empty(e, *shape, dtype=x, device="cuda")
    for i in range(e):
        s["b"][i] = _randn(g, *shape) / math.sqrt(k)
    if not c["b_rows"]:
        s["b"] = s["b"].transpose(1, 2)
    return s


# ------------------------------------------------------------------ the calls
def run(state):
    op = state["case"]["op"]
    if op == "quantize":
        return _run_quantize(state)
    if op == "product":
        return _run_product(state)
    return _run_forward(state) if state["case"]["direction"] == "forward" else _run_weights(state)


def _power_of_two(top, limit, least):
    """The least power of two p >= 2^least with limit * p >= top."""
    fraction, exponent = torch.frexp(top.double() / limit)
    exponent = torch.where(fraction == 0.5, exponent - 1, exponent)
    return torch.ldexp(torch.ones_like(fraction), exponent.clamp(min=least)).float()


def _plain_blocks(x, block, amax):
    """(index of |q|, sign, scale [rows, blocks], tensor scale or None) of finite fp32 x."""
    rows, cols = x.shape
    wide = torch.nn.functional.pad(x, (0, -cols % block)).view(rows, -1, block)
    top = wide.abs().amax(2)
    t = None
    if block == 16:
        t = torch.where(amax > 0, _power_of_two(amax, 2688.0, -126), torch.ones_like(amax))
        scale = (top / t / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn).float()
        unit = scale * t
    else:
        scale = unit = torch.where(top > 0, _power_of_two(top, 6.0, -127), torch.full_like(top, 2.0 ** -127))
    # a border between two levels times the unit is exact in fp32
    y, unit = wide.abs(), unit[:, :, None]
    index = torch.zeros(wide.shape, dtype=torch.int8, device=x.device)
    for border, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        index += y >= border * unit if up else y > border * unit
    index = torch.where(unit > 0, index, torch.zeros_like(index))
    return index.flatten(1)[:, :cols], torch.signbit(x), scale, t


def _run_quantize(s):
    c = s["case"]
    kept = torch.float32 if c["x"] == "f32" else torch.bfloat16  # both hold scale * level exactly
    if own:
        import sptiles_b200 as st

        q = st.quantize_fp4(s["x"], scale_dtype=torch.float8_e4m3fn if c["block"] == 16 else torch.float8_e8m0fnu,
                            amax=s["amax"])
        values = st.dequantize_fp4(q.codes, q.scale, q.tensor_scale, cols=c["cols"], out_dtype=kept)
        return {"values": values, "tensor_scale": q.tensor_scale}
    x = s["x"].float()
    index, negative, scale, t = _plain_blocks(x, c["block"], x.abs().amax() if s["amax"] is None else s["amax"])
    level = torch.tensor(LEVELS, device="cuda")[index.long()]
    unit = (scale if t is None else scale * t).repeat_interleave(c["block"], 1)[:, : c["cols"]]
    return {"values": (torch.where(negative, -level, level) * unit).to(kept), "tensor_scale": t}


def _run_product(s):
    c = s["case"]
    if own:
        import sptiles_b200 as st

        return st.matmul_fp4(s["a"], s["b"].t(), s["sa_tiled"], s["sb_tiled"], s["bias"], a_tensor_scale=s["ta"],
                             b_tensor_scale=s["tb"], out_dtype=TYPES[c["out"]])
    block = torch.arange(c["k"], device="cuda") // c["block"]
    a = _unpack(s["a"], c["k"]) * s["sa"].float()[:, block]
    b = _unpack(s["b"], c["k"]) * s["sb"].float()[:, block]
    out = a @ b.t()
    if s["ta"] is not None:
        out = out * (s["ta"] * s["tb"])
    if s["bias"] is not None:
        out = out + s["bias"]
    return out.to(TYPES[c["out"]])


def _run_forward(s):
    c = s["case"]
    if own:
        import sptiles_b200 as st

        return st.matmul_grouped(s["a"], s["b"], s["ends"], out_dtype=TYPES[c["out"]])
    out = torch.empty(c["rows"], c["n"], dtype=TYPES[c["out"]], device="cuda")
    first = 0
    for g, end in enumerate(s["host_ends"]):
        if end > first:
            out[first:end] = (s["a"][first:end].float() @ s["b"][g].float()).to(out.dtype)
        first = end
    return out


def _run_weights(s):
    c = s["case"]
    if own:
        import sptiles_b200 as st

        return st.matmul_grouped_weights(s["a"], s["dc"], s["ends"], out_dtype=TYPES[c["out"]])
    out = torch.zeros(c["groups"], c["k"], c["n"], dtype=TYPES[c["out"]], device="cuda")
    first = 0
    for g, end in enumerate(s["host_ends"]):
        if end > first:
            out[g] = (s["a"][first:end].float().t() @ s["dc"][first:end].float()).to(out.dtype)
        first = end
    return out


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "quantize":
        n = c["rows"] * c["cols"]
        codes = c["rows"] * ((c["cols"] + 1) // 2 + -(-c["cols"] // c["block"]))
        # quantised, and taken back to the values that are compared
        return {"bytes": n * SIZE[c["x"]] + 2 * codes + n * (4 if c["x"] == "f32" else 2), "flops": 4 * n}
    if c["op"] == "product":
        m, n, k = c["m"], c["n"], c["k"]
        row = (k + 1) // 2 + -(-k // c["block"])
        return {"bytes": (m + n) * row + m * n * SIZE[c["out"]] + (4 * n if c["bias"] else 0), "flops": 2 * m * n * k}
    t, e, k, n = c["rows"], c["groups"], c["k"], c["n"]
    if c["direction"] == "weights":
        return {"bytes": t * (k + n) * SIZE[c["x"]] + e * k * n * SIZE[c["out"]], "flops": 2 * t * k * n}
    met = sum(1 for s in _sizes(c) if s)
    return {"bytes": (t * k + met * k * n) * SIZE[c["x"]] + t * n * SIZE[c["out"]], "flops": 2 * t * k * n}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = s["case"]
    if c["op"] == "quantize":
        return _exact_quantize(s)
    if c["op"] == "product":
        return _exact_product(s)
    parts = [0] + s["host_ends"]
    pairs = list(zip(parts[:-1], parts[1:]))
    if c["direction"] == "weights":
        return torch.stack([torch.mm(s["a"][i:j].double().t(), s["dc"][i:j].double()) for i, j in pairs])
    return torch.cat([torch.mm(s["a"][i:j].double(), s["b"][g].double()) for g, (i, j) in enumerate(pairs)])


def _nearest(y, levels):
    """The index of the level nearest to y; between two, the even index; above the last, the last."""
    mid = [(p + q) / 2 for p, q in zip(levels[:-1], levels[1:])]
    # y on a border goes to the lower index: where the upper one is even the border moves a hair down
    mid = [math.nextafter(b, 0.0) if i % 2 else b for i, b in enumerate(mid)]
    return torch.bucketize(y, torch.tensor(mid, dtype=torch.float64, device=y.device))


def _exact_quantize(s):
    c = s["case"]
    e4m3 = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)]
    e4m3 = e4m3[:-1]  # the last code is NaN
    t = None
    if c["block"] == 16:
        top = float(s["amax"] if s["amax"] is not None else s["x"].abs().max())
        t = 1.0
        if top > 0:
            t = 2.0 ** -126
            while 2688.0 * t < top:
                t *= 2.0
    out = []
    for rows in s["x"].split(1024):
        x = rows.double()
        cut = x.shape[1]
        parts = torch.cat((x, x.new_zeros(x.shape[0], -cut % c["block"])), 1).unflatten(1, (-1, c["block"]))
        top = parts.abs().max(2).values
        if t is not None:
            unit = torch.tensor(e4m3, dtype=torch.float64, device=x.device)[_nearest(top / (6 * t), e4m3)] * t
        else:
            unit = torch.exp2(torch.ceil(torch.log2(top / 6)).clamp(-127, 127))
            unit = torch.where(6 * unit < top, 2 * unit, torch.where(3 * unit >= top, unit / 2, unit)).clamp(min=2.0 ** -127)
        q = parts / torch.where(unit > 0, unit, torch.ones_like(unit))[:, :, None]
        level = torch.tensor(LEVELS, dtype=torch.float64, device=x.device)[_nearest(q.abs(), LEVELS)]
        out.append((torch.sign(q) * level * unit[:, :, None]).flatten(1)[:, :cut])
    return {"values": torch.cat(out), "tensor_scale": None if t is None else torch.tensor(t, dtype=torch.float64, device="cuda")}


def _exact_product(s):
    c = s["case"]

    def values(code, scale, t):
        low, high = code.to(torch.int64) % 16, code.to(torch.int64) // 16
        table = torch.tensor(LEVELS + tuple(-v for v in LEVELS), dtype=torch.float64, device=code.device)
        both = torch.empty(code.shape[0], 2 * code.shape[1], dtype=torch.float64, device=code.device)
        both[:, 0::2], both[:, 1::2] = table[low], table[high]
        both = both[:, : c["k"]] * scale.double().repeat_interleave(c["block"], 1)[:, : c["k"]]
        return both if t is None else both * t.double()

    out = torch.mm(values(s["a"], s["sa"], s["ta"]), values(s["b"], s["sb"], s["tb"]).t())
    return out if s["bias"] is None else out + s["bias"].double()
