"""The operators that a training step of the pair stack needs beside its transition: the relative
position embedding with its gradient, matrix products of 4-bit operands with their gradients, and
the orthogonalised update of weight matrices.

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs, weights and buffers on the GPU
    run(state)          one pass: through localfold_amd.device where `own`, else in plain torch
    work(case)          bytes and operations that the pass cannot do without
    exact(case, seed)   the same outputs in float64, written apart from the plain form

Kinds: "position" (a learned row per bucket of p_i - p_j for every pair, forward or backward),
"linear4" (activations quantised to 4 bits, times a packed weight), "linear4_backward" (the gradient
quantised both ways, the input's, weight's and bias's gradients) and "update" (matrices made
orthogonal by Newton-Schulz products, alone or as an optimiser step with momentum and decay).

A bucket is the number of ascending boundaries that are at most p_i - p_j.  With segments, pairs of
different segments take the table's last row, and a negative segment is padding: its pairs get
nothing and give nothing.

4 bits are e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives), two a byte, the lower column
in the lower half, rows padded to a multiple of 128 columns with zeros; 32 columns of a row share a
power of two 2^(b - 127), the smallest that puts them within 6, its bytes b as [groups, rows rounded
up to 16].
"""
import math

import torch

own = False

GROUP = 32           # columns that share a scale
LARGEST = 6.0        # of e2m1
EPS = 1e-7
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
RATE, DECAY, MOMENTUM = 0.02, 0.1, 0.95
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACT_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
WIDTHS = (64, 128, 256, 384)   # extra-MSA, pair, MSA and single channels


def listed():
    return [
        # the pair track of a short protein (59 residues), clipped at 32: one launch's latency
        {"name": "position_59", "kind": "position", "direction": "forward", "queries": 59, "keys": 59, "c": 128,
         "scheme": "clip", "reach": 32, "buckets": 65, "segments": False, "base": False, "dtype": "f32"},
        # added to the pair track of a long complex (825 residues in chains, some padding)
        {"name": "position_825", "kind": "position", "direction": "forward", "queries": 825, "keys": 825, "c": 128,
         "scheme": "clip", "reach": 32, "buckets": 65, "segments": True, "base": True, "dtype": "bf16"},
        # the table's gradient at a training crop (384 residues)
        {"name": "position_grad_384", "kind": "position", "direction": "backward", "queries": 384, "keys": 384,
         "c": 128, "scheme": "clip", "reach": 32, "buckets": 65, "segments": True, "base": False, "dtype": "bf16"},
        # the gradient of a bias per head, logarithmic buckets, odd lengths, full precision
        {"name": "position_grad_log_1003", "kind": "position", "direction": "backward", "queries": 777, "keys": 1003,
         "c": 16, "scheme": "log", "reach": 512, "buckets": 32, "segments": False, "base": False, "dtype": "f32"},
        # one row through a wide layer, where the weights are what is read
        {"name": "linear4_row", "kind": "linear4", "rows": 1, "inputs": 4096, "outputs": 4096, "dtype": "bf16",
         "relu": False, "residual": False},
        # the first product of the pair transition at the training crop
        {"name": "linear4_pair_384", "kind": "linear4", "rows": 384 * 384, "inputs": 128, "outputs": 512,
         "dtype": "bf16", "relu": True, "residual": False},
        # a large generic product, where the matrix cores are the limit
        {"name": "linear4_4096", "kind": "linear4", "rows": 8192, "inputs": 4096, "outputs": 4096, "dtype": "bf16",
         "relu": False, "residual": False},
        # the backward pass of a pair projection at an ordinary length, full precision gradients
        {"name": "linear4_grad_301", "kind": "linear4_backward", "rows": 301 * 301, "inputs": 128, "outputs": 128,
         "dtype": "f32"},
        # the backward pass of the MSA transition's first product at full MSA depth
        {"name": "linear4_grad_msa_384", "kind": "linear4_backward", "rows": 512 * 384, "inputs": 256,
         "outputs": 1024, "dtype": "bf16"},
        # one extra-MSA transition matrix by itself
        {"name": "update_extra", "kind": "update", "batch": 1, "rows": 64, "cols": 256, "steps": 5, "step": False,
         "dtype": "f32"},
        # the optimiser's step of the pair transitions of 48 blocks
        {"name": "update_pair_48", "kind": "update", "batch": 48, "rows": 128, "cols": 512, "steps": 5, "step": True,
         "dtype": "f32"},
        # a large generic matrix in 16 bits, taller than wide
        {"name": "update_4096", "kind": "update", "batch": 1, "rows": 4096, "cols": 1024, "steps": 5, "step": True,
         "dtype": "bf16"},
    ]


def draw(rng):
    def log_int(lo, hi):
        hi = max(lo, hi)
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def width(lo, hi):   # one of the trunk's, or any
        return rng.choice([rng.choice(WIDTHS), rng.choice(WIDTHS), log_int(lo, hi)])

    kind = rng.choice(["position", "position", "linear4", "linear4", "linear4_backward", "update"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
    if kind == "position":
        c["direction"] = rng.choice(["forward", "backward"])
        c["c"] = rng.choice([128, 128, 64, 16, log_int(1, 384)])
        most = 825 * 825 * 128 // c["c"]
        c["queries"] = log_int(1, 1024)
        c["keys"] = rng.choice([c["queries"], log_int(16, 2048)])
        c["queries"] = max(1, min(c["queries"], most // c["keys"]))
        c["scheme"] = rng.choice(["clip", "clip", "log"])
        c["reach"] = log_int(1, 64) if c["scheme"] == "clip" else log_int(64, 2048)
        c["buckets"] = 2 * c["reach"] + 1 if c["scheme"] == "clip" else 2 * rng.randint(4, 64)
        c["segments"] = rng.choice([False, True])
        c["base"] = c["direction"] == "forward" and rng.choice([False, True])
    elif kind == "linear4":
        c["inputs"], c["outputs"] = width(22, 4096), width(22, 4096)
        c["rows"] = log_int(1, min(512 * 384, 8192 * 4096 * 4096 // (c["inputs"] * c["outputs"]),
                                   512 * 384 * 512 // (c["inputs"] + c["outputs"])))
        c["relu"], c["residual"] = rng.choice([False, True]), rng.choice([False, True])
    elif kind == "linear4_backward":
        c["inputs"], c["outputs"] = width(22, 1536), width(22, 1536)
        c["rows"] = log_int(1, min(512 * 384, 512 * 384 * 256 * 1024 // (c["inputs"] * c["outputs"]),
                                   512 * 384 * 1024 // (c["inputs"] + c["outputs"])))
    else:
        c["rows"], c["cols"] = rng.sample([width(8, 1024), width(8, 2048)], 2)
        small, large = sorted((c["rows"], c["cols"]))
        most = 1024 * 1024 * (4 * 4096 + 2 * 1024) // (small * small * (4 * large + 2 * small))
        c["batch"] = log_int(1, min(96, most))
        c["steps"], c["step"] = rng.choice([4, 5, 5, 6]), rng.choice([False, True])
    return c


# ---- what a user's program has in hand ---------------------------------------------------------

def _pitch(cols):
    return -(-cols // 128) * 128


def _scale_byte(most):
    """b of the smallest 2^(b - 127) that is at least most / 6, 1 at least."""
    m, e = torch.frexp(most)
    b = e - 3 + (m > 0.75).to(e.dtype) + 127
    return torch.where(most > 0, b, torch.ones_like(b)).clamp(1, 254)


def _power(b):
    return torch.ldexp(torch.ones_like(b, dtype=torch.float32), b - 127)


def _e2m1(v):
    """float32 within 6 rounded to e2m1, ties to even."""
    step = torch.where(v.abs() < 2, 0.5, torch.where(v.abs() < 4, 1.0, 2.0))
    return torch.round(v / step) * step


def _groups(x):
    """float32 rows padded to whole groups, [rows, groups, 32], and their scale bytes."""
    rows, cols = x.shape
    p = torch.zeros(rows, _pitch(cols), device=x.device)
    p[:, :cols] = x
    p = p.view(rows, -1, GROUP)
    return p, _scale_byte(p.abs().amax(-1))


def _quantised(x):
    """float32 rows as they are after a round trip through 4 bits."""
    p, b = _groups(x)
    f = _power(b)[:, :, None]
    return (_e2m1(p / f) * f).view(x.shape[0], -1)[:, :x.shape[1]]


def _encode(x):
    """Codes [rows, pitch / 2] and scale bytes [groups, rows to 16] of finite float32 rows."""
    p, b = _groups(x)
    v = _e2m1(p / _power(b)[:, :, None]).view(x.shape[0], -1)
    a = v.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8)
    code |= (v < 0).to(torch.uint8) << 3
    scales = torch.full((b.shape[1], -(-x.shape[0] // 16) * 16), 127, dtype=torch.uint8, device=x.device)
    scales[:, :x.shape[0]] = b.t().to(torch.uint8)
    return (code[:, 0::2] | code[:, 1::2] << 4).contiguous(), scales


def _decode(codes, scales, cols):
    code = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1)[:, :cols].to(torch.int64)
    v = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], device=codes.device)[code & 7]
    v = torch.where(code >= 8, -v, v)
    f = _power(scales[:, :codes.shape[0]].t().to(torch.int32))
    return v * f.repeat_interleave(GROUP, 1)[:, :cols]


def _activations(gen, rows, c, dtype):
    """A residual stream: unit noise around a mean per channel, a few channels several times larger,
    and rows of different size."""
    d = gen.device
    x = torch.randn(rows, c, generator=gen, device=d)
    x += torch.randn(c, generator=gen, device=d) * 0.3
    x *= torch.where(torch.rand(c, generator=gen, device=d) < 0.02, 8.0, 1.0)
    x *= torch.exp(0.4 * torch.randn(rows, 1, generator=gen, device=d))
    return x.to(DTYPES[dtype])


def _gradient(gen, rows, c, dtype):
    """A gradient: small, of very different size from row to row, nothing in the padded rows."""
    d = gen.device
    g = torch.randn(rows, c, generator=gen, device=d)
    g *= 1e-2 * torch.exp(torch.randn(rows, 1, generator=gen, device=d))
    g[rows - rows // 24:] = 0
    return g.to(DTYPES[dtype])


def _vector(gen, n, spread):
    return spread * (2 * torch.rand(n, generator=gen, device=gen.device) - 1)


def _weight_gradients(gen, batch, rows, cols, dtype):
    """Weight gradients: a few strong directions over a floor of noise."""
    d = gen.device
    rank = max(1, min(rows, cols) // 4)
    strength = 1 / torch.arange(1, rank + 1, device=d)
    g = torch.stack([(torch.randn(rows, rank, generator=gen, device=d) * strength)
                     @ torch.randn(rank, cols, generator=gen, device=d) for _ in range(batch)])
    g += 0.1 * torch.randn(batch, rows, cols, generator=gen, device=d)
    return (1e-3 * g).to(DTYPES[dtype])


def _chain(gen, n, start):
    """Residue numbers with a break, and the chain of each residue, the last ones padding."""
    d = gen.device
    p = torch.arange(start, start + n, dtype=torch.int32, device=d)
    at = int(torch.randint(0, n, (1,), generator=gen, device=d))
    p[at:] += 200
    cut = torch.randint(0, n, (2,), generator=gen, device=d)
    seg = sum((torch.arange(n, device=d) >= c).to(torch.int32) for c in cut)
    seg[n - n // 24:] = -1
    return p, seg


def _boundaries(case, device):
    """Ascending distances at which the bucket changes."""
    if case["scheme"] == "clip":
        b = list(range(1 - case["reach"], case["reach"] + 1))
    else:
        half, far = case["buckets"] // 2, case["reach"]
        near = max(1, half // 2)
        # of distances n > 0: single ones up to `near`, then ratios of (far / near)^(1 / (half - near))
        steps = [1 + i for i in range(near)]
        for j in range(1, half - near + 1):
            n = near
            while n ** (half - near) < near ** (half - near - j) * far ** j:
                n += 1
            steps.append(n)
        b = sorted([1 - s for s in steps[1:]]) + steps      # distances 0 and below mirror those above
    return torch.tensor(b, dtype=torch.int32, device=device)


_handles = {}


def _context():
    """The library handle: made once, as a program does."""
    if "ctx" not in _handles:
        from localfold_amd import device
        _handles["D"], _handles["ctx"] = device, device.Context(0)
    return _handles["D"], _handles["ctx"]


def _inputs(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    kind, dt = case["kind"], case["dtype"]
    s = {"case": dict(case)}
    if kind == "position":
        q, k, c = case["queries"], case["keys"], case["c"]
        s["boundaries"] = _boundaries(case, gen.device)
        s["kp"], s["ks"] = _chain(gen, k, 1)
        if q == k:
            s["qp"], s["qs"] = s["kp"], s["ks"]
        else:                     # the last rows of the keys', or a longer run
            s["qp"], s["qs"] = _chain(gen, q, max(1, k - q))
        if not case["segments"]:
            s["qs"] = s["ks"] = None
        rows = len(s["boundaries"]) + 1 + case["segments"]
        if case["direction"] == "forward":
            s["table"] = torch.randn(rows, c, generator=gen, device=gen.device) / math.sqrt(rows)
            s["bias"] = _vector(gen, c, 0.1)
            s["base"] = _activations(gen, q * k, c, dt).view(q, k, c) if case["base"] else None
        else:
            s["grad"] = _gradient(gen, q * k, c, dt).view(q, k, c)
    elif kind == "linear4":
        k, n = case["inputs"], case["outputs"]
        s["x"] = _activations(gen, case["rows"], k, dt)
        s["w"] = _encode(torch.randn(n, k, generator=gen, device=gen.device) / math.sqrt(k))
        s["bias"] = _vector(gen, n, 0.1)
        if case["residual"]:
            s["residual"] = _activations(gen, case["rows"], n, dt)
    elif kind == "linear4_backward":
        k, n = case["inputs"], case["outputs"]
        s["grad"] = _gradient(gen, case["rows"], n, dt)
        # kept by the forward pass: the activations, quantised along the rows
        s["x"] = _encode(_activations(gen, case["rows"], k, dt).float().t().contiguous())
        s["w"] = _encode(torch.randn(k, n, generator=gen, device=gen.device) / math.sqrt(k))   # [in, out]
    else:
        shape = case["batch"], case["rows"], case["cols"]
        s["grad"] = _weight_gradients(gen, *shape, dt)
        if case["step"]:
            s["momentum"] = _weight_gradients(gen, *shape, "f32") * 5
            s["weight"] = (torch.randn(*shape, generator=gen, device=gen.device) / math.sqrt(shape[2])).to(DTYPES[dt])
    return s


def _update_scale(case):
    return 0.2 * math.sqrt(max(case["rows"], case["cols"]))


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:   # the handle, and the buffers that a program allocates once
        D, ctx = _context()
        kind, dev = case["kind"], ctx.device
        act = DTYPES[case["dtype"]]
        s["D"], s["ctx"] = D, ctx

        def new(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device=dev)

        if kind == "position" and case["direction"] == "forward":
            s["out"] = new(case["queries"], case["keys"], case["c"], dtype=act)
        elif kind == "position":
            s["dt"] = new(len(s["boundaries"]) + 1 + case["segments"], case["c"])
            s["db"] = new(case["c"])
        elif kind == "linear4":
            s["w4"] = D.Mx4(case["outputs"], case["inputs"], *s["w"])
            s["out"] = new(case["rows"], case["outputs"], dtype=act)
        elif kind == "linear4_backward":
            rows, k, n = case["rows"], case["inputs"], case["outputs"]
            s["w4"], s["x4"] = D.Mx4(k, n, *s["w"]), D.Mx4(k, rows, *s["x"])
            s["g4"], s["g4t"] = D.mx4_empty(rows, n, dev), D.mx4_empty(n, rows, dev)
            s["out"], s["dw"], s["db"] = new(rows, k, dtype=act), new(n, k), new(n)
        else:
            s["out"] = torch.empty_like(s["grad"])
            if case["step"]:
                s["momentum_out"] = torch.empty_like(s["momentum"])
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _run_own(s):
    case, D, ctx = s["case"], s["D"], s["ctx"]
    kind = case["kind"]
    if kind == "position":
        where = dict(key_positions=s["kp"], segments=s["qs"], key_segments=s["ks"])
        if case["direction"] == "forward":
            return D.relative_position(ctx, s["table"], s["boundaries"], s["qp"], bias=s["bias"], pair=s["base"],
                                       out=s["out"], **where)
        D.relative_position_backward(ctx, s["grad"], s["boundaries"], s["qp"], table_grad=s["dt"],
                                     bias_grad=s["db"], **where)
        return {"dtable": s["dt"], "dbias": s["db"]}
    if kind == "linear4":
        return D.mx4_linear(ctx, s["x"], s["w4"], s["bias"], relu=case["relu"], residual=s.get("residual"),
                            out=s["out"])
    if kind == "linear4_backward":
        D.mx4_pack(ctx, s["grad"], out=s["g4"], transposed=s["g4t"], sums=s["db"])
        D.mx4_linear(ctx, s["g4"], s["w4"], out=s["out"])
        D.mx4_linear(ctx, s["g4t"], s["x4"], out=s["dw"])
        return {"dx": s["out"], "dw": s["dw"], "db": s["db"]}
    if not case["step"]:
        return D.orthogonalize(ctx, s["grad"], steps=case["steps"], coefficients=COEFFICIENTS, epsilon=EPS, out=s["out"])
    D.muon_step(ctx, s["weight"], s["grad"], s["momentum"], rate=RATE, decay=DECAY, momentum_factor=MOMENTUM,
                nesterov=True, scale=_update_scale(case), steps=case["steps"], coefficients=COEFFICIENTS, epsilon=EPS,
                out=s["out"], momentum_out=s["momentum_out"])
    return {"weight": s["out"], "momentum": s["momentum_out"]}


def _rows_of(s):
    """The table's row of each pair, -1 where a residue is padding."""
    b = s["boundaries"]
    lo, hi = int(s["case"]["reach"]) * -1 - 1, int(s["case"]["reach"]) + 1     # past every boundary
    of = (torch.arange(lo, hi + 1, device=b.device)[:, None] >= b).sum(1)
    row = of[(s["qp"].long()[:, None] - s["kp"].long()).clamp(lo, hi) - lo]
    if s["qs"] is not None:
        row = torch.where(s["qs"][:, None] == s["ks"], row, len(b) + 1)
        row = torch.where((s["qs"][:, None] < 0) | (s["ks"] < 0), -1, row)
    return row


def _orthogonal(u, case):
    x = u / (torch.sqrt((u.double() ** 2).sum((1, 2), keepdim=True)).float() + EPS)
    flip = x.shape[1] > x.shape[2]
    if flip:
        x = x.transpose(1, 2).contiguous()
    a, b, c = COEFFICIENTS
    for _ in range(case["steps"]):
        g = torch.matmul(x, x.transpose(1, 2).contiguous())
        x = a * x + torch.matmul(b * g + c * torch.matmul(g, g), x)
    return x.transpose(1, 2) if flip else x


def _run_plain(s):
    case = s["case"]
    kind, act = case["kind"], DTYPES[case["dtype"]]
    if kind == "position":
        row = _rows_of(s)
        if case["direction"] == "forward":
            out = s["table"][row.clamp(min=0)] + s["bias"]
            out = torch.where(row[:, :, None] < 0, 0.0, out)
            return (out if s["base"] is None else s["base"].float() + out).to(act)
        rows = torch.arange(len(s["boundaries"]) + 1 + case["segments"], device=row.device)
        of = (row[:, None, :] == rows[:, None]).float()                              # [queries, rows, keys]
        table = torch.matmul(of, s["grad"].float()).sum(0, dtype=torch.float64)      # long sums
        return {"dtable": table.float(), "dbias": table.sum(0).float()}
    if kind == "linear4":
        out = _quantised(s["x"].float()) @ _decode(*s["w"], case["inputs"]).t() + s["bias"]
        if case["relu"]:
            out = out.clamp(min=0)
        if case["residual"]:
            out = out + s["residual"].float()
        return out.to(act)
    if kind == "linear4_backward":
        g = s["grad"].float()
        w, xt = _decode(*s["w"], case["outputs"]), _decode(*s["x"], case["rows"])
        gt = _quantised(g.t().contiguous())
        return {"dx": (_quantised(g) @ w.t()).to(act), "dw": gt @ xt.t(), "db": g.double().sum(0).float()}
    g = s["grad"].float()
    if not case["step"]:
        return _orthogonal(g, case).to(act)
    m = MOMENTUM * s["momentum"] + g
    o = _orthogonal(MOMENTUM * m + g, case)
    w = (1 - RATE * DECAY) * s["weight"].float() - RATE * _update_scale(case) * o
    return {"weight": w.to(act), "momentum": m}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    kind, b = case["kind"], ACT_BYTES[case["dtype"]]

    def kept(rows, cols):
        return rows * cols // 2 + rows * -(-cols // GROUP)

    if kind == "position":
        q, k, c = case["queries"], case["keys"], case["c"]
        table = 4 * c * (case["buckets"] + 2 + case["segments"])
        marks = 4 * (q + k) * (2 if case["segments"] else 1)
        return {"bytes": q * k * c * b * (2 if case["base"] else 1) + table + marks, "flops": q * k * c}
    if kind == "linear4":
        r, k, n = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": r * k * b + kept(n, k) + 4 * n + r * n * b * (2 if case["residual"] else 1),
                "flops": 2 * r * n * k}
    if kind == "linear4_backward":
        r, k, n = case["rows"], case["inputs"], case["outputs"]
        return {"bytes": r * n * b + kept(k, r) + kept(k, n) + r * k * b + 4 * n * k + 4 * n, "flops": 4 * r * n * k}
    count = case["batch"] * case["rows"] * case["cols"]
    m, n = sorted((case["rows"], case["cols"]))
    # a product of a matrix with its own transpose, or of a symmetric one with itself, is half a product
    return {"bytes": count * (3 * b + 8 if case["step"] else 2 * b),
            "flops": case["batch"] * case["steps"] * m * m * (3 * n + m)}


# ---- in float64, from the definitions -------------------------------------------------------------

def _quantised64(x):
    """Doubles through 4 bits, groups along the last dimension, by the nearest of e2m1's values."""
    out = torch.empty_like(x)
    for g in range(0, x.shape[1], GROUP):
        part = x[:, g:g + GROUP]
        most = part.abs().max(1, keepdim=True).values
        e = torch.floor(torch.log2(most.clamp(min=1e-300) / LARGEST))
        e = torch.where(most > LARGEST * torch.exp2(e), e + 1, e)       # log2 may be off by one either way
        e = torch.where(most <= LARGEST * torch.exp2(e - 1), e - 1, e)
        f = torch.exp2(torch.where(most > 0, e, torch.full_like(e, -126.0)).clamp(-126, 127))
        a = (part / f).abs()
        v = torch.zeros_like(a)
        # halfway points belong to the neighbour whose last bit is zero
        for border, up, tie in ((0.25, 0.5, False), (0.75, 1.0, True), (1.25, 1.5, False), (1.75, 2.0, True),
                                (2.5, 3.0, False), (3.5, 4.0, True), (5.0, 6.0, False)):
            v = torch.where((a >= border) if tie else (a > border), torch.full_like(v, up), v)
        out[:, g:g + GROUP] = torch.sign(part) * v * f
    return out


def _values64(codes, scales, cols):
    out = torch.empty(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    for half in (0, 1):
        c = (codes >> (4 * half)) & 15
        e, m = ((c >> 1) & 3).double(), (c & 1).double()
        v = torch.where(e == 0, m / 2, (1 + m / 2) * torch.exp2(e - 1))
        out[:, half::2] = torch.where(c >= 8, -v, v)
    b = scales[torch.arange(cols, device=codes.device) // GROUP][:, :codes.shape[0]].t()
    return out[:, :cols] * torch.exp2(b.double() - 127)


def _orthogonal64(u, steps):
    a, b, c = COEFFICIENTS
    out = []
    for x in u:
        tall = x.shape[0] > x.shape[1]
        x = x.t() if tall else x
        x = x / (torch.linalg.norm(x) + EPS)
        for _ in range(steps):
            g = x.mm(x.t())
            gx = g.mm(x)
            x = a * x + b * gx + c * g.mm(gx)
        out.append(x.t() if tall else x)
    return torch.stack(out)


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "position":
        b = s["boundaries"].long()
        d = s["qp"].long()[:, None] - s["kp"].long()
        row = torch.zeros_like(d)
        for bound in b:
            row += d >= bound
        there = torch.ones_like(d, dtype=torch.bool)
        if case["segments"]:
            row[s["qs"][:, None] != s["ks"][None, :]] = len(b) + 1
            there = (s["qs"][:, None] >= 0) & (s["ks"][None, :] >= 0)
        if case["direction"] == "forward":
            out = (s["table"].double()[row] + s["bias"].double()) * there[:, :, None]
            return out if s["base"] is None else out + s["base"].double()
        g = s["grad"].double()
        table = torch.stack([(g * ((row == r) & there)[:, :, None]).sum((0, 1))
                             for r in range(len(b) + 1 + case["segments"])])
        return {"dtable": table, "dbias": (g * there[:, :, None]).sum((0, 1))}
    if kind == "linear4":
        out = torch.matmul(_quantised64(s["x"].double()), _values64(*s["w"], case["inputs"]).t())
        out += s["bias"].double()
        if case["relu"]:
            out = torch.where(out < 0, torch.zeros_like(out), out)
        return out + s["residual"].double() if case["residual"] else out
    if kind == "linear4_backward":
        g = s["grad"].double()
        return {"dx": torch.matmul(_quantised64(g), _values64(*s["w"], case["outputs"]).t()),
                "dw": torch.matmul(_quantised64(g.t().contiguous()), _values64(*s["x"], case["rows"]).t()),
                "db": g.sum(0)}
    g = s["grad"].double()
    if not case["step"]:
        return _orthogonal64(g, case["steps"])
    m = g + MOMENTUM * s["momentum"].double()
    o = _orthogonal64(g + MOMENTUM * m, case["steps"])
    w = s["weight"].double()
    return {"weight": w - RATE * DECAY * w - RATE * _update_scale(case) * o, "momentum": m}
