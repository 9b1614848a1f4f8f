"""The operators that train a layer of the pair stack: LayerNorm with its gradient, activations kept
in 8 bits, matrix products of 8-bit operands with their gradients, and the transition they make up.

    listed()            the cases
    draw(rng)           one more case of the same ranges
    prepare(case, seed) inputs, weights and buffers on the GPU
    run(state)          one pass: through localfold_amd.device where `own`, else in plain torch
    work(case)          bytes and operations that the pass cannot do without
    exact(case, seed)   the same outputs in float64, written apart from the plain form

Kinds: "norm" (LayerNorm, forward or backward), "checkpoint" (activations packed to 8 bits and read
back), "linear" (activations packed, times a packed weight), "linear_backward" (the gradient
packed, the input's, weight's and bias's gradients) and "transition" (a training step of the
transition: forward, then backward).

Activations are kept as e4m3 codes [rows, pitch] (pitch: the columns rounded up to 64, zeros behind
the last) with one power of two 2^(b - 127) per row and 128 columns, the smallest that puts the
group within 448; the bytes b lie as [groups, rows rounded up to 16].  Weights have one such scale
per tile of 128 x 128, [tiles of outputs, tiles of inputs].
"""
import math

import torch

own = False

EPS = 1e-5
GROUP = 128          # columns that share a scale
LARGEST = 448.0      # of e4m3
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
ACT_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
WIDTHS = (64, 128, 256, 384)   # extra-MSA, pair, MSA and single channels


def listed():
    return [
        # the single track of a short protein (59 residues): one launch's latency
        {"name": "norm_single_59", "kind": "norm", "direction": "forward", "rows": 59, "c": 384, "dtype": "f32",
         "fast_variance": True, "kept": False},
        # the pair track of a training crop (384 residues), y and x kept in 8 bits, as a training step does
        {"name": "norm_pair_384", "kind": "norm", "direction": "forward", "rows": 384 * 384, "c": 128,
         "dtype": "bf16", "fast_variance": False, "kept": True},
        # the gradient at an ordinary length in full precision, from the activations themselves
        {"name": "norm_grad_301", "kind": "norm", "direction": "backward", "rows": 301 * 301, "c": 128,
         "dtype": "f32", "fast_variance": False, "kept": False},
        # the gradient of the MSA track (512 sequences of a 384 crop), from x kept in 8 bits
        {"name": "norm_grad_msa_384", "kind": "norm", "direction": "backward", "rows": 512 * 384, "c": 256,
         "dtype": "bf16", "fast_variance": False, "kept": True},
        # the pair activations of a long protein (825 residues) kept in 8 bits and read back
        {"name": "checkpoint_825", "kind": "checkpoint", "rows": 825 * 825, "c": 128, "dtype": "f32"},
        # a projection of the single track of a short protein
        {"name": "linear_single_59", "kind": "linear", "rows": 59, "inputs": 384, "outputs": 1536, "dtype": "bf16",
         "relu": False, "residual": False},
        # the first product of the pair transition at the training crop
        {"name": "linear_pair_384", "kind": "linear", "rows": 384 * 384, "inputs": 128, "outputs": 512,
         "dtype": "bf16", "relu": True, "residual": False},
        # a large generic product, where the matrix cores are the limit
        {"name": "linear_4096", "kind": "linear", "rows": 8192, "inputs": 4096, "outputs": 4096, "dtype": "bf16",
         "relu": False, "residual": False},
        # the backward pass of a pair projection at an ordinary length, full precision gradients
        {"name": "linear_grad_301", "kind": "linear_backward", "rows": 301 * 301, "inputs": 128, "outputs": 128,
         "dtype": "f32"},
        # the backward pass of the MSA transition's first product at full MSA depth
        {"name": "linear_grad_msa_384", "kind": "linear_backward", "rows": 512 * 384, "inputs": 256, "outputs": 1024,
         "dtype": "bf16"},
        # a training step of the pair transition at the training crop
        {"name": "transition_pair_384", "kind": "transition", "rows": 384 * 384, "c": 128, "hidden": 512,
         "dtype": "bf16", "residual": True},
        # a training step of the extra-MSA transition of a mid-size protein (203 residues, 1024 sequences), f16
        {"name": "transition_extra_203", "kind": "transition", "rows": 1024 * 203, "c": 64, "hidden": 256,
         "dtype": "f16", "residual": True},
    ]


def draw(rng):
    def log_int(lo, hi):
        hi = max(lo, hi)
        return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    def width(lo, hi):   # one of the trunk's, or any
        return rng.choice([rng.choice(WIDTHS), rng.choice(WIDTHS), log_int(lo, hi)])

    kind = rng.choice(["norm", "norm", "checkpoint", "linear", "linear", "linear_backward", "linear_backward",
                       "transition", "transition"])
    c = {"kind": kind, "dtype": rng.choice(["f32", "bf16", "bf16", "f16"])}
    if kind == "norm":
        c["direction"] = rng.choice(["forward", "backward"])
        c["c"] = width(22, 2048)
        c["rows"] = log_int(1, 512 * 384 * 256 // c["c"])
        c["fast_variance"] = rng.choice([False, True])
        c["kept"] = rng.choice([False, True])
    elif kind == "checkpoint":
        c["c"] = width(22, 2048)
        c["rows"] = log_int(1, 825 * 825 * 128 // c["c"])
    elif kind == "linear":
        c["inputs"], c["outputs"] = width(22, 4096), width(22, 4096)
        c["rows"] = log_int(1, min(512 * 384, 8192 * 4096 * 4096 // (c["inputs"] * c["outputs"]),
                                   512 * 384 * 512 // (c["inputs"] + c["outputs"])))
        c["relu"], c["residual"] = rng.choice([False, True]), rng.choice([False, True])
    elif kind == "linear_backward":
        c["inputs"], c["outputs"] = width(22, 1536), width(22, 1536)
        c["rows"] = log_int(1, min(512 * 384, 512 * 384 * 256 * 1024 // (c["inputs"] * c["outputs"]),
                                   512 * 384 * 1024 // (c["inputs"] + c["outputs"])))
    else:
        c["c"] = width(22, 384)
        c["hidden"] = rng.choice([4 * c["c"], 4 * c["c"], 2 * c["c"], log_int(22, 1536)])
        c["rows"] = log_int(16, min(1024 * 203, 384 * 384 * 128 * 512 // (c["c"] * c["hidden"]),
                                    384 * 384 * 640 // (c["c"] + c["hidden"])))
        c["residual"] = rng.choice([False, True])
    return c


# ---- what a user's program has in hand ---------------------------------------------------------

def _groups(n):
    return -(-n // GROUP)


def _pitch(cols):
    return -(-cols // 64) * 64


def _scale_byte(most):
    """b of the smallest 2^(b - 127) that is at least most / 448."""
    m, e = torch.frexp(most)
    b = e - 9 + (m > 0.875).to(e.dtype) + 127
    return torch.where(most > 0, b, torch.ones_like(b)).clamp(1, 254)


def _power(b):
    return torch.ldexp(torch.ones_like(b, dtype=torch.float32), b - 127)


def _encode(x):
    """Codes [rows, pitch] and scale bytes [groups, rows to 16] of finite float32 rows."""
    rows, cols = x.shape
    g = _groups(cols)
    p = torch.zeros(rows, g * GROUP, device=x.device)
    p[:, :cols] = x
    p = p.view(rows, g, GROUP)
    b = _scale_byte(p.abs().amax(-1))
    codes = (p / _power(b)[:, :, None]).view(rows, g * GROUP).to(torch.float8_e4m3fn).view(torch.uint8)
    scales = torch.full((g, -(-rows // 16) * 16), 127, dtype=torch.uint8, device=x.device)
    scales[:, :rows] = b.t().to(torch.uint8)
    return codes[:, :_pitch(cols)].contiguous(), scales


def _encode_weight(w):
    """Codes [out, pitch of in] and scale bytes [tiles of out, tiles of in] of a float32 weight."""
    n, k = w.shape
    gn, gk = _groups(n), _groups(k)
    p = torch.zeros(gn * GROUP, gk * GROUP, device=w.device)
    p[:n, :k] = w
    p = p.view(gn, GROUP, gk, GROUP)
    b = _scale_byte(p.abs().amax(3).amax(1))
    codes = (p / _power(b)[:, None, :, None]).view(gn * GROUP, gk * GROUP).to(torch.float8_e4m3fn).view(torch.uint8)
    return codes[:n, :_pitch(k)].contiguous(), b.to(torch.uint8)


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


def _vector(gen, n, spread, centre=0.0):
    return centre + spread * (2 * torch.rand(n, generator=gen, device=gen.device) - 1)


def _matrix(gen, a, b, fan_in):
    return torch.randn(a, b, generator=gen, device=gen.device) / math.sqrt(fan_in)


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
    kind, dt, rows = case["kind"], case["dtype"], case["rows"]
    s = {"case": dict(case)}
    if kind == "norm":
        c = case["c"]
        s["x"] = _activations(gen, rows, c, dt)
        s["scale"], s["offset"] = _vector(gen, c, 0.2, 1.0), _vector(gen, c, 0.1)
        if case["direction"] == "backward":
            s["grad"] = _gradient(gen, rows, c, dt)
            x = s["x"].double()   # the statistics that the forward pass kept
            var = x.var(-1, unbiased=False)
            s["stats"] = torch.stack([x.mean(-1), 1 / torch.sqrt(var + EPS)]).float()
            if case["kept"]:
                s["codes"], s["scales"] = _encode(s.pop("x").float())
    elif kind == "checkpoint":
        s["x"] = _activations(gen, rows, case["c"], dt)
    elif kind == "linear":
        k, n = case["inputs"], case["outputs"]
        s["x"] = _activations(gen, rows, k, dt)
        s["w_codes"], s["w_scales"] = _encode_weight(_matrix(gen, n, k, k))
        s["bias"] = _vector(gen, n, 0.1)
        if case["residual"]:
            s["residual"] = _activations(gen, rows, n, dt)
    elif kind == "linear_backward":
        k, n = case["inputs"], case["outputs"]
        s["grad"] = _gradient(gen, rows, n, dt)
        s["codes"], s["scales"] = _encode(_activations(gen, rows, k, dt).float())
        s["w_codes"], s["w_scales"] = _encode_weight(_matrix(gen, k, n, k))   # [in, out]: the backward's operand
    else:
        c, h = case["c"], case["hidden"]
        s["x"], s["grad"] = _activations(gen, rows, c, dt), _gradient(gen, rows, c, dt)
        s["w"] = {"layerNormScale": _vector(gen, c, 0.2, 1.0), "layerNormOffset": _vector(gen, c, 0.1),
                  "firstWeight": _matrix(gen, c, h, c), "firstBias": _vector(gen, h, 0.1),
                  "secondWeight": _matrix(gen, h, c, h), "secondBias": _vector(gen, c, 0.05)}
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if own:   # the handle, and the buffers that a program allocates once
        D, ctx = _context()
        kind, rows, dev = case["kind"], case["rows"], ctx.device
        act = DTYPES[case["dtype"]]
        s["D"], s["ctx"] = D, ctx

        def new(*shape, dtype=torch.float32):
            return torch.empty(shape, dtype=dtype, device=dev)

        if kind == "norm" and case["direction"] == "forward":
            s["stats"] = new(2, rows)
            if case["kept"]:
                s["x8"], s["y8"] = (D.checkpoint_empty(rows, case["c"], dev) for _ in range(2))
                s["x_back"], s["y_back"] = (new(rows, case["c"], dtype=torch.bfloat16) for _ in range(2))
            else:
                s["out"] = new(rows, case["c"], dtype=act)
        elif kind == "norm":
            s["out"], s["gs"], s["go"] = new(rows, case["c"], dtype=act), new(case["c"]), new(case["c"])
            if case["kept"]:
                s["x8"] = D.Checkpoint(rows, case["c"], s["codes"], s["scales"])
        elif kind == "checkpoint":
            s["x8"], s["out"] = D.checkpoint_empty(rows, case["c"], dev), new(rows, case["c"], dtype=act)
        elif kind == "linear":
            s["x8"] = D.checkpoint_empty(rows, case["inputs"], dev)
            s["w8"] = D.Fp8Weight(case["outputs"], case["inputs"], s["w_codes"], s["w_scales"])
            s["out"] = new(rows, case["outputs"], dtype=act)
        elif kind == "linear_backward":
            k, n = case["inputs"], case["outputs"]
            s["x8"] = D.Checkpoint(rows, k, s["codes"], s["scales"])
            s["g8"] = D.checkpoint_empty(rows, n, dev)
            s["w8"] = D.Fp8Weight(k, n, s["w_codes"], s["w_scales"])
            s["out"], s["dw"], s["db"] = new(rows, k, dtype=act), new(n, k), new(n)
        else:
            s["weights"] = D.transition_train_weights(s["w"])
            s["saved"] = D.transition_saved(rows, case["c"], case["hidden"], dev)
            s["out"], s["dx"] = new(rows, case["c"], dtype=act), new(rows, case["c"], dtype=act)
    return s


# ---- one pass ----------------------------------------------------------------------------------

def _run_own(s):
    case, D, ctx = s["case"], s["D"], s["ctx"]
    kind = case["kind"]
    if kind == "norm" and case["direction"] == "forward":
        if not case["kept"]:
            D.layer_norm(ctx, s["x"], s["scale"], s["offset"], epsilon=EPS, fast_variance=case["fast_variance"],
                         out=s["out"], stats=s["stats"])
            return {"y": s["out"], "stats": s["stats"]}
        D.layer_norm(ctx, s["x"], s["scale"], s["offset"], epsilon=EPS, fast_variance=case["fast_variance"],
                     stats=s["stats"], x_saved=s["x8"], y_saved=s["y8"])
        return {"x8": D.checkpoint_unpack(ctx, s["x8"], out=s["x_back"]),
                "y8": D.checkpoint_unpack(ctx, s["y8"], out=s["y_back"]), "stats": s["stats"]}
    if kind == "norm":
        D.layer_norm_backward(ctx, s["grad"], s["x8"] if case["kept"] else s["x"], s["scale"], s["stats"],
                              out=s["out"], grad_scale=s["gs"], grad_offset=s["go"])
        return {"dx": s["out"], "dscale": s["gs"], "doffset": s["go"]}
    if kind == "checkpoint":
        D.checkpoint_pack(ctx, s["x"], out=s["x8"])
        return D.checkpoint_unpack(ctx, s["x8"], out=s["out"])
    if kind == "linear":
        D.checkpoint_pack(ctx, s["x"], out=s["x8"])
        D.fp8_linear(ctx, s["x8"], s["w8"], s["bias"], relu=case["relu"], residual=s.get("residual"), out=s["out"])
        return s["out"]
    if kind == "linear_backward":
        D.checkpoint_pack(ctx, s["grad"], out=s["g8"])
        D.fp8_linear(ctx, s["g8"], s["w8"], out=s["out"])
        D.fp8_weight_grad(ctx, s["g8"], s["x8"], out=s["dw"], bias_out=s["db"])
        return {"dx": s["out"], "dw": s["dw"], "db": s["db"]}
    D.transition_train(ctx, s["x"], s["weights"], s["saved"], out=s["out"], accumulate=case["residual"], epsilon=EPS)
    dx, grads = D.transition_backward(ctx, s["grad"], s["weights"], s["saved"], out=s["dx"],
                                      accumulate=case["residual"], grad_dtype=torch.bfloat16)
    return {"out": s["out"], "dx": dx, "grads": grads}


def _decode(codes, scales, cols):
    rows = codes.shape[0]
    v = codes.view(torch.float8_e4m3fn).float()[:, :cols]
    f = _power(scales[:, :rows].t().to(torch.int32))
    return v * f.repeat_interleave(GROUP, 1)[:, :cols]


def _decode_weight(codes, scales, cols):
    v = codes.view(torch.float8_e4m3fn).float()[:, :cols]
    f = _power(scales.to(torch.int32))
    return v * f.repeat_interleave(GROUP, 0)[:v.shape[0]].repeat_interleave(GROUP, 1)[:, :cols]


def _kept(x):
    """float32 rows as they are after a round trip through 8 bits."""
    return _decode(*_encode(x), x.shape[1])


def _kept_weight(w):
    return _decode_weight(*_encode_weight(w), w.shape[1])


def _norm(x, scale, offset, fast_variance):
    mean = x.mean(-1, keepdim=True)
    var = (x * x).mean(-1, keepdim=True) - mean * mean if fast_variance else ((x - mean) ** 2).mean(-1, keepdim=True)
    r = torch.rsqrt(var + EPS)
    return (x - mean) * r * scale + offset, torch.stack([mean[:, 0], r[:, 0]])


def _norm_backward(grad, x, scale, stats):
    h = (x - stats[0][:, None]) * stats[1][:, None]
    g = grad * scale
    dx = stats[1][:, None] * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    return dx, (grad * h).sum(0), grad.sum(0)


def _run_plain(s):
    case = s["case"]
    kind, act = case["kind"], DTYPES[case["dtype"]]
    if kind == "norm" and case["direction"] == "forward":
        x = s["x"].float()
        y, stats = _norm(x, s["scale"], s["offset"], case["fast_variance"])
        if not case["kept"]:
            return {"y": y.to(act), "stats": stats}
        return {"x8": _kept(x).bfloat16(), "y8": _kept(y).bfloat16(), "stats": stats}
    if kind == "norm":
        x = _decode(s["codes"], s["scales"], case["c"]) if case["kept"] else s["x"].float()
        dx, gs, go = _norm_backward(s["grad"].float(), x, s["scale"], s["stats"])
        return {"dx": dx.to(act), "dscale": gs, "doffset": go}
    if kind == "checkpoint":
        return _kept(s["x"].float()).to(act)
    if kind == "linear":
        w = _decode_weight(s["w_codes"], s["w_scales"], case["inputs"])
        out = _kept(s["x"].float()) @ w.t() + s["bias"]
        if case["relu"]:
            out = out.clamp(min=0)
        if case["residual"]:
            out = out + s["residual"].float()
        return out.to(act)
    if kind == "linear_backward":
        g = _kept(s["grad"].float())
        x = _decode(s["codes"], s["scales"], case["inputs"])
        w = _decode_weight(s["w_codes"], s["w_scales"], case["outputs"])
        return {"dx": (g @ w.t()).to(act), "dw": g.t() @ x, "db": g.sum(0)}
    w, x, grad = s["w"], s["x"].float(), s["grad"].float()
    y, stats = _norm(x, w["layerNormScale"], w["layerNormOffset"], False)
    x8, y8 = _kept(x), _kept(y)
    w1, w2 = _kept_weight(w["firstWeight"]), _kept_weight(w["secondWeight"])
    h8 = _kept((y8 @ w1 + w["firstBias"]).clamp(min=0))
    out = h8 @ w2 + w["secondBias"]
    d8 = _kept(grad)
    e8 = _kept(torch.where(h8 > 0, d8 @ w2.t(), 0.0))
    dx, gs, go = _norm_backward(e8 @ w1.t(), x8, w["layerNormScale"], stats)
    if case["residual"]:
        out, dx = x + out, grad + dx
    grads = {"layerNormScale": gs, "layerNormOffset": go, "firstWeight": y8.t() @ e8, "firstBias": e8.sum(0),
             "secondWeight": h8.t() @ d8, "secondBias": d8.sum(0)}
    return {"out": out.to(act), "dx": dx.to(act), "grads": {k: v.bfloat16() for k, v in grads.items()}}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    kind, r, b = case["kind"], case["rows"], ACT_BYTES[case["dtype"]]

    def kept(c):
        return r * (c + _groups(c))

    if kind == "norm":
        c = case["c"]
        if case["direction"] == "forward":
            # kept: both checkpoints written, and read back to the values that they stand for
            out = 4 * kept(c) + 2 * r * c * 2 if case["kept"] else r * c * b
            return {"bytes": r * c * b + out + 8 * r + 8 * c, "flops": 8 * r * c}
        return {"bytes": 2 * r * c * b + (kept(c) if case["kept"] else r * c * b) + 8 * r + 12 * c,
                "flops": 14 * r * c}
    if kind == "checkpoint":
        return {"bytes": 2 * r * case["c"] * b + 2 * kept(case["c"]), "flops": 4 * r * case["c"]}
    if kind == "linear":
        k, n = case["inputs"], case["outputs"]
        return {"bytes": r * k * b + n * k + 4 * n + r * n * b * (2 if case["residual"] else 1),
                "flops": 2 * r * n * k}
    if kind == "linear_backward":
        k, n = case["inputs"], case["outputs"]
        return {"bytes": r * n * b + kept(k) + n * k + r * k * b + 4 * n * k + 4 * n, "flops": 4 * r * n * k}
    c, h = case["c"], case["hidden"]
    return {"bytes": 4 * r * c * b + 2 * (2 * kept(c) + kept(h)) + 16 * r + 2 * c * h * (4 + 2),
            "flops": 12 * r * c * h}


# ---- in float64, from the definitions -------------------------------------------------------------

def _binary_exponent(v):
    """floor(log2(v)) of positive doubles."""
    return torch.frexp(v)[1].double() - 1


def _e4m3(v):
    """Doubles rounded to e4m3 (3 mantissa bits, smallest normal 2^-6, ties to even)."""
    a = v.abs()
    e = torch.where(a > 0, _binary_exponent(a.clamp(min=1e-300)), torch.full_like(a, -6.0)).clamp(min=-6.0)
    step = torch.exp2(e - 3)
    return torch.round(v / step) * step


def _scale64(most):
    e = _binary_exponent(most.clamp(min=1e-300)) - 8
    e = torch.where(most > LARGEST * torch.exp2(e), e + 1, e)
    return torch.exp2(torch.where(most > 0, e, torch.full_like(e, -126.0)).clamp(-126, 127))


def _kept64(x):
    out = torch.empty_like(x)
    for g in range(0, x.shape[1], GROUP):
        part = x[:, g:g + GROUP]
        f = _scale64(part.abs().max(1, keepdim=True).values)
        out[:, g:g + GROUP] = _e4m3(part / f) * f
    return out


def _kept_weight64(w):
    out = torch.empty_like(w)
    for i in range(0, w.shape[0], GROUP):
        for j in range(0, w.shape[1], GROUP):
            part = w[i:i + GROUP, j:j + GROUP]
            f = _scale64(part.abs().max())
            out[i:i + GROUP, j:j + GROUP] = _e4m3(part / f) * f
    return out


def _values64(codes, bytes_of, cols):
    """What codes and the scale byte of each value, [rows, cols], stand for."""
    c = codes[:, :cols].to(torch.int64)
    sign, e, m = c >> 7, (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8 + m) * torch.exp2(e.double() - 10))
    return torch.where(sign == 1, -v, v) * torch.exp2(bytes_of.double() - 127)


def _activations64(codes, scales, cols):
    b = scales[:, :codes.shape[0]].t()
    return _values64(codes, b[:, torch.arange(cols, device=codes.device) // GROUP], cols)


def _weight64(codes, scales, cols):
    i = torch.arange(codes.shape[0], device=codes.device) // GROUP
    j = torch.arange(cols, device=codes.device) // GROUP
    return _values64(codes, scales[i][:, j], cols)


def _norm64(x, scale, offset):
    mean = x.sum(1, keepdim=True) / x.shape[1]
    d = x - mean
    r = 1 / torch.sqrt((d * d).sum(1, keepdim=True) / x.shape[1] + EPS)
    return d * r * scale.double() + offset.double(), torch.cat([mean, r], 1).t()


def _norm_backward64(grad, x, scale, stats):
    c = x.shape[1]
    r = stats[1].double()[:, None]
    h = (x - stats[0].double()[:, None]) * r
    g = grad * scale.double()
    dx = r * (g - g.sum(1, keepdim=True) / c - h * ((g * h).sum(1, keepdim=True) / c))
    return dx, (grad * h).sum(0), grad.sum(0)


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "norm" and case["direction"] == "forward":
        x = s["x"].double()
        y, stats = _norm64(x, s["scale"], s["offset"])
        if not case["kept"]:
            return {"y": y, "stats": stats}
        return {"x8": _kept64(x), "y8": _kept64(y), "stats": stats}
    if kind == "norm":
        x = _activations64(s["codes"], s["scales"], case["c"]) if case["kept"] else s["x"].double()
        dx, gs, go = _norm_backward64(s["grad"].double(), x, s["scale"], s["stats"])
        return {"dx": dx, "dscale": gs, "doffset": go}
    if kind == "checkpoint":
        return _kept64(s["x"].double())
    if kind == "linear":
        out = torch.matmul(_kept64(s["x"].double()), _weight64(s["w_codes"], s["w_scales"], case["inputs"]).t())
        out += s["bias"].double()
        if case["relu"]:
            out = torch.where(out < 0, torch.zeros_like(out), out)
        return out + s["residual"].double() if case["residual"] else out
    if kind == "linear_backward":
        g = _kept64(s["grad"].double())
        w = _weight64(s["w_codes"], s["w_scales"], case["outputs"])
        return {"dx": torch.matmul(g, w.t()),
                "dw": torch.matmul(g.t(), _activations64(s["codes"], s["scales"], case["inputs"])), "db": g.sum(0)}
    w = {k: v.double() for k, v in s["w"].items()}
    x, grad = s["x"].double(), s["grad"].double()
    y, stats = _norm64(x, w["layerNormScale"], w["layerNormOffset"])
    y8, d8 = _kept64(y), _kept64(grad)
    w1, w2 = _kept_weight64(w["firstWeight"]), _kept_weight64(w["secondWeight"])
    pre = torch.matmul(y8, w1) + w["firstBias"]
    h8 = _kept64(torch.where(pre > 0, pre, torch.zeros_like(pre)))
    out = torch.matmul(h8, w2) + w["secondBias"]
    e8 = _kept64(torch.matmul(d8, w2.t()) * (h8 > 0))
    dx, gs, go = _norm_backward64(torch.matmul(e8, w1.t()), _kept64(x), w["layerNormScale"], stats)
    if case["residual"]:
        out, dx = out + x, dx + grad
    return {"out": out, "dx": dx,
            "grads": {"layerNormScale": gs, "layerNormOffset": go, "firstWeight": torch.matmul(y8.t(), e8),
                      "firstBias": e8.sum(0), "secondWeight": torch.matmul(h8.t(), d8), "secondBias": d8.sum(0)}}
