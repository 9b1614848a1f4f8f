"""Training operators: LayerNorm and its gradient, activations kept in 8 bits, 8-bit products, weight
gradients and the transition's training step, against float64 restatements.

Tolerances.  U = 2^-24 is half a step of float32; a sum whose terms pass through at most D additions is
off by at most D * 2U times the sum of magnitudes (2U: an addition may cut instead of round).  A stored
value adds half a step of its type, relative to it.  The 8-bit matrix instruction drops, of 8 products
that it adds at a time, what lies 2^-13 below the largest: at most 8 * 2^-13 of the magnitudes' sum."""
import math

import numpy as np
import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


# ---- float64 restatements ------------------------------------------------------------------------

def e4m3_values():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c >= 128, -v, v)


VALUES = e4m3_values()


def round_e4m3(v):
    a = np.abs(v)
    e = np.maximum(np.floor(np.log2(np.where(a > 0, a, 1.0))), -6)
    step = 2.0 ** (e - 3)
    return np.round(v / step) * step      # half to even


def scale_of(most):
    """The smallest power of two, at least 2^-126, that puts `most` within 448."""
    m, e = np.frexp(most)
    return np.where(most > 0, 2.0 ** np.maximum(e - 9 + (m > 0.875), -126.0), 2.0 ** -126)


def kept64(x):
    """x after a round trip through 8 bits."""
    out = np.array(x, np.float64)
    for g in range(0, x.shape[1], 128):
        p = out[:, g:g + 128]
        f = scale_of(np.max(np.where(np.isfinite(p), np.abs(p), 0.0), axis=1, keepdims=True))
        with np.errstate(invalid="ignore"):
            out[:, g:g + 128] = np.where(np.isfinite(p), round_e4m3(np.where(np.isfinite(p), p, 0) / f) * f, np.nan)
    return out


def kept_weight64(w):
    out = np.array(w, np.float64)
    for i in range(0, w.shape[0], 128):
        for j in range(0, w.shape[1], 128):
            p = out[i:i + 128, j:j + 128]
            f = scale_of(np.max(np.abs(p)))
            out[i:i + 128, j:j + 128] = round_e4m3(p / f) * f
    return out


def values_of(kept):
    """What a Checkpoint's codes stand for, read here from its documented layout."""
    codes, scales = kept.codes.cpu().numpy(), kept.scales.cpu().numpy()
    f = 2.0 ** (scales[:, :kept.rows].T.astype(np.float64) - 127)
    return VALUES[codes[:, :kept.cols]] * np.repeat(f, 128, axis=1)[:, :kept.cols]


def weight_values(w):
    codes, scales = w.codes.cpu().numpy(), w.scales.cpu().numpy()
    f = np.repeat(np.repeat(2.0 ** (scales.astype(np.float64) - 127), 128, 0), 128, 1)
    return VALUES[codes[:, :w.inputs]] * f[:w.outputs, :w.inputs]


def norm64(x, s, o, eps, fast=False):
    m = x.mean(1, keepdims=True)
    v = (x * x).mean(1, keepdims=True) - m * m if fast else ((x - m) ** 2).mean(1, keepdims=True)
    r = 1 / np.sqrt(v + eps)
    return (x - m) * r * s + o, m, r


def norm_backward64(dy, x, s, m, r):
    h, g = (x - m) * r, dy * s
    dx = r * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    return dx, (dy * h).sum(0), dy.sum(0)


def test_norm_backward_formula_by_differences():
    rng = np.random.default_rng(0)
    x, dy, s, o = rng.normal(size=(3, 7)), rng.normal(size=(3, 7)), rng.normal(size=7), rng.normal(size=7)
    _, m, r = norm64(x, s, o, 1e-5)
    dx, ds, do = norm_backward64(dy, x, s, m, r)

    def loss(x, s, o):
        return (norm64(x, s, o, 1e-5)[0] * dy).sum()

    for a, d, f in ((x, dx, lambda t: loss(t, s, o)), (s, ds, lambda t: loss(x, t, o)), (o, do, lambda t: loss(x, s, t))):
        for i in np.ndindex(a.shape):
            e = np.zeros_like(a)
            e[i] = 1e-6
            assert abs((f(a + e) - f(a - e)) / 2e-6 - d[i]) < 1e-7


def test_checkpoint_layout_is_checked():
    from localfold_amd import device as D
    c = D.checkpoint_empty(17, 130, "cpu")
    assert c.codes.shape == (17, 192) and c.scales.shape == (2, 32)
    with pytest.raises(ValueError):
        D.Checkpoint(17, 130, c.codes[:, :130], c.scales)
    with pytest.raises(ValueError):
        D.Checkpoint(17, 130, c.codes, c.scales[:, :17].contiguous())
    with pytest.raises(ValueError):
        D.Fp8Weight(130, 70, torch.zeros(130, 128, dtype=torch.uint8), torch.zeros(2, 2, dtype=torch.uint8))


def test_dimensions_past_32_bits_are_refused():
    """They would arrive in C as other numbers."""
    from localfold_amd import device as D
    x = torch.empty((2 ** 32 + 5, 1), device="meta")
    with pytest.raises(ValueError, match="rows"):
        D._rows(x)
    codes, scales = (torch.empty(s, dtype=torch.uint8, device="meta") for s in ((2 ** 32 + 5, 64), (1, 2 ** 32 + 16)))
    with pytest.raises(ValueError, match="at most"):
        D.Checkpoint(2 ** 32 + 5, 1, codes, scales)
    with pytest.raises(ValueError, match="at most"):
        D.Fp8Weight(2 ** 32 + 5, 1, codes, scales)


def test_struct_layouts(tmp_path):
    """sizeof of the training structs in C and in Python."""
    import ctypes as C
    import os
    import subprocess
    from localfold_amd import capi
    names = [n for n in dir(capi) if n.startswith(("lf_checkpoint", "lf_layer_norm", "lf_fp8", "lf_transition_saved",
                                                   "lf_transition_train", "lf_transition_backward"))
             and isinstance(getattr(capi, n), type) and issubclass(getattr(capi, n), C.Structure)]
    assert len(names) >= 10
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "localfold.h"\nint main(void) {\n' + "".join(
        f'printf("{n} %zu\\n", sizeof({n}));\n' for n in names) + "return 0;}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "sizes")], check=True)
    for line in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines():
        n, size = line.split()
        assert C.sizeof(getattr(capi, n)) == int(size), n


def test_scratch_sizes_need_no_device():
    from localfold_amd import capi
    lib = capi.load()
    assert lib.lf_layer_norm_backward_scratch(5, 128) >= 2 * 128 * 4
    assert lib.lf_fp8_weight_grad_scratch(5, 30, 40) >= 30 * 40 * 4
    assert lib.lf_transition_backward_scratch(5, 64, 256) > lib.lf_transition_train_scratch(5, 64, 256) > 0
    assert lib.lf_fp8_weight_grad_scratch(0, 30, 40) == lib.lf_transition_train_scratch(5, -1, 4) == 0


def test_entry_points_refuse_null():
    import ctypes as C
    from localfold_amd import capi
    lib = capi.load()
    for name in ("lf_checkpoint_pack", "lf_layer_norm", "lf_layer_norm_backward", "lf_fp8_linear", "lf_transition_train"):
        fn = getattr(lib, name)
        assert fn(None, None) == capi.LF_ERR_INVALID and name.encode() in lib.lf_last_error()


# ---- on the GPU ----------------------------------------------------------------------------------

def rows_of(rng, rows, c, dt, spread=1.0):
    x = rng.normal(size=(rows, c)) * np.exp(spread * rng.normal(size=(rows, 1))) + 0.3 * rng.normal(size=c)
    return torch.as_tensor(x).to(dt)


def f64(t):
    return t.detach().cpu().double().numpy()


def vec(rng, ctx, n, spread, centre=0.0):
    return torch.as_tensor(centre + spread * rng.uniform(-1, 1, n)).float().to(ctx.device)


def close(got, want, slack, dt, label=""):
    """|got - want| within `slack` (before the store) and the store's half step."""
    got = f64(got) if isinstance(got, torch.Tensor) else got
    bound = slack + HALF[dt] * (np.abs(want) + slack) + TINY[dt]
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (label, int(bad.sum()), np.argwhere(bad)[:4].tolist(),
                           float(np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300))))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,c", [(1, 1), (1, 128), (3, 22), (17, 64), (50, 65), (33, 127), (129, 128), (64, 129),
                                    (7, 200), (20, 384), (5, 1000), (1000, 256), (2, 5000)])
def test_checkpoint_round_trip(ctx, dt, rows, c):
    from localfold_amd import device as D
    rng = np.random.default_rng(rows * 7 + c)
    x = rows_of(rng, rows, c, dt)
    x[rows // 2] = 0
    kept = D.checkpoint_pack(ctx, x.to(ctx.device))
    back = D.checkpoint_unpack(ctx, kept)
    torch.cuda.synchronize()
    want = kept64(f64(x))
    assert np.array_equal(values_of(kept), want)
    assert np.array_equal(f64(back), want)
    assert (kept.codes[:, c:] == 0).all()
    b16 = f64(D.checkpoint_unpack(ctx, kept, torch.bfloat16))
    assert np.array_equal(b16, want)


@pytest.mark.gpu
def test_checkpoint_special_values(ctx):
    """Scales at their ends, groups whose largest value sits on 448 and just above, halves between
    codes, infinities and NaN, float32 subnormals."""
    from localfold_amd import device as D
    x = np.zeros((13, 256), np.float32)
    x[0, :3] = [448, -447, 1]
    x[1, :3] = [np.nextafter(np.float32(448), np.float32(500)), 1, 2 ** -9]
    x[2, 0], x[2, 1] = np.float32(3.4e38), 1
    x[3, 0] = np.float32(1e-40)
    x[4, :4] = [np.inf, 2.5, -np.inf, np.nan]
    x[5, 200] = np.nan
    grid = np.concatenate([VALUES[:127], (VALUES[:126] + VALUES[1:127]) / 2]).astype(np.float32)
    x[6, :127], x[6, 127] = grid[:127], 448
    x[7, :126], x[7, 127] = grid[127:], 448
    x[8] = -x[6]
    x[9] = -x[7]
    x[10, 128:] = 2.0 ** -126
    x[11, :] = np.finfo(np.float32).tiny * np.linspace(-3, 3, 256)
    x[12] = np.inf
    kept = D.checkpoint_pack(ctx, torch.as_tensor(x).to(ctx.device))
    back = D.checkpoint_unpack(ctx, kept)
    torch.cuda.synchronize()
    want = kept64(x.astype(np.float64))
    assert np.array_equal(values_of(kept), want, equal_nan=True)
    # 3.4e38 lies above 15.5 / 16 of 2^128, so its code stands for 2^128, which float32 stores as infinity
    assert want[2, 0] == 2.0 ** 128
    with np.errstate(over="ignore"):
        assert np.array_equal(back.cpu().numpy(), want.astype(np.float32), equal_nan=True)


@pytest.mark.gpu
def test_checkpoint_leaves_the_neighbours(ctx):
    """Rows behind the last and codes behind the buffer stay as they were."""
    from localfold_amd import device as D
    big = torch.full((40, 192), 77, dtype=torch.uint8, device=ctx.device)
    scales = torch.full((2, 32), 78, dtype=torch.uint8, device=ctx.device)
    x = torch.randn(19, 130, device=ctx.device)
    D.checkpoint_pack(ctx, x, out=D.Checkpoint(19, 130, big[:19], scales))
    torch.cuda.synchronize()
    assert (big[19:] == 77).all() and (scales[:, 19:] == 78).all() and (scales[:, :19] != 78).any()


def norm_slack(x, s, o, m, r, c, kept=False):
    # sums over c values pass through at most c / 8 + 16 additions whatever the team, never over 64
    depth = min(c, 64) + 8
    size = np.abs(x).mean(1, keepdims=True) + np.abs(x)
    # the variance's relative error, halved by the root, times |h|; m's error times r; each product's rounding
    rel = 2 * depth * U * (1 + r * r * (x * x).mean(1, keepdims=True))
    return (np.abs((x - m) * r) * rel + depth * 2 * U * size * r) * np.abs(s) + 4 * U * (np.abs((x - m) * r * s) + np.abs(o))


NORM_SHAPES = [(1, 1), (1, 128), (59, 384), (5, 22), (33, 49), (40, 64), (100, 65), (300, 128), (17, 129), (70, 256),
               (9, 385), (6, 513), (11, 1024), (3, 1025), (5, 1536), (4, 2048), (2, 2049), (3, 4095), (2, 4096)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,c", NORM_SHAPES)
def test_layer_norm(ctx, dt, rows, c):
    from localfold_amd import device as D
    rng = np.random.default_rng(rows + 31 * c)
    for fast in (False, True):
        x, s, o = rows_of(rng, rows, c, dt, 0.3), vec(rng, ctx, c, 0.3, 1.0), vec(rng, ctx, c, 0.2)
        xd = x.to(ctx.device)
        stats = torch.empty(2, rows, device=ctx.device)
        xs, ys = D.checkpoint_empty(rows, c, ctx.device), D.checkpoint_empty(rows, c, ctx.device)
        out = D.layer_norm(ctx, xd, s, o, fast_variance=fast, out=torch.empty_like(xd), stats=stats, x_saved=xs, y_saved=ys)
        alone = D.layer_norm(ctx, xd, s, o, fast_variance=fast)
        torch.cuda.synchronize()
        x64, s64, o64 = f64(x), f64(s), f64(o)
        y, m, r = norm64(x64, s64, o64, float(np.float32(1e-5)), fast)
        slack = norm_slack(x64, s64, o64, m, r, c)
        if c == 1 and fast:     # the variance's true value is zero: its rounding decides; y - o = 0 all the same
            slack = slack + 1e-6
        close(out, y, slack, dt, f"y {fast}")
        assert torch.equal(out, alone)
        assert np.array_equal(values_of(xs), kept64(x64))
        # y kept: y's own slack, then half a step of the code (2^-4, or 2^-10 of the scale below 2^-6 of it)
        f = np.repeat(scale_of(np.stack([np.abs(y[:, g:g + 128]).max(1) * (1 + 1e-5) for g in range(0, c, 128)], 1)), 128, 1)[:, :c]
        assert (np.abs(values_of(ys) - y) <= slack + (np.abs(y) + slack) * 2.0 ** -4 + f * 2.0 ** -10).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,c", NORM_SHAPES + [(5000, 128), (2100, 384)])
def test_layer_norm_backward(ctx, dt, rows, c):
    from localfold_amd import device as D
    rng = np.random.default_rng(rows + 17 * c)
    x, dy, s = rows_of(rng, rows, c, dt, 0.3), rows_of(rng, rows, c, dt, 1.0), vec(rng, ctx, c, 0.3, 1.0)
    if rows > 2:
        dy[rows // 2] = 0      # a padded row
    res = rows_of(rng, rows, c, dt)
    kept = D.checkpoint_pack(ctx, x.to(ctx.device))
    _, m, r = norm64(f64(x), 1.0, 0.0, 1e-5)
    stats = torch.as_tensor(np.concatenate([m, r], 1).T.copy()).float().to(ctx.device)
    m32, r32 = f64(stats)[0][:, None], f64(stats)[1][:, None]
    for xin, x64, residual in ((x.to(ctx.device), f64(x), None), (kept, values_of(kept), res.to(ctx.device))):
        out, gs, go = D.layer_norm_backward(ctx, dy.to(ctx.device), xin, s, stats, residual=residual)
        torch.cuda.synchronize()
        d64, s64 = f64(dy), f64(s)
        dx, ds, do = norm_backward64(d64, x64, s64, m32, r32)
        h, g = (x64 - m32) * r32, d64 * s64
        dh = 2 * U * (np.abs(x64) + np.abs(m32)) * r32        # h's own error
        depth = min(c, 64) + 8
        b = np.abs(g * h).mean(1, keepdims=True)
        slack = r32 * (4 * U * np.abs(g) + depth * 2 * U * np.abs(g).mean(1, keepdims=True)
                       + np.abs(h) * (depth * 2 * U * b + (np.abs(g) * dh).mean(1, keepdims=True)) + dh * b)
        slack = slack + 4 * U * np.abs(dx)
        if residual is not None:
            dx = dx + f64(res)
            slack = slack + 2 * U * np.abs(dx)
        close(out, dx, slack, dt, "dx")
        # rows of one block, a block's teams, the blocks
        depth = 32 + 16 + 80
        close(gs, ds, depth * 2 * U * np.abs(d64 * h).sum(0) + (np.abs(d64) * dh).sum(0), torch.float32, "dscale")
        close(go, do, depth * 2 * U * np.abs(d64).sum(0), torch.float32, "doffset")


@pytest.mark.gpu
def test_layer_norm_backward_in_place_types_and_repeats(ctx):
    """The gradient written over grad and over the residual, 16-bit parameter gradients, the parts
    alone, and the same bits from the same call."""
    from localfold_amd import device as D
    rng = np.random.default_rng(5)
    rows, c = 777, 128
    x, dy, s = (t.to(ctx.device) for t in (rows_of(rng, rows, c, torch.bfloat16), rows_of(rng, rows, c, torch.bfloat16),
                                           vec(rng, ctx, c, 0.3, 1.0)))
    stats = torch.empty(2, rows, device=ctx.device)
    D.layer_norm(ctx, x, s, s, stats=stats)
    want, gs, go = D.layer_norm_backward(ctx, dy, x, s, stats, residual=x)
    g2 = dy.clone()
    _, hs, ho = D.layer_norm_backward(ctx, g2, x, s, stats, residual=x, out=g2, grad_dtype=torch.bfloat16)
    x2 = x.clone()
    D.layer_norm_backward(ctx, dy, x, s, stats, residual=x2, out=x2)
    for _ in range(3):
        again = D.layer_norm_backward(ctx, dy, x, s, stats, residual=x)
        assert all(torch.equal(p, q) for p, q in zip(again, (want, gs, go)))
    torch.cuda.synchronize()
    assert torch.equal(g2, want) and torch.equal(x2, want)
    assert torch.equal(hs, gs.bfloat16()) and torch.equal(ho, go.bfloat16())
    y = x.clone()
    D.layer_norm(ctx, y, s, s, out=y)
    assert torch.equal(y, D.layer_norm(ctx, x, s, s))


@pytest.mark.gpu
def test_layer_norm_extreme_rows(ctx):
    """Constant rows, rows far from zero, rows with an infinity or a NaN beside ordinary ones."""
    from localfold_amd import device as D
    rng = np.random.default_rng(6)
    x = rng.normal(size=(8, 128))
    x[0], x[1] = 5.0, x[1] + 1000
    x[2, 7], x[3, 9], x[4] = np.inf, np.nan, x[4] * 1e-20
    xt = torch.as_tensor(x).float()
    one, zero = torch.ones(128, device=ctx.device), torch.zeros(128, device=ctx.device)
    ys = D.checkpoint_empty(8, 128, ctx.device)
    out = D.layer_norm(ctx, xt.to(ctx.device), one, zero, out=torch.empty(8, 128, device=ctx.device), y_saved=ys)
    torch.cuda.synchronize()
    got, x64 = f64(out), f64(xt)
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all() and np.isnan(values_of(ys)[2:4]).all()
    for i in (0, 1, 4, 5, 6, 7):
        y, m, r = norm64(x64[i:i + 1], 1.0, 0.0, float(np.float32(1e-5)))
        close(got[i:i + 1], y, norm_slack(x64[i:i + 1], np.ones(128), np.zeros(128), m, r, 128), torch.float32, str(i))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("a,b", [(1, 1), (64, 256), (128, 128), (130, 70), (300, 513), (384, 22)])
def test_weight_pack(ctx, dt, a, b):
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(a + b)
    w = torch.as_tensor(rng.normal(size=(a, b)) * np.exp(rng.normal(size=(a, 1)))).to(dt)
    wd = w.to(ctx.device)
    plain, turned = kept_weight64(f64(w)), kept_weight64(f64(w)).T
    for layout, backward, want in ((capi.LF_OUT_IN, False, plain), (capi.LF_IN_OUT, False, turned),
                                   (capi.LF_OUT_IN, True, turned), (capi.LF_IN_OUT, True, plain)):
        p = D.fp8_weight(ctx, wd, layout, backward)
        torch.cuda.synchronize()
        assert (p.outputs, p.inputs) == want.shape
        assert np.array_equal(weight_values(p), want)
        assert (p.codes[:, p.inputs:] == 0).all()


LINEAR_SHAPES = [(1, 1, 1), (1, 128, 128), (3, 22, 49), (16, 64, 64), (59, 384, 1536), (77, 100, 130), (130, 129, 257),
                 (257, 128, 512), (300, 192, 100), (65, 640, 64), (513, 256, 256), (260, 1000, 300), (40, 65, 384),
                 (1030, 64, 128), (700, 512, 768)]


def linear_slack(xv, wv, k, exact):
    size = np.abs(xv) @ np.abs(wv).T
    depth = 32 + k / 32 + 4
    return size * (depth * 2 * U + (0 if exact else 2.0 ** -10))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES)
def test_linear(ctx, dt, rows, k, n):
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(rows + k + n)
    x8 = D.checkpoint_pack(ctx, rows_of(rng, rows, k, torch.float32, 2.0).to(ctx.device))
    w8 = D.fp8_weight(ctx, torch.as_tensor(rng.normal(size=(n, k)) / math.sqrt(k)).float().to(ctx.device), capi.LF_OUT_IN)
    bias, res = vec(rng, ctx, n, 1.0), rows_of(rng, rows, n, dt).to(ctx.device)
    xv, wv = values_of(x8), weight_values(w8)
    plain = xv @ wv.T
    slack = linear_slack(xv, wv, k, dt == torch.float32)
    close(D.fp8_linear(ctx, x8, w8, dtype=dt), plain, slack, dt, "plain")
    with_bias = plain + f64(bias)
    slack = slack + 2 * U * np.abs(with_bias)
    close(D.fp8_linear(ctx, x8, w8, bias, relu=True, dtype=dt), np.maximum(with_bias, 0), slack, dt, "relu")
    mask = D.checkpoint_pack(ctx, rows_of(rng, rows, n, torch.float32).to(ctx.device))
    gated = np.where(values_of(mask) > 0, plain, 0)
    close(D.fp8_linear(ctx, x8, w8, relu_of=mask, dtype=dt), gated, np.where(values_of(mask) > 0, slack, 0), dt, "gate")
    total = with_bias + f64(res)
    want_slack = slack + 2 * U * np.abs(total)
    close(D.fp8_linear(ctx, x8, w8, bias, residual=res, out=torch.empty_like(res)), total, want_slack, dt, "residual")
    close(D.fp8_linear(ctx, x8, w8, bias, residual=res, out=res), total, want_slack, dt, "in place")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES)
def test_linear_kept(ctx, rows, k, n):
    """A product kept in 8 bits: within half a code of the float64 product, scales as documented, zero
    codes in the padding and nothing behind the last row."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(rows + 3 * k + n)
    x8 = D.checkpoint_pack(ctx, rows_of(rng, rows, k, torch.float32).to(ctx.device))
    w8 = D.fp8_weight(ctx, torch.as_tensor(rng.normal(size=(n, k)) / math.sqrt(k)).float().to(ctx.device), capi.LF_OUT_IN)
    bias = vec(rng, ctx, n, 1.0)
    codes = torch.full((rows + 3, -(-n // 64) * 64), 9, dtype=torch.uint8, device=ctx.device)
    scales = torch.full((-(-n // 128), -(-rows // 16) * 16), 9, dtype=torch.uint8, device=ctx.device)
    out = D.Checkpoint(rows, n, codes[:rows], scales)
    D.fp8_linear(ctx, x8, w8, bias, relu=True, out=out)
    torch.cuda.synchronize()
    xv, wv = values_of(x8), weight_values(w8)
    want = np.maximum(xv @ wv.T + f64(bias), 0)
    slack = linear_slack(xv, wv, k, False) + 2 * U * np.abs(want)
    got = values_of(out)
    top = np.stack([(want + slack)[:, g:g + 128].max(1) for g in range(0, n, 128)], 1)
    low = np.stack([np.maximum(want - slack, 0)[:, g:g + 128].max(1) for g in range(0, n, 128)], 1)
    f = 2.0 ** (scales.cpu().numpy()[:, :rows].T.astype(np.float64) - 127)
    assert (f <= scale_of(top)).all() and (f >= scale_of(low)).all()
    wide = np.repeat(scale_of(top), 128, 1)[:, :n]
    assert (np.abs(got - want) <= slack + (want + slack) * 2.0 ** -4 + wide * 2.0 ** -10).all()
    assert (codes[:rows, n:] == 0).all() and (codes[rows:] == 9).all() and (scales[:, rows:] == 9).all()


@pytest.mark.gpu
def test_linear_specials(ctx):
    """A NaN in a row stays in that row, in a weight's row in that column; ReLU keeps it; rows of very
    different size do not disturb each other."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(3)
    x = rng.normal(size=(300, 256)) * 10.0 ** rng.integers(-12, 12, size=(300, 1))
    x[5, 200] = np.nan
    w = rng.normal(size=(200, 256)) / 16
    w8 = D.fp8_weight(ctx, torch.as_tensor(w).float().to(ctx.device), capi.LF_OUT_IN)
    x8 = D.checkpoint_pack(ctx, torch.as_tensor(x).float().to(ctx.device))
    for dt in (torch.float32, torch.bfloat16):
        out = f64(D.fp8_linear(ctx, x8, w8, relu=True, dtype=dt))
        assert np.isnan(out[5]).all()
        xv, wv = values_of(x8), weight_values(w8)
        xv[5] = 0
        out[5] = 0
        close(out, np.maximum(xv @ wv.T, 0), linear_slack(xv, wv, 256, dt == torch.float32), dt)
    kept = D.checkpoint_empty(300, 200, ctx.device)
    D.fp8_linear(ctx, x8, w8, out=kept)
    v = values_of(kept)
    assert np.isnan(v[5]).all() and np.isfinite(v[:5]).all() and np.isfinite(v[6:]).all()


# Reductions too long for resident weights: steps of whole groups, half a group at the end, tails of rows
# and outputs on both sides of a 256 x 256 tile.
LONG_SHAPES = [(1, 1153, 1), (3, 1216, 130), (257, 1280, 257), (300, 2112, 384), (59, 4096, 64), (1025, 1408, 500),
               (2100, 1500, 129)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,n", LONG_SHAPES)
def test_linear_long(ctx, dt, rows, k, n):
    test_linear(ctx, dt, rows, k, n)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", LONG_SHAPES)
def test_linear_long_kept(ctx, rows, k, n):
    test_linear_kept(ctx, rows, k, n)


@pytest.mark.gpu
def test_linear_long_specials(ctx):
    """NaN stays in its row and its column, and garbage scales behind the last row change nothing."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(4)
    x = rng.normal(size=(270, 1344)) * 10.0 ** rng.integers(-12, 12, size=(270, 1))
    x[5, 1340] = np.nan
    w8 = D.fp8_weight(ctx, torch.as_tensor(rng.normal(size=(200, 1344)) / 36).float().to(ctx.device), capi.LF_OUT_IN)
    x8 = D.checkpoint_pack(ctx, torch.as_tensor(x).float().to(ctx.device))
    x8.scales[:, 270:] = 255
    for dt in (torch.float32, torch.bfloat16):
        out = f64(D.fp8_linear(ctx, x8, w8, relu=True, dtype=dt))
        assert np.isnan(out[5]).all()
        xv, wv = values_of(x8), weight_values(w8)
        xv[5] = 0
        out[5] = 0
        close(out, np.maximum(xv @ wv.T, 0), linear_slack(xv, wv, 1344, dt == torch.float32), dt)


# Products large enough for the kernels that stage weights, resident and streamed.
MANY_SHAPES = [(20000, 64, 100), (9000, 128, 257), (6001, 192, 300), (3100, 1000, 512), (49001, 22, 17), (4000, 384, 513),
               (12300, 128, 128), (25000, 1153, 130), (8200, 1216, 400), (5000, 2112, 650)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,n", MANY_SHAPES)
def test_linear_many(ctx, dt, rows, k, n):
    test_linear(ctx, dt, rows, k, n)


GRAD_SHAPES = [(1, 1, 1), (1, 128, 128), (15, 22, 49), (64, 64, 64), (100, 130, 70), (333, 128, 512), (1000, 384, 129),
               (257, 512, 256), (4100, 256, 64), (70000, 64, 128), (37, 1536, 384)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", GRAD_SHAPES)
def test_weight_grad(ctx, rows, n, k):
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(rows + n + k)
    g8 = D.checkpoint_pack(ctx, rows_of(rng, rows, n, torch.float32).to(ctx.device))
    x8 = D.checkpoint_pack(ctx, rows_of(rng, rows, k, torch.float32).to(ctx.device))
    gv, xv = values_of(g8), values_of(x8)
    want, size = gv.T @ xv, np.abs(gv).T @ np.abs(xv)
    # 32 products an instruction, at most 1024 instructions a split, at most 1024 splits joined in runs
    depth = 32 + min(rows / 32, 1024) + min(rows / 32, 80)
    for layout, dt in ((capi.LF_OUT_IN, torch.float32), (capi.LF_IN_OUT, torch.float32), (capi.LF_IN_OUT, torch.bfloat16)):
        bias = torch.empty(n, dtype=dt, device=ctx.device)
        out = D.fp8_weight_grad(ctx, g8, x8, layout, bias_out=bias, grad_dtype=dt)
        alone = D.fp8_weight_grad(ctx, g8, x8, layout, grad_dtype=dt)
        torch.cuda.synchronize()
        turn = (lambda t: t) if layout == capi.LF_OUT_IN else np.transpose
        close(out, turn(want), depth * 2 * U * turn(size), dt, f"dw {layout} {dt}")
        close(bias, gv.sum(0), depth * 2 * U * np.abs(gv).sum(0), dt, "db")
        assert torch.equal(out, alone)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(300, 1536, 1500), (1000, 2100, 260), (40, 3000, 2000), (3000, 700, 700)])
def test_weight_grad_many_tiles(ctx, rows, n, k):
    test_weight_grad(ctx, rows, n, k)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 64, 50001), (32, 200, 49000), (1, 1300, 65536)])
def test_linear_one_tile_of_rows(ctx, rows, k, n):
    test_linear(ctx, torch.bfloat16, rows, k, n)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(5, 130, 70), (97, 64, 128), (1001, 200, 40), (16500, 128, 256)])
def test_weight_grad_garbage_behind_the_rows(ctx, rows, n, k):
    """Scales behind the last row may hold anything, and a NaN stays in its own output."""
    from localfold_amd import device as D
    rng = np.random.default_rng(rows)
    g, x = rng.normal(size=(rows, n)), rng.normal(size=(rows, k)) * 10.0 ** rng.integers(-6, 6, size=(rows, 1))
    g[rows - 1, n - 1] = np.nan
    g8, x8 = (D.checkpoint_pack(ctx, torch.as_tensor(t).float().to(ctx.device)) for t in (g, x))
    for t in (g8, x8):
        t.scales[:, rows:] = 255
    bias = torch.empty(n, device=ctx.device)
    out = f64(D.fp8_weight_grad(ctx, g8, x8, bias_out=bias))
    db = f64(bias)
    gv, xv = values_of(g8), values_of(x8)
    assert np.isnan(out[n - 1]).all() and np.isnan(db[n - 1])
    depth = 32 + min(rows / 32, 1024) + min(rows / 32, 80)
    close(out[:n - 1], (gv.T @ xv)[:n - 1], depth * 2 * U * (np.abs(gv).T @ np.abs(xv))[:n - 1], torch.float32, "dw")
    close(db[:n - 1], gv.sum(0)[:n - 1], depth * 2 * U * np.abs(gv).sum(0)[:n - 1], torch.float32, "db")


def transition_case(ctx, rng, c, h, dt, bias=True):
    w = {"layerNormScale": vec(rng, ctx, c, 0.2, 1.0), "layerNormOffset": vec(rng, ctx, c, 0.1),
         "firstWeight": torch.as_tensor(rng.normal(size=(c, h)) / math.sqrt(c)).to(dt).to(ctx.device),
         "secondWeight": torch.as_tensor(rng.normal(size=(h, c)) / math.sqrt(h)).to(dt).to(ctx.device)}
    if bias:
        w["firstBias"], w["secondBias"] = vec(rng, ctx, h, 0.1), vec(rng, ctx, c, 0.1)
    return w


def transition_step(ctx, rows, c, h, dt, wdt, residual, fast, shift=0):
    """The training step stage by stage: each stage's float64 form from what the stage before it kept,
    so that a code that falls the other way is no difference."""
    from localfold_amd import device as D
    rng = np.random.default_rng(rows + c)
    w = transition_case(ctx, rng, c, h, wdt, bias=rows != 45)
    ws, saved = D.transition_train_weights(w), D.transition_saved(rows, c, h, ctx.device)
    x, grad = rows_of(rng, rows, c, dt, 0.3).to(ctx.device), (rows_of(rng, rows, c, dt) * 0.01).to(dt).to(ctx.device)
    out, dx = torch.empty_like(x), torch.empty_like(grad)
    if shift:       # everything that many elements behind an aligned address
        x, grad, out, dx = (torch.cat([t.new_zeros(shift), t.flatten()])[shift:].view(rows, c) for t in (x, grad, out, dx))
    D.transition_train(ctx, x, ws, saved, out=out, accumulate=residual, fast_variance=fast)
    _, grads = D.transition_backward(ctx, grad, ws, saved, out=dx, accumulate=residual)
    torch.cuda.synchronize()
    x64, g64 = f64(x), f64(grad)
    zero = {"firstBias": np.zeros(h), "secondBias": np.zeros(c)}
    p = {k: f64(w[k]) if k in w else zero[k] for k in ("layerNormScale", "layerNormOffset", "firstWeight", "firstBias",
                                                       "secondWeight", "secondBias")}
    w1, w2 = kept_weight64(p["firstWeight"]), kept_weight64(p["secondWeight"])
    y, m, r = norm64(x64, p["layerNormScale"], p["layerNormOffset"], float(np.float32(1e-5)), fast)
    assert np.array_equal(values_of(saved.act), kept64(x64))
    y8, h8 = values_of(saved.normed), values_of(saved.hidden)
    code = 2.0 ** -4 + 2.0 ** -9      # half a code, and what moves a value to the next one
    low = 2.0 ** -10 * 2.0 ** -7      # half the smallest code, relative to the group's largest value
    top = np.abs(y).max(1, keepdims=True)
    assert (np.abs(y8 - y) <= np.abs(y) * code + top * low).all()
    pre = np.maximum(y8 @ w1 + p["firstBias"], 0)
    top = np.maximum(pre.max(1, keepdims=True), 1e-30)
    assert (np.abs(h8 - pre) <= pre * code + top * low + 2.0 ** -10 * (np.abs(y8) @ np.abs(w1))).all()
    upd = h8 @ w2 + p["secondBias"]
    total = upd + x64 if residual else upd
    close(out, total, (np.abs(h8) @ np.abs(w2)) * (2.0 ** -10 + 2 * U * 80) + 4 * U * (np.abs(total) + np.abs(x64)), dt, "out")

    d8 = kept64(g64)
    size = np.abs(h8).T @ np.abs(d8)
    close(grads["secondWeight"], h8.T @ d8, 200 * 2 * U * size, torch.float32, "dw2")
    pre_e = np.where(h8 > 0, d8 @ w2.T, 0)
    slack_e = np.where(h8 > 0, np.abs(pre_e) * code + np.abs(pre_e).max(1, keepdims=True) * low
                       + 2.0 ** -10 * (np.abs(d8) @ np.abs(w2.T)), 0)
    close(grads["firstWeight"], y8.T @ pre_e, np.abs(y8).T @ slack_e + 1e-6 * (np.abs(y8).T @ np.abs(pre_e)), torch.float32, "dw1")
    if "firstBias" in w:
        close(grads["firstBias"], pre_e.sum(0), slack_e.sum(0) + 1e-6 * np.abs(pre_e).sum(0), torch.float32, "db1")
        close(grads["secondBias"], d8.sum(0), 200 * 2 * U * np.abs(d8).sum(0), torch.float32, "db2")
    dy = pre_e @ w1.T
    slack_y = slack_e @ np.abs(w1.T) + (np.abs(pre_e) @ np.abs(w1.T)) * 2.0 ** -9 + np.abs(dy) * HALF[dt] + TINY[dt]
    st = f64(saved.stats)
    x8, s = values_of(saved.act), p["layerNormScale"]
    m32, r32 = st[0][:, None], st[1][:, None]
    want, ds, do = norm_backward64(dy, x8, s, m32, r32)
    hh, gs = (x8 - m32) * r32, slack_y * np.abs(s)
    slack = r32 * (gs + gs.mean(1, keepdims=True) + np.abs(hh) * (gs * np.abs(hh)).mean(1, keepdims=True)) + 1e-5 * np.abs(want)
    if residual:
        want = want + g64
    close(dx, want, slack + 1e-5 * np.abs(want), dt, "dx")
    close(grads["layerNormScale"], ds, (slack_y * np.abs(hh)).sum(0) + 1e-5 * np.abs(dy * hh).sum(0), torch.float32, "ds")
    close(grads["layerNormOffset"], do, slack_y.sum(0) + 1e-5 * np.abs(dy).sum(0), torch.float32, "do")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,h,dt,wdt,residual,fast", [
    (1, 128, 512, torch.float32, torch.float32, True, False), (37, 64, 256, torch.float16, torch.float32, True, True),
    (300, 128, 512, torch.bfloat16, torch.bfloat16, True, False), (150, 256, 1024, torch.float32, torch.float16, False, False),
    (90, 384, 100, torch.bfloat16, torch.float32, False, True), (45, 22, 70, torch.float32, torch.float32, True, False),
    (600, 49, 130, torch.float16, torch.bfloat16, False, False)])
def test_transition_step(ctx, rows, c, h, dt, wdt, residual, fast):
    transition_step(ctx, rows, c, h, dt, wdt, residual, fast)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,h,dt,wdt,residual,fast", [
    (33, 64, 128, torch.bfloat16, torch.float32, True, False), (31, 128, 128, torch.float16, torch.float16, False, True),
    (257, 64, 512, torch.float32, torch.float32, False, False), (1000, 128, 384, torch.float32, torch.bfloat16, True, True),
    (66001, 64, 128, torch.bfloat16, torch.float32, True, False)])
def test_transition_step_fused(ctx, rows, c, h, dt, wdt, residual, fast):
    """Widths that run as one kernel a direction: tails, more tiles of rows than waves."""
    transition_step(ctx, rows, c, h, dt, wdt, residual, fast)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,h,dt,shift", [(70, 128, 256, torch.bfloat16, 1), (70, 64, 128, torch.float16, 4),
                                               (70, 128, 128, torch.float32, 1), (131, 64, 640, torch.bfloat16, 0)])
def test_transition_step_composed(ctx, rows, c, h, dt, shift):
    """The same widths where the fused kernels do not apply: activations off a 16-byte address, wide hidden layers."""
    transition_step(ctx, rows, c, h, dt, torch.float32, True, False, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,h,dt", [(8100, 384, 1200, torch.bfloat16), (6200, 256, 512, torch.float16)])
def test_transition_step_many(ctx, rows, c, h, dt):
    """Composed, with products large enough for the kernels that stage weights, streamed and resident."""
    transition_step(ctx, rows, c, h, dt, torch.float32, True, False)


@pytest.mark.gpu
def test_transition_gradients_by_differences(ctx):
    """The step's gradients against differences of its own float32 forward pass along random
    directions.  The codes' roundings (2^-4 each, unbiased, over rows x hidden of them) leave a few
    percent; a wrong factor, sign or missing term is far outside."""
    from localfold_amd import device as D
    rng = np.random.default_rng(11)
    rows, c, h = 2048, 128, 512
    w = transition_case(ctx, rng, c, h, torch.float32)
    x, grad = (torch.as_tensor(rng.normal(size=(rows, c))).float().to(ctx.device) for _ in range(2))
    saved = D.transition_saved(rows, c, h, ctx.device)
    ws = D.transition_train_weights(w)
    D.transition_train(ctx, x, ws, saved, accumulate=True)
    dx, grads = D.transition_backward(ctx, grad, ws, saved, accumulate=True)
    torch.cuda.synchronize()

    def loss(x, w):
        y, _, _ = norm64(f64(x), f64(w["layerNormScale"]), f64(w["layerNormOffset"]), 1e-5)
        hid = np.maximum(y @ f64(w["firstWeight"]) + f64(w["firstBias"]), 0)
        return ((f64(x) + hid @ f64(w["secondWeight"]) + f64(w["secondBias"])) * f64(grad)).sum()

    # along the gradient itself: the difference is its squared length
    for name, t, g in [("x", x, dx)] + [(k, w[k], grads[k]) for k in grads]:
        d = g.double()
        length = float((d * d).sum())
        eps = 1e-3 * float(t.double().norm()) / max(float(d.norm()), 1e-30)
        up, down = (t.double() + eps * d).to(t.dtype), (t.double() - eps * d).to(t.dtype)
        if name == "x":
            got = (loss(up, w) - loss(down, w)) / (2 * eps)
        else:
            got = (loss(x, {**w, name: up}) - loss(x, {**w, name: down})) / (2 * eps)
        assert abs(got - length) < 0.1 * length, (name, got, length)


@pytest.mark.gpu
def test_training_step_in_place_and_other_stream(ctx):
    """out written over the activations, dx over the gradient; the whole step on another stream."""
    from localfold_amd import device as D
    rng = np.random.default_rng(2)
    rows, c, h = 500, 128, 512
    w = transition_case(ctx, rng, c, h, torch.bfloat16)
    ws, saved = D.transition_train_weights(w), D.transition_saved(rows, c, h, ctx.device)
    x, grad = rows_of(rng, rows, c, torch.bfloat16).to(ctx.device), rows_of(rng, rows, c, torch.bfloat16).to(ctx.device)
    want = D.transition_train(ctx, x, ws, saved, accumulate=True)
    dx, grads = D.transition_backward(ctx, grad, ws, saved, accumulate=True)
    x2, g2 = x.clone(), grad.clone()
    D.transition_train(ctx, x2, ws, saved, out=x2, accumulate=True)
    _, again = D.transition_backward(ctx, g2, ws, saved, out=g2, accumulate=True)
    torch.cuda.synchronize()
    assert torch.equal(x2, want) and torch.equal(g2, dx) and all(torch.equal(grads[k], again[k]) for k in grads)
    s = torch.cuda.Stream()
    try:
        with torch.cuda.stream(s):
            ctx.bind_stream()
            x3, g3 = x.clone(), grad.clone()
            D.transition_train(ctx, x3, ws, saved, out=x3, accumulate=True)
            _, third = D.transition_backward(ctx, g3, ws, saved, out=g3, accumulate=True)
        s.synchronize()
    finally:
        ctx.bind_stream()
    assert torch.equal(x3, want) and torch.equal(g3, dx) and all(torch.equal(grads[k], third[k]) for k in grads)


@pytest.mark.gpu
def test_training_step_in_a_graph(ctx):
    """Two captured steps with scratch of their own, replayed in turn with eager steps (which move the
    context's workspace) between them, against the eager results; without scratch the capture is refused."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(4)
    rows, c, h = 700, 128, 256
    cases = []
    for k in range(2):
        w = transition_case(ctx, rng, c, h, torch.float32)
        ws, saved = D.transition_train_weights(w), D.transition_saved(rows, c, h, ctx.device)
        x, grad = rows_of(rng, rows, c, torch.float32).to(ctx.device), rows_of(rng, rows, c, torch.float32).to(ctx.device)
        out, dx = torch.empty_like(x), torch.empty_like(x)
        grads = {n: torch.zeros_like(w[n]) for n in w}
        need = max(ctx.lib.lf_transition_train_scratch(rows, c, h), ctx.lib.lf_transition_backward_scratch(rows, c, h))
        scratch = torch.empty(need, dtype=torch.uint8, device=ctx.device)

        def step(scratch, x=x, grad=grad, ws=ws, saved=saved, out=out, dx=dx, grads=grads):
            D.transition_train(ctx, x, ws, saved, out=out, accumulate=True, scratch=scratch)
            D.transition_backward(ctx, grad, ws, saved, out=dx, accumulate=True, grads=grads, scratch=scratch)

        step(scratch)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(g):
                ctx.bind_stream()
                with pytest.raises(capi.LocalfoldError, match="scratch"):
                    step(None)
                step(scratch)
        finally:
            ctx.bind_stream()
        cases.append((g, x, w, (out, dx, grads), step))
    for turn in range(4):
        for g, x, w, (out, dx, grads), step in cases:
            x += 0.25
            w["secondWeight"] *= 0.9
            g.replay()
            torch.cuda.synchronize()
            got = [out.clone(), dx.clone()] + [grads[n].clone() for n in sorted(grads)]
            big = torch.randn(4000 * (turn + 1), 128, device=ctx.device)      # moves the workspace
            D.layer_norm_backward(ctx, big, big, w["layerNormScale"], torch.ones(2, big.shape[0], device=ctx.device))
            step(None)
            torch.cuda.synchronize()
            want = [out, dx] + [grads[n] for n in sorted(grads)]
            assert all(torch.equal(p, q) for p, q in zip(got, want)), turn


@pytest.mark.gpu
def test_training_from_inference_weights(ctx):
    """The struct that transition_weights builds for lf_transition works here too."""
    from localfold_amd import device as D
    rng = np.random.default_rng(8)
    w = transition_case(ctx, rng, 128, 256, torch.float32)
    x, grad = rows_of(rng, 100, 128, torch.float32).to(ctx.device), rows_of(rng, 100, 128, torch.float32).to(ctx.device)
    got = []
    for ws in (D.transition_train_weights(w),
               D.transition_weights(D.DeviceWeights(ctx.device), {k: t.cpu().numpy() for k, t in w.items()})):
        saved = D.transition_saved(100, 128, 256, ctx.device)
        out = D.transition_train(ctx, x, ws, saved)
        dx, grads = D.transition_backward(ctx, grad, ws, saved)
        torch.cuda.synchronize()
        got.append([out, dx, *grads.values()])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_refusals(ctx):
    import ctypes as C
    from localfold_amd import capi, device as D
    dev = ctx.device
    x = torch.randn(10, 128, device=dev)
    s = torch.ones(128, device=dev)
    k = D.checkpoint_pack(ctx, x)
    w = D.fp8_weight(ctx, torch.randn(128, 64, device=dev))
    stats = torch.ones(2, 10, device=dev)
    with pytest.raises(ValueError):
        D.checkpoint_pack(ctx, x[:, ::2])
    with pytest.raises(TypeError):
        D.checkpoint_pack(ctx, x.double())
    with pytest.raises(ValueError):
        D.layer_norm(ctx, x.cpu(), s, s)
    with pytest.raises(TypeError):
        D.layer_norm(ctx, x, s.half(), s)
    with pytest.raises(ValueError):
        D.layer_norm(ctx, x, s[:64].contiguous(), s)
    with pytest.raises(capi.LocalfoldError, match="epsilon"):
        D.layer_norm(ctx, x, s, s, epsilon=0.0)
    with pytest.raises(capi.LocalfoldError, match="wide"):
        D.layer_norm(ctx, torch.randn(2, 4097, device=dev), torch.ones(4097, device=dev), torch.ones(4097, device=dev))
    with pytest.raises(capi.LocalfoldError, match="positive"):
        D.layer_norm(ctx, torch.empty(0, 128, device=dev), s, s)
    with pytest.raises(ValueError):
        D.fp8_linear(ctx, D.checkpoint_pack(ctx, x[:, :100].contiguous()), w)
    with pytest.raises(ValueError):
        D.fp8_linear(ctx, k, w, residual=torch.zeros(10, 64, device=dev), out=D.checkpoint_empty(10, 64, dev))
    with pytest.raises(ValueError):
        D.fp8_weight_grad(ctx, k, D.checkpoint_empty(11, 128, dev))
    with pytest.raises(capi.LocalfoldError, match="scratch has"):
        D.fp8_weight_grad(ctx, k, k, scratch=torch.empty(16, dtype=torch.uint8, device=dev))
    with pytest.raises(capi.LocalfoldError, match="aligned"):
        D.layer_norm_backward(ctx, x, x, s, stats, scratch=torch.empty(1 << 20, dtype=torch.uint8, device=dev)[3:])
    bad = D.Checkpoint(10, 128, torch.empty(10 * 128 + 8, dtype=torch.uint8, device=dev)[8:].view(10, 128), k.scales)
    with pytest.raises(capi.LocalfoldError, match="aligned"):
        D.checkpoint_pack(ctx, x, out=bad)
    a = capi.lf_layer_norm_backward_args()
    a.rows, a.channels, a.act_dtype, a.grad = 10, 128, capi.LF_F32, x.data_ptr()
    assert ctx.lib.lf_layer_norm_backward(ctx.handle, C.byref(a)) == capi.LF_ERR_INVALID
    assert b"either act or act_kept" in ctx.lib.lf_last_error()
    weights = transition_case(ctx, np.random.default_rng(0), 128, 64, torch.float32)
    ws = D.transition_train_weights(weights)
    with pytest.raises(ValueError):
        D.transition_train(ctx, x, ws, D.transition_saved(11, 128, 64, dev))
    with pytest.raises(capi.LocalfoldError, match="hidden"):
        D.transition_train(ctx, x, ws, D.transition_saved(10, 128, 65, dev))
    ws.w1.dtype = capi.LF_INT8
    with pytest.raises(capi.LocalfoldError, match="not trained"):
        D.transition_train(ctx, x, ws, D.transition_saved(10, 128, 64, dev))
    before = torch.cuda.current_device()
    assert before == 0


def dominated(rng, rows, k, n):
    """Operands whose first two products are a thousand times the others and cancel: what an instruction
    that drops the small ones beside them leaves out is all there is."""
    x, w = rng.normal(size=(rows, k)), rng.normal(size=(n, k)) / 4
    x[:, :2], w[:, 0], w[:, 1] = 32, 32, -32
    return torch.as_tensor(x).float(), torch.as_tensor(w).float()


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,n", [(59, 384, 1536), (3, 22, 49), (9000, 128, 257), (6001, 192, 300), (3100, 1000, 512),
                                      (59, 4096, 64), (25000, 1153, 130)])
def test_linear_sums_are_of_32_bits(ctx, dt, rows, k, n):
    """The small, resident and streamed products, whole and half groups of columns: whatever the output's
    type, sums are float32's."""
    from localfold_amd import capi, device as D
    x, w = dominated(np.random.default_rng(rows + k), rows, k, n)
    x8, w8 = D.checkpoint_pack(ctx, x.to(ctx.device)), D.fp8_weight(ctx, w.to(ctx.device), capi.LF_OUT_IN)
    xv, wv = values_of(x8), weight_values(w8)
    assert (xv[:, 0] * wv[:, :1] + xv[:, 1] * wv[:, 1:2]).max() == 0
    close(D.fp8_linear(ctx, x8, w8, dtype=dt), xv @ wv.T, linear_slack(xv, wv, k, True), dt)


# ---- the transition's step, each stage from what the stage before it kept ---------------------------
#
# Hidden gradients are not at hand.  A code is that of a number within its sum's float32 error (code_range),
# so all but those next to a border between two codes, a few in 10^4, are known, and what follows from them
# is held to float32's errors.

def code_range(lo, hi):
    """The smallest and the largest that a number within [lo, hi] may stand for once it is kept."""
    least, most = np.empty_like(lo), np.empty_like(hi)
    for g in range(0, lo.shape[1], 128):
        l, h = lo[:, g:g + 128], hi[:, g:g + 128]
        inner = np.where((l <= 0) & (h >= 0), 0.0, np.minimum(np.abs(l), np.abs(h)))
        fs = [scale_of(m.max(1, keepdims=True)) for m in (inner, np.maximum(np.abs(l), np.abs(h)))]
        least[:, g:g + 128] = np.minimum(*(np.maximum(round_e4m3(l / f), -448) * f for f in fs))
        most[:, g:g + 128] = np.maximum(*(np.minimum(round_e4m3(h / f), 448) * f for f in fs))
    return least, most


def sum_depth(k):
    return 32 + k / 32 + 4      # products of an instruction, instructions, waves that are joined


def check_step(dt, x, grad, p, residual, fast, saved, got):
    """A step's results against float64.  p: parameters by name; saved: the values of act, normed and
    hidden, and stats; got: out, dx and grads, as stored."""
    rows, c = x.shape
    h = saved["hidden"].shape[1]
    w1, w2, s, o = kept_weight64(p["firstWeight"]), kept_weight64(p["secondWeight"]), p["layerNormScale"], p["layerNormOffset"]
    y8, h8, x8 = saved["normed"], saved["hidden"], saved["act"]
    d1, d2 = sum_depth(c) * 2 * U, sum_depth(h) * 2 * U

    def within(v, lo, hi, label):
        lo, hi = code_range(lo, hi)
        bad = ~((v >= lo) & (v <= hi))
        assert not bad.any(), (label, int(bad.sum()), np.argwhere(bad)[:4].tolist())

    assert np.array_equal(x8, kept64(x)), "act"
    y, m, r = norm64(x, s, o, float(np.float32(1e-5)), fast)
    slack = norm_slack(x, s, o, m, r, c)
    within(y8, y - slack, y + slack, "normed")
    depth = 2 * (min(c, 64) + 8) * U
    size = (x * x).mean(1)
    close(saved["stats"][0], m[:, 0], depth * np.abs(x).mean(1), torch.float32, "mean")
    close(saved["stats"][1], r[:, 0], r[:, 0] * (depth * (1 + r[:, 0] ** 2 * size) + 4 * U), torch.float32, "rstd")
    pre = y8 @ w1 + p["firstBias"]
    slack = (np.abs(y8) @ np.abs(w1) + np.abs(p["firstBias"])) * d1
    within(h8, np.maximum(pre - slack, 0), np.maximum(pre + slack, 0), "hidden")
    total = h8 @ w2 + p["secondBias"]
    slack = (np.abs(h8) @ np.abs(w2) + np.abs(p["secondBias"])) * d2
    if residual:
        total = total + x
    close(got["out"], total, slack + 2 * U * np.abs(total), dt, "out")

    # gradients: of the weights over the rows (32 an instruction, three teams in turn, 256 splits joined in runs)
    d8, over = kept64(grad), (32 + rows / 96 + 51) * 2 * U
    close(got["grads"]["secondWeight"], h8.T @ d8, over * (np.abs(h8).T @ np.abs(d8)), torch.float32, "dw2")
    gate = h8 > 0
    pre = d8 @ w2.T
    slack = (np.abs(d8) @ np.abs(w2.T)) * d1
    lo, hi = code_range(np.where(gate, pre - slack, 0), np.where(gate, pre + slack, 0))
    e, off = (lo + hi) / 2, (hi - lo) / 2
    assert (off > 0).mean() < 0.01
    close(got["grads"]["firstWeight"], y8.T @ e, np.abs(y8).T @ (off + over * (np.abs(e) + off)), torch.float32, "dw1")
    if "firstBias" in got["grads"]:
        close(got["grads"]["firstBias"], e.sum(0), (off + over * (np.abs(e) + off)).sum(0), torch.float32, "db1")
        close(got["grads"]["secondBias"], d8.sum(0), over * np.abs(d8).sum(0), torch.float32, "db2")
    dy, off = e @ w1.T, (off + d2 * (np.abs(e) + off)) @ np.abs(w1.T)
    m, r = saved["stats"][0][:, None], saved["stats"][1][:, None]
    dx, ds, do = norm_backward64(dy, x8, s, m, r)
    hh, g, go = (x8 - m) * r, dy * s, off * np.abs(s)
    dh = 2 * U * (np.abs(x8) + np.abs(m)) * r
    b = np.abs(g * hh).mean(1, keepdims=True)
    slack = r * (4 * U * np.abs(g) + depth * np.abs(g).mean(1, keepdims=True) + dh * b
                 + np.abs(hh) * (depth * b + (np.abs(g) * dh).mean(1, keepdims=True)))
    slack = slack + r * (go + go.mean(1, keepdims=True) + np.abs(hh) * (go * np.abs(hh)).mean(1, keepdims=True)) + 4 * U * np.abs(dx)
    if residual:
        dx = dx + grad
        slack = slack + 2 * U * np.abs(dx)
    close(got["dx"], dx, slack, dt, "dx")
    # a lane's rows, a block's lanes, the blocks
    over = (rows / 256 + 128) * 2 * U
    close(got["grads"]["layerNormScale"], ds, (off * np.abs(hh) + over * np.abs(dy * hh) + np.abs(dy) * dh).sum(0), torch.float32, "ds")
    close(got["grads"]["layerNormOffset"], do, (off + over * np.abs(dy)).sum(0), torch.float32, "do")


def params64(w, c, h):
    zero = {"firstBias": np.zeros(h), "secondBias": np.zeros(c)}
    return {k: f64(w[k]) if k in w else zero[k] for k in ("layerNormScale", "layerNormOffset", "firstWeight", "firstBias",
                                                          "secondWeight", "secondBias")}


def checked_step(ctx, rows, c, h, dt, wdt, residual, fast, shift=0, spike=None, layouts=None):
    """Runs a step and checks it.  shift: everything that many elements behind an aligned address; layouts:
    of the two matrices as they are stored; spike: two hidden units a thousand times the others that cancel
    in the output, or whose gradients cancel in the first channel of the norm's output."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(rows + 5 * c + h)
    w = transition_case(ctx, rng, c, h, wdt, bias=rows != 45)
    if spike == "out":
        w["firstWeight"][:, :2], w["firstBias"][:2] = 0, 20
        w["secondWeight"][0] = torch.as_tensor(rng.normal(size=c)).to(wdt)
        w["secondWeight"][1] = -w["secondWeight"][0]
    elif spike == "dy":
        w["firstWeight"][:, :2], w["firstBias"][:2] = 0, 40
        w["firstWeight"][0, 0], w["firstWeight"][0, 1] = 4, -4
        w["secondWeight"][0] = torch.as_tensor(rng.normal(size=c)).to(wdt)
        w["secondWeight"][1] = w["secondWeight"][0]
    ws, saved = D.transition_train_weights(w), D.transition_saved(rows, c, h, ctx.device)
    turned = [l == capi.LF_OUT_IN for l in layouts] if layouts else [False, False]
    if layouts:
        stored = [w[n].t().contiguous() if t else w[n] for n, t in zip(("firstWeight", "secondWeight"), turned)]
        ws.w1, ws.w2 = (D._live_weight("w", t, l) for t, l in zip(stored, layouts))
    x, grad = rows_of(rng, rows, c, dt, 0.3).to(ctx.device), (rows_of(rng, rows, c, dt) * 0.01).to(dt).to(ctx.device)
    if rows > 2:
        grad[rows // 2] = 0      # a padded row
    out, dx = torch.empty_like(x), torch.empty_like(grad)
    if shift:
        x, grad, out, dx = (torch.cat([t.new_zeros(shift), t.flatten()])[shift:].view(rows, c) for t in (x, grad, out, dx))
    D.transition_train(ctx, x, ws, saved, out=out, accumulate=residual, fast_variance=fast)
    _, grads = D.transition_backward(ctx, grad, ws, saved, out=dx, accumulate=residual)
    torch.cuda.synchronize()
    got = {"out": f64(out), "dx": f64(dx), "grads": {k: f64(t) for k, t in grads.items()}}
    for n, t in zip(("firstWeight", "secondWeight"), turned):
        if t:
            got["grads"][n] = got["grads"][n].T
    kept = {"act": values_of(saved.act), "normed": values_of(saved.normed), "hidden": values_of(saved.hidden),
            "stats": f64(saved.stats)}
    check_step(dt, f64(x), f64(grad), params64(w, c, h), residual, fast, kept, got)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,c,h", [(300, 128, 512), (300, 64, 256), (150, 256, 320), (8100, 384, 1200)])
@pytest.mark.parametrize("spike", ["out", "dy"])
def test_transition_sums_are_of_32_bits(ctx, rows, c, h, dt, spike):
    """The step's products too, fused and composed: the float32 gradients of the norm's vectors come from them."""
    checked_step(ctx, rows, c, h, dt, torch.float32, False, False, spike=spike)


STEP_SHAPES = [(1, 128, 512, torch.float32, torch.float32, True, False), (37, 64, 256, torch.float16, torch.float32, True, True),
               (300, 128, 512, torch.bfloat16, torch.bfloat16, True, False), (33, 64, 128, torch.bfloat16, torch.float32, True, False),
               (31, 128, 128, torch.float16, torch.float16, False, True), (257, 64, 512, torch.float32, torch.float32, False, False),
               (1000, 128, 384, torch.float32, torch.bfloat16, True, True), (45, 128, 256, torch.float32, torch.float32, True, False),
               (66001, 64, 128, torch.bfloat16, torch.float32, True, False), (33003, 128, 128, torch.float16, torch.float32, False, False),
               # widths that run as single operators
               (150, 256, 1024, torch.float32, torch.float16, False, False), (90, 384, 100, torch.bfloat16, torch.float32, False, True),
               (45, 22, 70, torch.float32, torch.float32, True, False), (600, 49, 130, torch.float16, torch.bfloat16, False, False),
               (131, 64, 640, torch.bfloat16, torch.float32, True, False), (8100, 384, 1200, torch.bfloat16, torch.float32, True, False),
               (6200, 256, 512, torch.float16, torch.float32, True, False)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,h,dt,wdt,residual,fast", STEP_SHAPES)
def test_transition_step_to_f32(ctx, rows, c, h, dt, wdt, residual, fast):
    checked_step(ctx, rows, c, h, dt, wdt, residual, fast)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,c,h,dt,shift", [(70, 128, 256, torch.bfloat16, 1), (70, 64, 128, torch.float16, 4),
                                               (70, 128, 128, torch.float32, 1)])
def test_transition_step_off_alignment_to_f32(ctx, rows, c, h, dt, shift):
    checked_step(ctx, rows, c, h, dt, torch.float32, True, False, shift)


@pytest.mark.gpu
@pytest.mark.parametrize("first,second", [(0, 1), (1, 0), (1, 1)])
@pytest.mark.parametrize("rows,c,h,wdt", [(70, 128, 256, torch.float32), (50, 64, 128, torch.bfloat16), (90, 49, 130, torch.float16)])
def test_transition_step_layouts(ctx, rows, c, h, wdt, first, second):
    """Matrices stored [outputs, inputs], whose gradients come in that layout."""
    from localfold_amd import capi
    kinds = (capi.LF_IN_OUT, capi.LF_OUT_IN)
    checked_step(ctx, rows, c, h, torch.float32, wdt, True, False, layouts=(kinds[first], kinds[second]))


def test_transition_checks_see_mistakes():
    """check_step passes a step computed here, and none with a mistake in one of its results: zeros, another
    sign, columns in another order, a column's values off by a twentieth, a tile of rows left out of a sum."""
    rng = np.random.default_rng(1)
    for rows, c, h, dt, residual in ((300, 128, 256, torch.bfloat16, True), (700, 64, 128, torch.float32, False)):
        p = {"layerNormScale": 1 + 0.2 * rng.uniform(-1, 1, c), "layerNormOffset": 0.1 * rng.uniform(-1, 1, c),
             "firstWeight": rng.normal(size=(c, h)) / math.sqrt(c), "firstBias": 0.1 * rng.uniform(-1, 1, h),
             "secondWeight": rng.normal(size=(h, c)) / math.sqrt(h), "secondBias": 0.1 * rng.uniform(-1, 1, c)}
        x, grad = f64(rows_of(rng, rows, c, dt, 0.3)), f64((rows_of(rng, rows, c, dt) * 0.01).to(dt))

        def stored(v, t=torch.float32):
            return f64(torch.as_tensor(v).to(t))

        y, m, r = norm64(x, p["layerNormScale"], p["layerNormOffset"], float(np.float32(1e-5)))
        w1, w2 = kept_weight64(p["firstWeight"]), kept_weight64(p["secondWeight"])
        x8, y8, d8 = kept64(x), kept64(y), kept64(grad)
        h8 = kept64(np.maximum(y8 @ w1 + p["firstBias"], 0))
        e8 = kept64(np.where(h8 > 0, d8 @ w2.T, 0))
        stats = stored(np.concatenate([m, r], 1).T)
        dy = e8 @ w1.T
        dx, ds, do = norm_backward64(dy, x8, p["layerNormScale"], stats[0][:, None], stats[1][:, None])
        out = h8 @ w2 + p["secondBias"]
        got = {"out": stored(out + x if residual else out, dt), "dx": stored(dx + grad if residual else dx, dt),
               "grads": {k: stored(v) for k, v in (("firstWeight", y8.T @ e8), ("firstBias", e8.sum(0)),
                                                   ("secondWeight", h8.T @ d8), ("secondBias", d8.sum(0)),
                                                   ("layerNormScale", ds), ("layerNormOffset", do))}}
        saved = {"act": x8, "normed": y8, "hidden": h8, "stats": stats}
        check_step(dt, x, grad, p, residual, False, saved, got)

        def refused(saved, got):
            with pytest.raises(AssertionError):
                check_step(dt, x, grad, p, residual, False, saved, got)

        def one_column(v):
            v = v.copy()
            v[..., 5] *= 1.05
            return v

        wrong = {"zeros": np.zeros_like, "sign": np.negative, "order": lambda v: np.roll(v, 4, -1), "column": one_column}
        for how, f in wrong.items():
            for k in ("out", "dx"):
                refused(saved, {**got, k: f(got[k])})
            for k in got["grads"]:
                refused(saved, {**got, "grads": {**got["grads"], k: f(got["grads"][k])}})
        tail = slice(0, rows - 32)       # a tile of rows
        for k, v in (("layerNormScale", norm_backward64(dy[tail], x8[tail], p["layerNormScale"], stats[0][tail, None],
                                                        stats[1][tail, None])[1]), ("layerNormOffset", dy[tail].sum(0)),
                     ("firstWeight", y8[tail].T @ e8[tail]), ("firstBias", e8[tail].sum(0))):
            refused(saved, {**got, "grads": {**got["grads"], k: stored(v)}})
        for k in ("normed", "hidden"):
            refused({**saved, k: np.roll(saved[k], 1, 1)}, got)
        # the norm's incoming gradient rounded to 16 bits on its way
        if dt != torch.float32:
            _, ds, do = norm_backward64(stored(dy, dt), x8, p["layerNormScale"], stats[0][:, None], stats[1][:, None])
            refused(saved, {**got, "grads": {**got["grads"], "layerNormScale": stored(ds)}})
            refused(saved, {**got, "grads": {**got["grads"], "layerNormOffset": stored(do)}})


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", LINEAR_SHAPES + LONG_SHAPES + [(9000, 128, 257), (6001, 192, 300), (2500, 1216, 400)])
def test_linear_kept_sums_are_of_32_bits(ctx, rows, k, n):
    """A kept product is the code of a number within float32's error of the product, also where its
    largest terms cancel."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(rows + 7 * k + n)
    plain = rows_of(rng, rows, k, torch.float32), torch.as_tensor(rng.normal(size=(n, k)) / math.sqrt(k)).float()
    for x, w in (plain, dominated(rng, rows, k, n)) if k > 2 else (plain,):
        x8, w8 = D.checkpoint_pack(ctx, x.to(ctx.device)), D.fp8_weight(ctx, w.to(ctx.device), capi.LF_OUT_IN)
        bias = vec(rng, ctx, n, 1.0)
        got = D.checkpoint_empty(rows, n, ctx.device)
        D.fp8_linear(ctx, x8, w8, bias, out=got)
        xv, wv = values_of(x8), weight_values(w8)
        want = xv @ wv.T + f64(bias)
        slack = linear_slack(xv, wv, k, True) + 2 * U * (np.abs(want) + np.abs(f64(bias)))
        lo, hi = code_range(want - slack, want + slack)
        v = values_of(got)
        assert ((v >= lo) & (v <= hi)).all()


# A half group of columns at the end: the small, resident and streamed products.
@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(40, 192, 200), (40, 64, 200), (9000, 192, 200), (40, 1344, 200), (13000, 1344, 260)])
def test_linear_weight_specials(ctx, rows, k, n):
    """A NaN or an infinity in a weight's row stays in that output, wherever it lies in the row."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(rows + k)
    w = (rng.normal(size=(n, k)) / math.sqrt(k)).astype(np.float32).astype(np.float64)
    w[17, 5], w[41, k - 1], w[n - 1, k // 2], w[130, 0] = np.nan, np.inf, -np.inf, np.nan
    bad = np.zeros(n, bool)
    bad[[17, 41, n - 1, 130]] = True
    x8 = D.checkpoint_pack(ctx, torch.as_tensor(rng.normal(size=(rows, k))).float().to(ctx.device))
    wt = torch.as_tensor(w).float().to(ctx.device)
    w8 = D.fp8_weight(ctx, wt, capi.LF_OUT_IN)
    turned = D.fp8_weight(ctx, wt.t().contiguous(), capi.LF_IN_OUT)
    assert torch.equal(w8.codes & 127, turned.codes & 127) and torch.equal(w8.scales, turned.scales)
    xv, wv = values_of(x8), weight_values(w8)
    assert np.array_equal(np.isnan(wv), ~np.isfinite(w))
    assert np.array_equal(wv[~bad], kept_weight64(np.where(np.isfinite(w), w, 0))[~bad])
    want, slack = xv @ wv[~bad].T, linear_slack(xv, wv[~bad], k, True)
    for dt in TYPES:
        out = f64(D.fp8_linear(ctx, x8, w8, relu=True, dtype=dt))
        assert np.isnan(out[:, bad]).all()
        close(out[:, ~bad], np.maximum(want, 0), slack, dt)
    kept = D.checkpoint_empty(rows, n, ctx.device)
    D.fp8_linear(ctx, x8, w8, out=kept)
    v = values_of(kept)
    assert np.isnan(v[:, bad]).all() and np.isfinite(v[:, ~bad]).all()


@pytest.mark.gpu
def test_weight_grad_of_one_split_takes_no_workspace(ctx):
    """Few rows are not split: their sums go straight to the result."""
    from localfold_amd import device as D
    rng = np.random.default_rng(0)
    rows, n, k = 40, 3000, 2000
    own = D.Context(0)
    try:
        g8, x8 = (D.checkpoint_pack(own, rows_of(rng, rows, c, torch.float32).to(own.device)) for c in (n, k))
        before = own.memory_stats()
        bias = torch.empty(n, device=own.device)
        out = D.fp8_weight_grad(own, g8, x8, bias_out=bias)
        torch.cuda.synchronize()
        assert own.memory_stats() == before
        given = torch.empty(own.lib.lf_fp8_weight_grad_scratch(rows, n, k), dtype=torch.uint8, device=own.device)
        assert torch.equal(out, D.fp8_weight_grad(own, g8, x8, scratch=given))
        many = D.checkpoint_pack(own, rows_of(rng, 5000, 64, torch.float32).to(own.device))
        D.fp8_weight_grad(own, many, many)
        torch.cuda.synchronize()
        assert own.memory_stats()["currentBytes"] > before["currentBytes"]
    finally:
        own.close()


def test_scratch_of_a_step_of_few_rows():
    """A step whose weight gradients are not split asks for no partial sums of them."""
    from localfold_amd import capi
    lib = capi.load()
    rows, c, h = 59, 384, 1536
    operands = 2 * 2 * h * c + rows * (3 * (c + h) + 4 * c)     # packed weights, kept gradients, the norm's gradient
    assert lib.lf_transition_backward_scratch(rows, c, h) < operands + 2 * c * 4 * 600


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_checkpoint_scale_of_a_group_with_nothing_finite(ctx, dt):
    """It has no largest finite value, so its scale is that of zeros, whether infinities or NaN are what it holds."""
    from localfold_amd import device as D
    for c in (64, 128, 200):
        x = torch.ones(4, c, dtype=dt)
        x[0], x[1], x[2, :] = float("nan"), float("inf"), float("nan")
        x[2, 0] = -float("inf")
        kept = D.checkpoint_pack(ctx, x.to(ctx.device))
        ys = D.checkpoint_empty(4, c, ctx.device)      # a row with a NaN is normalised to NaN
        D.layer_norm(ctx, x.to(ctx.device), torch.ones(c, device=ctx.device), torch.zeros(c, device=ctx.device), y_saved=ys)
        torch.cuda.synchronize()
        assert np.isnan(values_of(kept)[:3]).all() and np.isnan(values_of(ys)[:3]).all()
        assert (kept.scales[:, :3] == 1).all() and (kept.scales[:, 3] == 119).all()
        assert (ys.scales[:, :3] == 1).all()


@pytest.mark.gpu
def test_products_at_the_ends_of_the_scales(ctx):
    """Kept values are exact operands at scale bytes 3 to 246; below, multiples of 2^-133; from 2^128 on, infinities."""
    from localfold_amd import capi, device as D
    rows = 254
    scales = torch.full((1, 256), 127, dtype=torch.uint8)
    scales[0, :rows] = torch.arange(1, rows + 1)
    w8 = D.fp8_weight(ctx, torch.eye(16, 128, device=ctx.device), capi.LF_OUT_IN)
    for first, n in ((0x01, 126), (0x81, 126)):
        for start in range(0, n, 16):
            codes = torch.zeros(rows, 128, dtype=torch.uint8)
            codes[:, :16] = torch.arange(first + start, first + start + 16).clamp(max=first + n - 1)
            x8 = D.Checkpoint(rows, 128, codes.to(ctx.device), scales.to(ctx.device))
            out, v = f64(D.fp8_linear(ctx, x8, w8, dtype=torch.float32)), values_of(x8)[:, :16]
            assert np.array_equal(out[2:246], v[2:246])
            assert (out[:2] % 2.0 ** -133 == 0).all() and (np.abs(out[:2] - v[:2]) <= 2.0 ** -134).all()
            small = np.abs(v).max(1) < 2.0 ** 128     # beyond, an infinity times the other weights' zeros
            assert np.array_equal(out[2:][small[2:]], v[2:][small[2:]]) and not np.isfinite(out[~small]).any()


@pytest.mark.gpu
def test_size_limits(ctx):
    """Refused by the host, which launches nothing."""
    import ctypes as C
    from localfold_amd import capi
    x = torch.zeros(1024, device=ctx.device)
    for rows, cols, word in ((2 ** 28 + 1, 64, b"2^34"), (2 ** 28 + 1, 1, b"2^34"), (1, 65537, b"wide"), (0, 64, b"positive")):
        kept = capi.lf_checkpoint(rows, cols, x.data_ptr(), x.data_ptr())
        for entry in ("lf_checkpoint_pack", "lf_checkpoint_unpack"):
            a = capi.lf_checkpoint_args(capi.LF_F32, x.data_ptr(), C.pointer(kept))
            assert getattr(ctx.lib, entry)(ctx.handle, C.byref(a)) == capi.LF_ERR_INVALID
            assert word in ctx.lib.lf_last_error()
    w = capi.lf_fp8_weight_args()
    out = capi.lf_fp8_weight(65537, 8, x.data_ptr(), x.data_ptr())
    w.w = capi.lf_weight(capi.LF_F32, capi.LF_OUT_IN, 65537, 8, 0, x.data_ptr(), None, None)
    w.out = C.pointer(out)
    assert ctx.lib.lf_fp8_pack_weight(ctx.handle, C.byref(w)) == capi.LF_ERR_INVALID and b"65536" in ctx.lib.lf_last_error()


@pytest.mark.gpu
def test_weight_grad_of_one_split_in_a_graph(ctx):
    """It needs no scratch, so a captured call may come without; rows that are split are refused."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(9)
    g8, x8 = (D.checkpoint_pack(ctx, rows_of(rng, 50, c, torch.float32).to(ctx.device)) for c in (130, 70))
    many = D.checkpoint_pack(ctx, rows_of(rng, 5000, 64, torch.float32).to(ctx.device))
    out, bias = torch.empty(130, 70, device=ctx.device), torch.empty(130, device=ctx.device)
    big = torch.empty(64, 64, device=ctx.device)
    D.fp8_weight_grad(ctx, g8, x8, out=out, bias_out=bias)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    try:
        with torch.cuda.graph(graph):
            ctx.bind_stream()
            with pytest.raises(capi.LocalfoldError, match="scratch"):
                D.fp8_weight_grad(ctx, many, many, out=big)
            D.fp8_weight_grad(ctx, g8, x8, out=out, bias_out=bias)
    finally:
        ctx.bind_stream()
    for turn in range(3):
        D.checkpoint_pack(ctx, rows_of(rng, 50, 130, torch.float32).to(ctx.device), out=g8)
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone(), bias.clone()
        D.fp8_weight_grad(ctx, many, many, out=big)      # eager, with the workspace
        D.fp8_weight_grad(ctx, g8, x8, out=out, bias_out=bias)
        torch.cuda.synchronize()
        assert torch.equal(got[0], out) and torch.equal(got[1], bias), turn
