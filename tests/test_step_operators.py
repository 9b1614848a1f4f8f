"""Relative positions, products of 4 bits and orthogonalised updates, against float64 restatements.

Tolerances.  U = 2^-24 is half a step of float32; a sum whose terms pass through at most D additions is off by
at most D * 2U times the sum of magnitudes (2U: an addition may cut instead of round).  A stored value adds half a
step of its type, relative to it."""
import ast
import ctypes as C
import glob
import inspect
import math
import os
import re
import subprocess

import numpy as np
import pytest
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -133}
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NS = (3.4445, -4.7750, 2.0315)
EPS = 1e-7


def f64(t):
    return t.detach().cpu().double().numpy()


def close(got, want, slack, dt, label=""):
    """|got - want| within `slack` (before the store) and the store's half step."""
    got = f64(got) if isinstance(got, torch.Tensor) else got
    bound = slack + HALF[dt] * (np.abs(want) + slack) + TINY[dt]
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (label, int(bad.sum()), np.argwhere(bad)[:4].tolist(),
                           float(np.nanmax(np.abs(got - want) / np.maximum(bound, 1e-300))))


# ---- restatements --------------------------------------------------------------------------------

def rows64(boundaries, qp, kp, qs=None, ks=None):
    d = qp.astype(np.int64)[:, None] - kp.astype(np.int64)
    row = np.searchsorted(boundaries.astype(np.int64), d.ravel(), side="right").reshape(d.shape)
    if qs is not None:
        row = np.where(qs[:, None] == ks, row, len(boundaries) + 1)
        row = np.where((qs[:, None] < 0) | (ks < 0), -1, row)
    return row


E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def round_e2m1(v):
    a = np.abs(v)
    step = np.where(a < 2, 0.5, np.where(a < 4, 1.0, 2.0))
    return np.copysign(np.round(a / step) * step, v)


def mx64(x):
    """x after a round trip through 4 bits, groups of 32 columns."""
    out = np.array(x, np.float64)
    for g in range(0, x.shape[1], 32):
        p = out[:, g:g + 32]
        most = np.abs(p).max(1, keepdims=True)
        m, e = np.frexp(np.where(np.isfinite(most), most, 1.0))
        f = 2.0 ** np.where(most > 0, np.maximum(e - 3 + (m > 0.75), -126), -126.0)
        with np.errstate(invalid="ignore"):
            out[:, g:g + 32] = np.where(np.isfinite(most), round_e2m1(np.where(np.isfinite(most), p, 0) / f) * f, np.nan)
    return out


def bytes64(x):
    """Scale bytes [groups, rows] of finite rows."""
    p = np.zeros((x.shape[0], -(-x.shape[1] // 128) * 128))
    p[:, :x.shape[1]] = np.abs(x)
    most = p.reshape(x.shape[0], -1, 32).max(2)
    m, e = np.frexp(most)
    return np.where(most > 0, np.maximum(e - 3 + (m > 0.75) + 127, 1), 1).T


def values_of(m):
    """What an Mx4 holds, by its bytes."""
    codes, scales = m.codes.cpu().numpy(), m.scales.cpu().numpy().astype(int)
    c = np.stack([codes & 15, codes >> 4], -1).reshape(m.rows, -1)
    v = np.where(c >= 8, -1, 1) * E2M1[c & 7]
    b = np.repeat(scales[:, :m.rows].T, 32, axis=1)
    return np.where(b == 255, np.nan, v * 2.0 ** (b - 127)), b


def schulz64(u, steps, coefficients=NS, epsilon=EPS):
    """O(u), and a bound of what float32 products may be off by in the Frobenius norm.

    A step maps singular values by p(s) = a s + b s^3 + c s^5, so a difference in X grows at most by the largest |p'|
    on [-s, s] (the divided differences of p).  The step's own rounding: sums of n products of factors that keep 22
    bits are off by gamma(n) of the magnitudes' sum, at most the product of the Frobenius norms."""
    x = u / (np.linalg.norm(u) + epsilon)
    tall = x.shape[0] > x.shape[1]
    x = x.T if tall else x
    m, n = x.shape
    co = [coefficients] * steps if np.ndim(coefficients) == 1 else coefficients
    gamma = lambda k: 2.0 ** -21 + 3 * (k / 32 + 8) * 2 * U
    e = 4 * U
    for a, b, c in co:
        s, f = np.linalg.norm(x, 2), np.linalg.norm(x)
        g = x @ x.T
        p = a * np.eye(m) + b * g + c * g @ g
        dg = gamma(n) * f * f
        dp = (abs(b) + 2 * abs(c) * s * s) * dg + gamma(m) * abs(c) * np.linalg.norm(g) ** 2 + 2.0 ** -21 * np.linalg.norm(p)
        t = np.linspace(0, s, 2001)
        grow = np.abs(a + 3 * b * t ** 2 + 5 * c * t ** 4).max()
        x = p @ x
        e = grow * e + s * dp + gamma(m) * np.linalg.norm(p) * f + 2.0 ** -21 * np.linalg.norm(x)
    return (x.T if tall else x), e


# ---- on the CPU ----------------------------------------------------------------------------------

def test_boundaries():
    from localfold_amd import device as D
    b = D.clipped_boundaries(32).numpy()
    d = np.arange(-300, 301)
    assert (np.searchsorted(b, d, side="right") == np.clip(d, -32, 32) + 32).all()
    for buckets, far in ((32, 128), (4, 1), (8, 64), (64, 4096), (6, 10)):
        b = D.log_boundaries(buckets, far).numpy().astype(int)
        assert len(b) == buckets - 1 and (np.diff(b) >= 0).all() and b[-1] == far
        half, near = buckets // 2, max(1, buckets // 4)
        assert (b[half - 1:][1:] == 1 - b[:half - 1][::-1]).all()          # distances 0 and below mirror those above
        for n in range(near, min(far, 500)):
            if far == near:
                break
            x = (half - near) * math.log(n / near) / math.log(far / near)
            if abs(x - round(x)) > 1e-9:
                assert np.searchsorted(b[half - 1:], n, side="right") == near + math.floor(x), (buckets, far, n)
    for bad in ((3, 8), (2, 8), (32, 7)):
        with pytest.raises(ValueError):
            D.log_boundaries(*bad)
    with pytest.raises(ValueError):
        D.clipped_boundaries(0)


def test_log_boundaries_of_far_distances():
    """Up to what positions can differ by, at once; past what an int32 holds is refused."""
    from localfold_amd import device as D
    for buckets, far in ((32, 10 ** 6), (64, 2 ** 31 - 1), (4096, 2 ** 31 - 1)):
        b = D.log_boundaries(buckets, far)
        half, near = buckets // 2, buckets // 4
        steps = [int(v) for v in b[half - 1:]]
        assert b.dtype == torch.int32 and len(b) == buckets - 1 and steps[:near] == list(range(1, near + 1)) and steps[-1] == far
        for j in (1, 2, (half - near) // 2, half - near - 1):        # the first whole number at (far / near)^(j / half - near) near
            n, k = steps[near - 1 + j], half - near
            assert (n - 1) ** k < near ** (k - j) * far ** j <= n ** k, (buckets, far, j)
    for far in (2 ** 31, 10 ** 30):
        with pytest.raises(ValueError, match="max_distance"):
            D.log_boundaries(32, far)


def documented_examples():
    """The Python examples of the documents beside the package that call its device module, as (document, code)."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    for path in sorted(glob.glob(os.path.join(root, "*.md"))):
        with open(path, encoding="utf-8") as f:
            for code in re.findall(r"^```python\n(.*?)^```", f.read(), re.S | re.M):
                if "device as D" in code:
                    yield os.path.basename(path), code


def test_documented_calls():
    """Every call of an example has the function's arguments, and what it takes apart is a tuple of as many."""
    from localfold_amd import device as D

    def returned(f):
        return [n.value for n in ast.walk(ast.parse(inspect.getsource(f))) if isinstance(n, ast.Return)]

    seen = set()
    for where, code in documented_examples():
        tree = ast.parse(code)
        for call in (n for n in ast.walk(tree) if isinstance(n, ast.Call)):
            if isinstance(call.func, ast.Attribute) and isinstance(call.func.value, ast.Name) and call.func.value.id == "D":
                seen.add(call.func.attr)
                f = getattr(D, call.func.attr)
                inspect.signature(f).bind(*call.args, **{k.arg: k.value for k in call.keywords})
        for n in ast.walk(tree):
            if isinstance(n, ast.Assign) and isinstance(n.targets[0], ast.Tuple) and isinstance(n.value, ast.Call):
                f = getattr(D, n.value.func.attr)
                assert all(isinstance(v, ast.Tuple) and len(v.elts) == len(n.targets[0].elts) for v in returned(f)), (where, ast.unparse(n))
    assert {"relative_position", "relative_position_backward", "mx4_pack", "mx4_linear", "muon_step"} <= seen


def test_struct_layouts(tmp_path):
    from localfold_amd import capi
    names = [n for n in dir(capi) if n.startswith(("lf_relative", "lf_mx4", "lf_orthogonalize", "lf_muon"))
             and isinstance(getattr(capi, n), type) and issubclass(getattr(capi, n), C.Structure)]
    assert len(names) == 9
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "localfold.h"\nint main(void) {\n' + "".join(
        f'printf("{n} - %zu\\n", sizeof({n}));\n' + "".join(
            f'printf("{n} {f[0]} %zu\\n", offsetof({n}, {f[0]}));\n' for f in getattr(capi, n)._fields_)
        for n in names) + "return 0;}\n")
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "sizes")], check=True)
    for line in subprocess.run([str(tmp_path / "sizes")], check=True, capture_output=True, text=True).stdout.splitlines():
        n, field, size = line.split()
        s = getattr(capi, n)
        assert (C.sizeof(s) if field == "-" else getattr(s, field).offset) == int(size), (n, field)


def test_mx4_layout_is_checked():
    from localfold_amd import device as D
    m = D.mx4_empty(17, 130, "cpu")
    assert m.codes.shape == (17, 128) and m.scales.shape == (8, 32)
    with pytest.raises(ValueError):
        D.Mx4(17, 130, m.codes[:, :65], m.scales)
    with pytest.raises(ValueError):
        D.Mx4(17, 130, m.codes, m.scales[:5])
    codes, scales = torch.empty((2 ** 32 + 5, 64), dtype=torch.uint8, device="meta"), torch.empty((4, 2 ** 32 + 16), dtype=torch.uint8, device="meta")
    with pytest.raises(ValueError, match="at most"):
        D.Mx4(2 ** 32 + 5, 1, codes, scales)


def test_scratch_sizes_and_null_need_no_device():
    from localfold_amd import capi
    lib = capi.load()
    pairs = capi.lf_relative_pairs(100, 90, None, None, None, None, 64, None)
    assert lib.lf_relative_position_backward_scratch(C.byref(pairs), 128) >= 66 * 128 * 4
    assert lib.lf_relative_position_backward_scratch(None, 128) == lib.lf_relative_position_backward_scratch(C.byref(pairs), 0) == 0
    assert lib.lf_mx4_pack_scratch(5, 30) >= 30 * 4 and lib.lf_mx4_pack_scratch(0, 30) == 0
    assert lib.lf_mx4_linear_scratch(-1, 3, 3, 1) == 0
    assert lib.lf_muon_scratch(2, 300, 500) >= 2 * 300 * 500 * 4 and lib.lf_muon_scratch(0, 3, 3) == 0
    for name in ("lf_relative_position", "lf_relative_position_backward", "lf_mx4_pack", "lf_mx4_unpack", "lf_mx4_linear",
                 "lf_orthogonalize", "lf_muon_step"):
        assert getattr(lib, name)(None, None) == capi.LF_ERR_INVALID and name.encode() in lib.lf_last_error()


def test_scratch_of_the_most_keys():
    """256 blocks at most leave partial sums, also of 2^31 - 1 keys, which rounded up to whole units are more."""
    from localfold_amd import capi
    lib = capi.load()
    for q, k in ((1, 2 ** 31 - 1), (1, 2 ** 31 - 200), (8, 2 ** 31 - 1), (2 ** 31 - 1, 1)):
        pairs = capi.lf_relative_pairs(q, k, None, None, None, None, 1, None)
        assert lib.lf_relative_position_backward_scratch(C.byref(pairs), 1) == 256 * 3 * 4, (q, k)


def test_coefficients_are_checked():
    from localfold_amd import device as D
    assert list(D._coefficients((1, 2, 3), 2)) == [1, 2, 3, 1, 2, 3]
    assert list(D._coefficients([(1, 2, 3), (4, 5, 6)], 2)) == [1, 2, 3, 4, 5, 6]
    for bad in (((1, 2), 2), ([(1, 2, 3)], 2), ((1, 2, 3), 0), ((1, 2, 3), 33)):
        with pytest.raises(ValueError):
            D._coefficients(*bad)


def test_schulz_bound_holds_for_float32():
    """The bound that the GPU tests use, on float32 products here."""
    rng = np.random.default_rng(0)
    for m, n in ((5, 9), (40, 30), (64, 200)):
        u = rng.normal(size=(m, n))
        want, bound = schulz64(u, 5)
        x = (u / (np.linalg.norm(u) + EPS)).astype(np.float32)
        x = x.T if m > n else x
        for _ in range(5):
            g = x @ x.T
            x = np.float32(NS[0]) * x + (np.float32(NS[1]) * g + np.float32(NS[2]) * (g @ g)) @ x
        d = np.linalg.norm((x.T if m > n else x) - want)
        assert d <= bound < 0.05 * np.linalg.norm(want)


# ---- relative positions --------------------------------------------------------------------------

def chain(rng, n, segments):
    p = np.arange(n, dtype=np.int32) - 3
    if n > 2:
        p[rng.integers(0, n):] += 200
    s = np.sort(rng.integers(0, 3, n)).astype(np.int32)
    if n > 3:
        s[rng.integers(0, n, n // 8 + 1)] = -1
    return p, (s if segments else None)


def on(ctx, a):
    return None if a is None else torch.as_tensor(a).to(ctx.device)


PAIRS = [(1, 1, 1, 3), (1, 300, 128, 32), (59, 59, 128, 32), (7, 65, 22, 4), (33, 130, 1, 2), (5, 257, 130, 32), (64, 63, 16, 9),
         (3, 40, 515, 1), (300, 2, 64, 32), (40, 70, 37, 8), (90, 100, 384, 5), (200, 190, 8, 1), (300, 400, 22, 4),
         (400, 500, 130, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("segments", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("q,k,c,reach", PAIRS)
def test_position(ctx, q, k, c, reach, dt, segments):
    from localfold_amd import device as D
    rng = np.random.default_rng(q * 1000 + k)
    b = D.clipped_boundaries(reach).numpy()
    (qp, qs), (kp, ks) = chain(rng, q, segments), chain(rng, k, segments)
    rows = len(b) + 1 + segments
    tdt = TYPES[(q + k) % 3]
    table = torch.as_tensor(rng.normal(size=(rows, c))).to(tdt).to(ctx.device)
    bias = on(ctx, rng.normal(size=c).astype(np.float32)) if c % 2 else None
    base = torch.as_tensor(rng.normal(size=(q, k, c))).to(dt).to(ctx.device)
    where = dict(key_positions=on(ctx, kp), segments=on(ctx, qs), key_segments=on(ctx, ks))
    row = rows64(b, qp, kp, qs, ks)
    add = np.where(row[:, :, None] < 0, 0.0, f64(table)[np.maximum(row, 0)] + (0 if bias is None else f64(bias)))
    got = D.relative_position(ctx, table, on(ctx, b), on(ctx, qp), bias=bias, dtype=dt, **where)
    assert got.dtype == dt and got.shape == (q, k, c)
    close(got, add, 2 * U * np.abs(add), dt)
    want = add + f64(base)
    slack = 4 * U * (np.abs(add) + np.abs(want))
    got = D.relative_position(ctx, table, on(ctx, b), on(ctx, qp), bias=bias, pair=base, **where)
    close(got, want, slack, dt)
    kept = base.clone()
    D.relative_position(ctx, table, on(ctx, b), on(ctx, qp), bias=bias, pair=kept, out=kept, **where)
    assert torch.equal(kept, got)


@pytest.mark.gpu
@pytest.mark.parametrize("segments", [False, True])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("q,k,c,reach", PAIRS + [(200, 190, 128, 32), (21, 700, 8, 64), (30, 30, 12, 300)])
def test_position_backward(ctx, q, k, c, reach, dt, segments):
    """(30, 30, 12, 300): more rows than a block holds at once."""
    from localfold_amd import device as D
    rng = np.random.default_rng(q * 1000 + k + 1)
    b = D.clipped_boundaries(reach).numpy()
    (qp, qs), (kp, ks) = chain(rng, q, segments), chain(rng, k, segments)
    rows = len(b) + 1 + segments
    row = rows64(b, qp, kp, qs, ks)
    g = rng.normal(size=(q, k, c))
    grad = torch.as_tensor(g).to(dt)
    grad[torch.as_tensor(row < 0)] = math.nan                # padding, whatever it holds
    grad = grad.to(ctx.device)
    want, mags = np.zeros((rows, c)), np.zeros((rows, c))
    flat = np.nan_to_num(f64(grad)).reshape(-1, c)
    np.add.at(want, np.maximum(row.ravel(), 0), np.where(row.ravel()[:, None] < 0, 0, flat))
    np.add.at(mags, np.maximum(row.ravel(), 0), np.where(row.ravel()[:, None] < 0, 0, np.abs(flat)))
    count = np.bincount(row.ravel()[row.ravel() >= 0], minlength=rows)
    gdt = TYPES[(q + c) % 3]
    where = dict(key_positions=on(ctx, kp), segments=on(ctx, qs), key_segments=on(ctx, ks))
    db = torch.empty(c, dtype=gdt, device=ctx.device)
    got = D.relative_position_backward(ctx, grad, on(ctx, b), on(ctx, qp), bias_grad=db, grad_dtype=gdt, **where)
    close(got, want, 2 * U * count[:, None] * mags, gdt, "table")
    close(db, want.sum(0), 2 * U * count.sum() * mags.sum(0), gdt, "bias")
    again = D.relative_position_backward(ctx, grad, on(ctx, b), on(ctx, qp), grad_dtype=gdt, **where)
    assert torch.equal(got, again)
    assert (f64(got)[count == 0] == 0).all()


@pytest.mark.gpu
def test_position_far_apart_and_odd_boundaries(ctx):
    """Differences past 32 bits, boundaries at both ends of the range, repeated, and none."""
    from localfold_amd import device as D
    lo, hi = -2 ** 31, 2 ** 31 - 1
    p = np.array([lo, lo + 1, -1, 0, 1, hi - 1, hi], np.int32)
    for b in ([], [0], [lo], [hi], [lo, lo, 0, 0, 0, hi], [-5, -5, 7]):
        b = np.array(b, np.int32)
        row = rows64(b, p, p)
        table = torch.arange(len(b) + 1, dtype=torch.float32, device=ctx.device)[:, None].contiguous()
        got = D.relative_position(ctx, table, on(ctx, b), on(ctx, p))
        assert (f64(got)[:, :, 0] == row).all(), b
        grad = torch.ones((7, 7, 1), device=ctx.device)
        dt = D.relative_position_backward(ctx, grad, on(ctx, b), on(ctx, p))
        assert (f64(dt)[:, 0] == np.bincount(row.ravel(), minlength=len(b) + 1)).all(), b


@pytest.mark.gpu
def test_position_of_the_most_keys(ctx):
    """2^31 - 1 keys of a query, one channel: both ends of the keys and of the buckets."""
    from localfold_amd import device as D
    k, half = 2 ** 31 - 1, 2 ** 30
    kp = torch.arange(k, dtype=torch.int32, device=ctx.device)
    qp = torch.tensor([half], dtype=torch.int32, device=ctx.device)
    b = torch.tensor([1, half], dtype=torch.int32, device=ctx.device)       # keys past `half`, those before it, key 0
    table = torch.tensor([[1.0], [2.0], [3.0]], device=ctx.device)
    out = torch.zeros((1, k, 1), dtype=torch.bfloat16, device=ctx.device)
    D.relative_position(ctx, table, b, qp, key_positions=kp, out=out)
    flat = out.view(-1)
    assert float(flat[0]) == 3 and bool((flat[1:half] == 2).all()) and bool((flat[half:] == 1).all())
    out.zero_()
    flat[:5], flat[half - 3:half + 4], flat[k - 6:] = 8, 1, 0.5             # few enough that every sum is exact
    db = torch.empty(1, device=ctx.device)
    got = D.relative_position_backward(ctx, out, b, qp, key_positions=kp, bias_grad=db)
    assert got[:, 0].tolist() == [4 + 3.0, 32 + 3.0, 8.0] and float(db) == 50


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_position_matches_the_embedder(ctx, dt):
    """The embedder with every other weight zero adds the same rows to zeros."""
    from localfold_amd import device as D, synthetic as S
    w, f = S.synthetic_input_embedder(90, 2, 1, c_m=64, c_z=128, c_e=64)
    keep = ("relativePositionWeight", "relativePositionBias")
    w = {k: v if k in keep else np.zeros_like(v) for k, v in w.items()}
    dw = D.DeviceWeights(ctx.device)
    fd = {k: torch.as_tensor(np.ascontiguousarray(v, np.float32)).to(ctx.device) for k, v in f.items()}
    _, pair, _ = D.input_embedder(ctx, fd, D.input_embedder_weights(dw, w), 64, 128, 64, dt)
    got = D.relative_position(ctx, on(ctx, w[keep[0]].astype(np.float32)), D.clipped_boundaries(32, ctx.device),
                              fd["residueIndex"].to(torch.int32), bias=on(ctx, w[keep[1]].astype(np.float32)), dtype=dt)
    assert torch.equal(pair, got)


@pytest.mark.gpu
def test_position_gradient_by_differences(ctx):
    """The gradient of <out, grad> in the table and the bias is what backward gives: out is linear in both, so a
    difference over a step of one is the derivative, up to the rounding of the two outs."""
    from localfold_amd import device as D
    rng = np.random.default_rng(3)
    q, k, c = 20, 31, 6
    (qp, qs), (kp, ks) = chain(rng, q, True), chain(rng, k, True)
    b = D.log_boundaries(8, 16, ctx.device)
    where = dict(key_positions=on(ctx, kp), segments=on(ctx, qs), key_segments=on(ctx, ks))
    table = on(ctx, rng.integers(-8, 9, (9, c)).astype(np.float32))        # whole numbers: exact
    bias = on(ctx, rng.integers(-8, 9, c).astype(np.float32))
    grad = on(ctx, rng.integers(-8, 9, (q, k, c)).astype(np.float32))
    db = torch.empty(c, device=ctx.device)
    dt = D.relative_position_backward(ctx, grad, b, on(ctx, qp), bias_grad=db, **where)
    loss = lambda t, s: float((f64(D.relative_position(ctx, t, b, on(ctx, qp), bias=s, **where)) * f64(grad)).sum())
    l0 = loss(table, bias)
    for r in range(9):
        for ch in (0, c - 1):
            t = table.clone()
            t[r, ch] += 1
            assert loss(t, bias) - l0 == float(dt[r, ch])
    for ch in range(c):
        s = bias.clone()
        s[ch] += 1
        assert loss(table, s) - l0 == float(db[ch])


# ---- 4 bits --------------------------------------------------------------------------------------

def stream(rng, rows, c, dt, spread=1.0):
    x = rng.normal(size=(rows, c)) * np.exp(spread * rng.normal(size=(rows, 1))) + 0.3 * rng.normal(size=c)
    return torch.as_tensor(x).to(dt)


PACKS = [(1, 1), (1, 128), (3, 22), (17, 64), (50, 65), (33, 127), (129, 128), (64, 129), (200, 300), (128, 32), (31, 1000)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,c", PACKS)
def test_mx4_pack(ctx, dt, rows, c):
    from localfold_amd import device as D
    rng = np.random.default_rng(rows * 1000 + c)
    x = stream(rng, rows, c, dt)
    want, want_t = mx64(f64(x)), mx64(f64(x).T)
    sums = torch.empty(c, dtype=torch.float32, device=ctx.device)
    alone = D.mx4_pack(ctx, x.to(ctx.device))
    m, t = D.mx4_empty(rows, c, ctx.device), D.mx4_empty(c, rows, ctx.device)
    D.mx4_pack(ctx, x.to(ctx.device), out=m, transposed=t, sums=sums)
    only = D.mx4_empty(c, rows, ctx.device)
    D.mx4_pack(ctx, x.to(ctx.device), transposed=only)
    for name, p, w in (("alone", alone, want), ("out", m, want), ("transposed", t, want_t), ("only", only, want_t)):
        v, b = values_of(p)
        assert (v[:, :p.cols] == w).all(), name
        assert (v[:, p.cols:] == 0).all() and (b[:, p.cols:] != 255).all(), name
        assert (b.T[::32] == bytes64(f64(x) if p.rows == rows and p is not t and p is not only else f64(x).T)).all(), name
        for out_dt in TYPES:
            u = D.mx4_unpack(ctx, p, out_dt)
            assert torch.equal(u.cpu(), torch.as_tensor(w).to(out_dt)), (name, out_dt)
    close(sums, f64(x).sum(0), 2 * U * rows * np.abs(f64(x)).sum(0), torch.float32)


@pytest.mark.gpu
def test_mx4_special_values(ctx):
    from localfold_amd import device as D
    v = np.zeros((12, 64), np.float32)
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0]
    v[0, :8], v[0, 8:16] = ties, [-t for t in ties]
    v[1, :8] = np.nextafter(np.float32(ties), np.float32(0))
    v[1, 8:16] = np.nextafter(np.float32(ties), np.float32(9))      # past 6: the scale doubles
    v[2, 3], v[2, 40] = np.inf, 1.0
    v[3, 3], v[3, 40] = np.nan, 1.0
    v[4] = 1e-45                                                    # below every scale
    v[5, 0] = 3.0e38
    v[6, 0], v[6, 1] = 2.0 ** -126 * 6, 2.0 ** -128
    v[7, :32] = -0.0
    v[8, 0] = 3.4e38                                                # rounds up to 2^128
    v[9, 31], v[9, 32] = -np.inf, 7.0
    v[10] = np.linspace(-6, 6, 64)
    v[11] = np.linspace(-9e-39, 9e-39, 64)
    x = torch.as_tensor(v)
    for transposed in (False, True):
        if transposed:
            m = D.mx4_empty(12, 64, ctx.device)
            D.mx4_pack(ctx, x.t().contiguous().to(ctx.device), transposed=m)
        else:
            m = D.mx4_pack(ctx, x.to(ctx.device))
        want = mx64(v.astype(np.float64))
        got = values_of(m)[0][:, :64]
        assert np.array_equal(got, want, equal_nan=True), np.argwhere(~((got == want) | np.isnan(want)))[:5]
        with np.errstate(over="ignore"):
            assert np.array_equal(f64(D.mx4_unpack(ctx, m)), want.astype(np.float32), equal_nan=True)


@pytest.mark.gpu
def test_mx4_unpack_reads_any_scale(ctx):
    """Bytes 0 and 255 too, which pack writes for nothing finite."""
    from localfold_amd import device as D
    m = D.mx4_empty(256, 32, ctx.device)
    m.codes.copy_(torch.arange(256, device=ctx.device, dtype=torch.int32).to(torch.uint8)[:, None].expand(256, 64))
    m.scales.copy_(torch.arange(256, device=ctx.device, dtype=torch.int32).to(torch.uint8)[None].expand(4, 256))
    want = values_of(m)[0][:, :32]
    with np.errstate(over="ignore"):
        assert np.array_equal(f64(D.mx4_unpack(ctx, m)), want.astype(np.float32), equal_nan=True)


LINEARS = [(1, 128, 128), (1, 1, 1), (1, 4096, 300), (2, 200, 1000), (5, 22, 49), (16, 130, 64), (17, 1000, 65), (59, 384, 1536),
           (64, 64, 64), (100, 128, 512), (129, 512, 128), (300, 640, 640), (257, 65, 129), (1000, 256, 100), (33, 5000, 40)]


def linear_case(ctx, rng, rows, k, n, dt, spread=1.0):
    from localfold_amd import device as D
    x, w = stream(rng, rows, k, dt, spread), stream(rng, n, k, torch.float32, spread) / math.sqrt(k)
    return x.to(ctx.device), D.mx4_pack(ctx, w.to(ctx.device)), torch.as_tensor(rng.normal(size=n)).float().to(ctx.device)


def linear_bound(x, w, k, extra):
    """An instruction adds four groups' exact sums to its addend; a reduction is split into at most 1024 parts.  The
    bias and the residual are two additions more."""
    depth = 5 * math.ceil(k / 128) + 11
    return 2 * U * (depth * (np.abs(x) @ np.abs(w).T) + 3 * extra)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,n", LINEARS)
def test_mx4_linear(ctx, dt, rows, k, n):
    from localfold_amd import device as D
    rng = np.random.default_rng(rows * 100 + k + n)
    x, w, bias = linear_case(ctx, rng, rows, k, n, dt)
    xq, wq = mx64(f64(x)), values_of(w)[0][:, :k]
    res = stream(rng, rows, n, dt).to(ctx.device)
    pure = xq @ wq.T
    odt = TYPES[(rows + n) % 3]
    got = D.mx4_linear(ctx, x, w, dtype=odt)
    close(got, pure, linear_bound(xq, wq, k, 0), odt, "plain")
    kept = D.mx4_pack(ctx, x)
    assert torch.equal(D.mx4_linear(ctx, kept, w, dtype=odt), got)
    got = D.mx4_linear(ctx, x, w, bias, relu=True, residual=res)
    extra = np.abs(f64(bias)) + np.abs(f64(res)) + np.abs(pure)
    close(got, np.maximum(pure + f64(bias), 0) + f64(res), linear_bound(xq, wq, k, extra), dt, "all")
    into = res.clone()
    D.mx4_linear(ctx, kept, w, bias, relu=True, residual=into, out=into)
    assert torch.equal(into, got)


# Products of more outputs than one block a run of them takes: weights resident for 1, 2, 4 and 8 steps of 128 columns and
# 8 that do not fit, both sizes of streamed tiles, whole and ragged, odd numbers of steps.
MANY = [(3001, 100, 300), (3001, 200, 300), (3001, 500, 300), (3001, 1000, 300), (3040, 1024, 320), (2000, 900, 1500),
        (4000, 1100, 1100), (8200, 1100, 1000), (8192, 640, 1024), (5001, 100, 300)]
# Sums over 3, 2, 8, 11 and 19 parts, tiles that do not divide by the XCDs, numbers of outputs that do not divide by 4.
SPLIT = [(601, 4096, 523), (901, 4000, 701), (200, 9000, 203), (129, 12500, 261), (301, 20000, 71)]


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("rows,k,n", MANY + SPLIT)
def test_mx4_linear_many(ctx, dt, rows, k, n):
    test_mx4_linear(ctx, dt, rows, k, n)


@pytest.mark.gpu
def test_mx4_pack_of_many_rows(ctx):
    """A block walks down more than one tile of rows."""
    from localfold_amd import device as D
    rng = np.random.default_rng(9)
    x = stream(rng, 300001, 5, torch.bfloat16)
    m, t = D.mx4_empty(300001, 5, ctx.device), D.mx4_empty(5, 300001, ctx.device)
    sums = torch.empty(5, device=ctx.device)
    D.mx4_pack(ctx, x.to(ctx.device), out=m, transposed=t, sums=sums)
    assert (values_of(m)[0][:, :5] == mx64(f64(x))).all() and (values_of(t)[0][:, :300001] == mx64(f64(x).T)).all()
    # a thread's sum of at most 2 x 32 rows, four of them, then doubles
    close(sums, f64(x).sum(0), 2 * U * 70 * np.abs(f64(x)).sum(0), torch.float32)


@pytest.mark.gpu
def test_mx4_pack_beyond_the_cache(ctx):
    """307 MB, whose loads pass by the cache: the same codes and bytes as of a part of it, and exact sums of whole numbers."""
    from localfold_amd import device as D
    rows, c, part = 600001, 128, 128 * 41
    x = torch.randint(-7, 8, (rows, c), device=ctx.device, dtype=torch.int32).float()
    x *= torch.exp2(torch.randint(-3, 4, (rows, 1), device=ctx.device).float())
    m, t, sums = D.mx4_empty(rows, c, ctx.device), D.mx4_empty(c, rows, ctx.device), torch.empty(c, device=ctx.device)
    D.mx4_pack(ctx, x, out=m, transposed=t, sums=sums)
    for r0 in (0, rows // 128 * 128 - 128 * 40):
        some = x[r0:r0 + part].contiguous()
        n = some.shape[0]
        sm, st = D.mx4_empty(n, c, ctx.device), D.mx4_empty(c, n, ctx.device)
        D.mx4_pack(ctx, some, out=sm, transposed=st)
        assert torch.equal(m.codes[r0:r0 + n], sm.codes) and torch.equal(m.scales[:, r0:r0 + n], sm.scales[:, :n])
        assert torch.equal(t.codes[:, r0 // 2:r0 // 2 + st.codes.shape[1]], st.codes)
        assert torch.equal(t.scales[r0 // 32:r0 // 32 + st.scales.shape[0], :c], st.scales[:, :c])
    close(sums, f64(x.double().sum(0)), 2 * U * 400 * f64(x.abs().double().sum(0)), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n,k", [(1, 1, 1), (300, 128, 128), (1000, 64, 130), (5000, 22, 49), (20000, 128, 64), (9000, 300, 70)])
def test_mx4_weight_gradient(ctx, rows, n, k):
    """The three products and sums of a linear layer's backward pass."""
    from localfold_amd import device as D
    rng = np.random.default_rng(rows + n)
    dy, x = stream(rng, rows, n, torch.bfloat16).to(ctx.device), stream(rng, rows, k, torch.bfloat16).to(ctx.device)
    w = stream(rng, n, k, torch.float32).to(ctx.device)
    g, gt, xt, wt = (D.mx4_empty(a, b, ctx.device) for a, b in ((rows, n), (n, rows), (k, rows), (k, n)))
    db = torch.empty(n, device=ctx.device)
    D.mx4_pack(ctx, x, transposed=xt)
    D.mx4_pack(ctx, w, transposed=wt)
    D.mx4_pack(ctx, dy, out=g, transposed=gt, sums=db)
    dx, dw = D.mx4_linear(ctx, g, wt, dtype=torch.float32), D.mx4_linear(ctx, gt, xt, dtype=torch.float32)
    gq, wq = mx64(f64(dy)), mx64(f64(w).T)
    close(dx, gq @ wq.T, linear_bound(gq, wq, n, 0), torch.float32, "dx")
    gq, xq = mx64(f64(dy).T), mx64(f64(x).T)
    close(dw, gq @ xq.T, linear_bound(gq, xq, rows, 0), torch.float32, "dw")
    close(db, f64(dy).sum(0), 2 * U * rows * np.abs(f64(dy)).sum(0), torch.float32, "db")
    assert torch.equal(dw, D.mx4_linear(ctx, gt, xt, dtype=torch.float32))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(1, 512, 100), (40, 192, 200), (600, 128, 130), (300, 1344, 200)])
def test_mx4_linear_specials(ctx, rows, k, n):
    """A NaN or an infinity makes its group, and so its row, NaN; bytes behind the last row are not read into others;
    large groups that cancel leave what the small ones add up to."""
    from localfold_amd import device as D
    rng = np.random.default_rng(k)
    x, w, _ = linear_case(ctx, rng, rows, k, n, torch.float32)
    x[rows - 1, k - 1] = math.nan
    if rows > 2:
        x[1, 0] = math.inf
    kept = D.mx4_pack(ctx, x)
    kept.scales[:, rows:] = 255
    w.scales[:, n:] = 255
    want = mx64(f64(x)) @ values_of(w)[0][:, :k].T
    for src in (x, kept):
        got = f64(D.mx4_linear(ctx, src, w, dtype=torch.float32))
        assert np.array_equal(np.isnan(got), np.isnan(want))
        for r in {rows - 1, min(1, rows - 1)} if rows > 2 else {rows - 1}:
            assert np.isnan(got[r]).all()
    # whole numbers times 2^12 in one group, cancelling, and 1/2 to 6 in another
    v = np.zeros((max(rows, 1), k), np.float32)
    v[:, 0:16], v[:, 16:32] = 6 * 4096, -6 * 4096
    v[:, 32:64] = rng.choice(E2M1, size=(v.shape[0], 32))
    ones = torch.ones(n, k, device=ctx.device)
    got = D.mx4_linear(ctx, torch.as_tensor(v).to(ctx.device), D.mx4_pack(ctx, ones), dtype=torch.float32)
    assert (f64(got) == v[:, 32:64].astype(np.float64).sum(1, keepdims=True)).all()


@pytest.mark.gpu
def test_mx4_leaves_the_neighbours(ctx):
    """Nothing is written outside of codes, scales, sums and out, whatever their alignment."""
    from localfold_amd import device as D
    rng = np.random.default_rng(1)
    for rows, k, n in ((1, 100, 33), (50, 65, 70), (129, 300, 63)):
        x, w, bias = linear_case(ctx, rng, rows, k, n, torch.bfloat16)
        arena = torch.full((3 + rows * n + 7,), 7.0, dtype=torch.bfloat16, device=ctx.device)
        out = arena[3:3 + rows * n].view(rows, n)
        D.mx4_linear(ctx, x, w, bias, out=out)
        assert torch.equal(out, D.mx4_linear(ctx, x, w, bias))
        assert (arena[:3] == 7).all() and (arena[3 + rows * n:] == 7).all()
        shifted = torch.empty(rows * k + 1, dtype=torch.bfloat16, device=ctx.device)[1:].view(rows, k).copy_(x)
        assert torch.equal(out, D.mx4_linear(ctx, shifted, w, bias))
        a = torch.full((rows * -(-k // 128) * 64 + 64,), 99, dtype=torch.uint8, device=ctx.device)
        b = torch.full((-(-k // 128) * 4 * (-(-rows // 16) * 16) + 64,), 99, dtype=torch.uint8, device=ctx.device)
        m = D.Mx4(rows, k, a[:-64].view(rows, -1), b[:-64].view(-(-k // 128) * 4, -1))
        D.mx4_pack(ctx, x, out=m)
        assert (a[-64:] == 99).all() and (b[-64:] == 99).all()


# ---- orthogonalised updates ----------------------------------------------------------------------

SIDES = [(1, 1, 1), (1, 64, 256), (2, 5, 9), (3, 22, 70), (2, 130, 64), (1, 128, 128), (2, 128, 512), (1, 300, 129), (1, 257, 1000),
         (1, 16, 700), (5, 1, 40), (2, 384, 100), (1, 200, 150), (2, 66, 1001), (9, 700, 100), (1, 1, 2000), (40, 260, 390)]


def gradients(rng, shape, dt):
    r = max(1, min(shape[1:]) // 4)
    u = rng.normal(size=(shape[0], shape[1], r)) / np.arange(1, r + 1) @ rng.normal(size=(shape[0], r, shape[2]))
    return torch.as_tensor(1e-3 * (u + 0.1 * rng.normal(size=shape))).to(dt)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("batch,rows,cols", SIDES)
def test_orthogonalize(ctx, dt, batch, rows, cols):
    from localfold_amd import device as D
    x = gradients(np.random.default_rng(rows * 1000 + cols), (batch, rows, cols), dt)
    for steps, co in ((1, NS), (5, NS), (3, [(1.5, -0.5, 0.0), (2.0, -1.5, 0.5), NS])):
        got = D.orthogonalize(ctx, x.to(ctx.device), steps=steps, coefficients=co)
        for b in range(batch):
            want, bound = schulz64(f64(x[b]), steps, co)
            d = np.linalg.norm(f64(got[b]) - want)
            store = HALF[dt] * (np.linalg.norm(want) + bound) + TINY[dt] * math.sqrt(rows * cols)
            assert d <= bound + store, (steps, b, d, bound, store)
        same = x.to(ctx.device)
        assert D.orthogonalize(ctx, same, steps=steps, coefficients=co, out=same) is same and torch.equal(same, got)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,cols", [(128, 512), (300, 70), (100, 129)])
def test_orthogonalize_batches(ctx, rows, cols):
    """Many matrices take other kernels than few; both are within the bound."""
    from localfold_amd import device as D
    x = gradients(np.random.default_rng(rows), (200, rows, cols), torch.float32)
    many, few = D.orthogonalize(ctx, x.to(ctx.device)), D.orthogonalize(ctx, x[:3].to(ctx.device))
    for b in (0, 1, 2, 100, 199):
        want, bound = schulz64(f64(x[b]), 5)
        for got in (many[b], few[b]) if b < 3 else (many[b],):
            assert np.linalg.norm(f64(got) - want) <= bound + U * np.linalg.norm(want)


@pytest.mark.gpu
def test_orthogonalize_large(ctx):
    """Sums over parts, in tiles of 128: a step of a matrix whose bound is close."""
    from localfold_amd import device as D
    x = gradients(np.random.default_rng(1), (1, 1025, 2300), torch.float32)
    got = D.orthogonalize(ctx, x.to(ctx.device), steps=2)
    want, bound = schulz64(f64(x[0]), 2)
    assert np.linalg.norm(f64(got[0]) - want) <= bound + U * np.linalg.norm(want)


@pytest.mark.gpu
def test_orthogonalize_is_of_f32_precision(ctx):
    """Singular values over four decades: a step's own error stays at float32's level of the largest, so what five steps
    make of the small ones is right to within its growth, not to bf16's."""
    from localfold_amd import device as D
    rng = np.random.default_rng(5)
    for m, n in ((64, 256), (128, 512), (100, 130)):
        q1, _ = np.linalg.qr(rng.normal(size=(m, m)))
        q2, _ = np.linalg.qr(rng.normal(size=(n, m)))
        u = torch.as_tensor(q1 * np.logspace(0, -4, m) @ q2.T).float()
        got = f64(D.orthogonalize(ctx, u.to(ctx.device)))
        want, bound = schulz64(f64(u), 5)
        assert np.linalg.norm(got - want) <= min(bound, 2e-2)
        s = np.linalg.svd(got, compute_uv=False)
        assert s.max() < 1.3


@pytest.mark.gpu
def test_orthogonalize_extremes(ctx):
    """Zeros, one entry, squares that overflow or underflow f32, NaN in one matrix of a batch."""
    from localfold_amd import device as D
    z = torch.zeros(2, 40, 70, device=ctx.device)
    assert (D.orthogonalize(ctx, z) == 0).all()
    assert torch.isnan(D.orthogonalize(ctx, z, epsilon=0.0)).all()
    rng = np.random.default_rng(0)
    u = rng.normal(size=(3, 40, 70))
    for size in (1e37, 1e-30):
        x = torch.as_tensor(u * size).float()
        got = D.orthogonalize(ctx, x.to(ctx.device), epsilon=0.0)
        for b in range(3):
            want, bound = schulz64(f64(x[b]), 5, epsilon=0.0)
            assert np.linalg.norm(f64(got[b]) - want) <= bound + U * np.linalg.norm(want)
    x = torch.as_tensor(u).float()
    fine = D.orthogonalize(ctx, x.to(ctx.device))
    x[1, 3, 4] = math.nan
    got = D.orthogonalize(ctx, x.to(ctx.device))
    assert torch.equal(got[0], fine[0]) and torch.equal(got[2], fine[2]) and torch.isnan(got[1]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("wdt,gdt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("nesterov", [False, True])
def test_muon_step(ctx, wdt, gdt, nesterov):
    from localfold_amd import device as D
    rng = np.random.default_rng(7)
    for batch, rows, cols in ((2, 40, 70), (1, 130, 64), (3, 128, 128)):
        shape = batch, rows, cols
        g, w = gradients(rng, shape, gdt), torch.as_tensor(rng.normal(size=shape)).to(wdt)
        m = gradients(rng, shape, torch.float32)
        rate, decay, mu, scale = 0.25, 0.125, 0.9375, 3.0
        for momentum in (m, None):
            m64 = f64(g) if momentum is None else mu * f64(momentum) + f64(g)
            u = m64 if momentum is None or not nesterov else f64(g) + mu * m64
            args = dict(rate=rate, decay=decay, momentum_factor=mu, nesterov=nesterov, scale=scale)
            out = torch.empty_like(w, device=ctx.device)
            mo = torch.empty_like(m, device=ctx.device) if momentum is not None else None
            dev = lambda t: None if t is None else t.to(ctx.device)
            D.muon_step(ctx, dev(w), dev(g), dev(momentum), out=out, momentum_out=mo, **args)
            if momentum is not None:
                close(mo, m64, 4 * U * (np.abs(f64(m)) + np.abs(f64(g))), torch.float32, "momentum")
            for b in range(batch):
                o, bound = schulz64(u[b], 5)
                want = (1 - rate * decay) * f64(w[b]) - rate * scale * o
                # u itself is off by a few U, which the steps' growth (4 a step at most) carries on
                bound += 8 * U * 4.0 ** 5
                store = (HALF[wdt] + 3 * U) * (np.linalg.norm(f64(w[b])) + rate * scale * (np.linalg.norm(o) + bound))
                assert np.linalg.norm(f64(out[b]) - want) <= rate * scale * bound + store
            w2, m2 = dev(w), dev(momentum)
            assert D.muon_step(ctx, w2, dev(g), m2, **args) is w2
            assert torch.equal(w2, out) and (momentum is None or torch.equal(m2, mo))


# ---- together, streams, graphs, refusals ---------------------------------------------------------

def step_state(ctx, rng, n=40, c=64, h=128):
    from localfold_amd import device as D
    s = {"table": rng.normal(size=(9, c)) / 3, "w": rng.normal(size=(h, c)) / 8, "momentum": np.zeros((h, c))}
    s = {k: torch.as_tensor(v).float().to(ctx.device) for k, v in s.items()}
    s["boundaries"], s["positions"] = D.log_boundaries(8, 16, ctx.device), torch.arange(n, dtype=torch.int32, device=ctx.device)
    s["segments"] = (s["positions"] > n // 2).to(torch.int32)
    s["dy"] = torch.as_tensor(rng.normal(size=(n * n, h))).float().to(ctx.device)
    e = lambda a, b: D.mx4_empty(a, b, ctx.device)
    s.update(w4=e(h, c), w4t=e(c, h), xt=e(c, n * n), g=e(n * n, h), gt=e(h, n * n))
    s.update(pair=torch.empty(n, n, c, device=ctx.device), y=torch.empty(n, n, h, device=ctx.device),
             dx=torch.empty(n, n, c, device=ctx.device), dw=torch.empty(h, c, device=ctx.device), db=torch.empty(h, device=ctx.device),
             dt=torch.empty_like(s["table"]), w_new=torch.empty_like(s["w"]), m_new=torch.empty_like(s["momentum"]))
    return s


def training_step(ctx, s, scratch=None):
    """Positions, a 4-bit layer, its gradients, the table's, and the weight's update."""
    from localfold_amd import device as D
    where = dict(segments=s["segments"])
    D.relative_position(ctx, s["table"], s["boundaries"], s["positions"], out=s["pair"], **where)
    D.mx4_pack(ctx, s["w"], out=s["w4"], transposed=s["w4t"])
    D.mx4_pack(ctx, s["pair"], transposed=s["xt"])
    D.mx4_linear(ctx, s["pair"], s["w4"], out=s["y"], scratch=scratch)
    D.mx4_pack(ctx, s["dy"], out=s["g"], transposed=s["gt"], sums=s["db"], scratch=scratch)
    D.mx4_linear(ctx, s["g"], s["w4t"], out=s["dx"], scratch=scratch)
    D.mx4_linear(ctx, s["gt"], s["xt"], out=s["dw"], scratch=scratch)
    D.relative_position_backward(ctx, s["dx"], s["boundaries"], s["positions"], table_grad=s["dt"], scratch=scratch, **where)
    D.muon_step(ctx, s["w"], s["dw"], s["momentum"], out=s["w_new"], momentum_out=s["m_new"], scratch=scratch)
    return [s[k] for k in ("pair", "y", "db", "dx", "dw", "dt", "w_new", "m_new")]


@pytest.mark.gpu
def test_training_step_together(ctx):
    rng = np.random.default_rng(2)
    n, c, h = 40, 64, 128
    s = step_state(ctx, rng, n, c, h)
    pair, y, db, dx, dw, dt, w_new, m_new = (f64(t) for t in training_step(ctx, s))
    p, seg = s["positions"].cpu().numpy(), s["segments"].cpu().numpy()
    row = rows64(s["boundaries"].cpu().numpy(), p, p, seg, seg)
    assert (pair == f64(s["table"])[row]).all()
    x, wq, wqt = pair.reshape(-1, c), mx64(f64(s["w"])), mx64(f64(s["w"]).T)
    xq = mx64(x)
    close(y.reshape(-1, h), xq @ wq.T, linear_bound(xq, wq, c, 0), torch.float32)
    gq = mx64(f64(s["dy"]))
    close(dx.reshape(-1, c), gq @ wqt.T, linear_bound(gq, wqt, h, 0), torch.float32)
    gt, xt = mx64(f64(s["dy"]).T), mx64(x.T)
    close(dw, gt @ xt.T, linear_bound(gt, xt, n * n, 0), torch.float32)
    want, mags = np.zeros((9, c)), np.zeros((9, c))
    np.add.at(want, row.ravel(), dx.reshape(-1, c))
    np.add.at(mags, row.ravel(), np.abs(dx.reshape(-1, c)))
    close(dt, want, 2 * U * n * n * mags, torch.float32)
    assert (m_new == dw).all()                                  # momentum was zero
    o, bound = schulz64(1.95 * dw, 5)
    scale = 0.02 * math.sqrt(2)
    assert np.linalg.norm(w_new - f64(s["w"]) + scale * o) <= scale * (bound + 8 * U * 4 ** 5) + 4 * U * np.linalg.norm(w_new)


@pytest.mark.gpu
def test_training_step_other_stream(ctx):
    rng = np.random.default_rng(2)
    s = step_state(ctx, rng)
    want = [t.clone() for t in training_step(ctx, s)]
    torch.cuda.synchronize()
    stream = torch.cuda.Stream(ctx.device)
    for t in (s["w_new"], s["dt"], s["y"]):
        t.zero_()
    stream.wait_stream(torch.cuda.current_stream(ctx.device))
    with torch.cuda.stream(stream):
        ctx.bind_stream()
        got = training_step(ctx, s)
    ctx.bind_stream()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_two_contexts_at_once(ctx):
    """Steps of two contexts on two streams, interleaved, each with a workspace of its own."""
    from localfold_amd import device as D
    other = D.Context(0)
    streams = [torch.cuda.Stream(ctx.device) for _ in range(2)]
    states = [step_state(ctx, np.random.default_rng(k)) for k in range(2)]
    large = [torch.randn(2, 200, 300, device=ctx.device) for _ in range(2)]
    want = [[t.clone() for t in training_step(ctx, s)] + [D.orthogonalize(ctx, x)] for s, x in zip(states, large)]
    torch.cuda.synchronize()
    got = [None, None]
    try:
        for c, s in zip((ctx, other), streams):
            c.bind_stream(s)
        for _ in range(5):
            for k, c in enumerate((ctx, other)):
                with torch.cuda.stream(streams[k]):
                    got[k] = training_step(c, states[k]) + [D.orthogonalize(c, large[k])]
        torch.cuda.synchronize()
    finally:
        ctx.bind_stream()
        other.close()
    for a, b in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.gpu
def test_training_step_in_a_graph(ctx):
    """Two captured steps with scratch of their own, replayed in turn, with eager steps between that move the context's
    workspace."""
    from localfold_amd import capi, device as D
    rng = np.random.default_rng(4)
    cases = []
    large = torch.ones(200, 300, device=ctx.device)
    large_out = torch.empty_like(large)
    for _ in range(2):
        s = step_state(ctx, rng)
        n = s["positions"].shape[0]
        pairs = capi.lf_relative_pairs(n, n, None, None, 1, 1, s["boundaries"].shape[0], None)
        need = max(ctx.lib.lf_relative_position_backward_scratch(C.byref(pairs), 64), ctx.lib.lf_muon_scratch(1, 128, 64),
                   ctx.lib.lf_mx4_pack_scratch(n * n, 128), ctx.lib.lf_mx4_linear_scratch(n * n, 64, 128, 1),
                   ctx.lib.lf_mx4_linear_scratch(n * n, 128, 64, 0), ctx.lib.lf_mx4_linear_scratch(128, n * n, 64, 0))
        scratch = torch.empty(need, dtype=torch.uint8, device=ctx.device)
        training_step(ctx, s, scratch)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(g):
                ctx.bind_stream()
                with pytest.raises(capi.LocalfoldError, match="scratch"):
                    D.orthogonalize(ctx, large, out=large_out)
                with pytest.raises(capi.LocalfoldError, match="scratch"):
                    D.relative_position_backward(ctx, s["dx"], s["boundaries"], s["positions"], table_grad=s["dt"],
                                                 segments=s["segments"])
                training_step(ctx, s, scratch)
        finally:
            ctx.bind_stream()
        cases.append((g, s))
    for turn in range(4):
        for g, s in cases:
            s["table"] += 0.25
            s["dy"] *= 1.25
            s["w"] -= 0.125
            g.replay()
            torch.cuda.synchronize()
            got = [s[k].clone() for k in ("pair", "y", "db", "dx", "dw", "dt", "w_new", "m_new")]
            D.orthogonalize(ctx, torch.randn(4 * (turn + 1), 200, 256, device=ctx.device))      # moves the workspace
            want = training_step(ctx, s)
            torch.cuda.synchronize()
            assert all(torch.equal(p, q) for p, q in zip(got, want)), turn


@pytest.mark.gpu
def test_refusals(ctx):
    from localfold_amd import capi, device as D
    dev = ctx.device
    t = torch.zeros(4, 4, device=dev)
    b = D.clipped_boundaries(2, dev)
    pos = torch.arange(4, dtype=torch.int32, device=dev)
    table = torch.zeros(5, 4, device=dev)
    bad = lambda *e: pytest.raises(e or (ValueError, TypeError, capi.LocalfoldError))
    with bad(ValueError):
        D.relative_position(ctx, table[:4], b, pos)
    with bad(ValueError):
        D.relative_position(ctx, table, b, pos, segments=pos, key_positions=pos)
    with bad(ValueError):
        D.relative_position(ctx, table, b, pos, key_segments=pos)
    with bad(TypeError):
        D.relative_position(ctx, table, b, pos.long())
    with bad(TypeError):
        D.relative_position(ctx, table, b.float(), pos)
    with bad(TypeError):
        D.relative_position(ctx, table.double(), b, pos)
    with bad(ValueError):
        D.relative_position(ctx, table, b.cpu(), pos)
    with bad(ValueError):
        D.relative_position(ctx, table.t(), b, pos)
    with bad(ValueError):
        D.relative_position(ctx, table, b, pos, out=torch.zeros(4, 4, 5, device=dev))
    with bad(TypeError):
        D.relative_position(ctx, table, b, pos, out=torch.zeros(4, 4, 4, device=dev), pair=torch.zeros(4, 4, 4, device=dev).half())
    with bad(capi.LocalfoldError):
        D.relative_position(ctx, table, b, pos[:0])
    with bad(capi.LocalfoldError):
        D.relative_position(ctx, torch.zeros(5, 4097, device=dev), b, pos)
    with bad(capi.LocalfoldError):
        D.relative_position(ctx, torch.zeros(4098, 1, device=dev), torch.zeros(4097, dtype=torch.int32, device=dev), pos)
    with bad(ValueError):
        D.relative_position_backward(ctx, torch.zeros(4, 5, 4, device=dev), b, pos)
    with bad(capi.LocalfoldError):
        D.relative_position_backward(ctx, torch.zeros(4, 4, 4, device=dev), b, pos, scratch=torch.zeros(16, dtype=torch.uint8, device=dev))
    m = D.mx4_pack(ctx, t)
    with bad(ValueError):
        D.mx4_pack(ctx, t, out=D.mx4_empty(4, 5, dev))
    with bad(ValueError):
        D.mx4_pack(ctx, torch.zeros(4, 5, device=dev), transposed=D.mx4_empty(4, 5, dev))
    with bad(ValueError):
        D.mx4_pack(ctx, t, sums=torch.zeros(5, device=dev))
    with bad(TypeError):
        D.mx4_pack(ctx, t.double())
    with bad(ValueError):
        D.mx4_pack(ctx, t[:, ::2])
    with bad(ValueError):
        D.mx4_unpack(ctx, m, out=torch.zeros(4, 5, device=dev))
    with bad(ValueError):
        D.mx4_linear(ctx, torch.zeros(4, 5, device=dev), m)
    with bad(ValueError):
        D.mx4_linear(ctx, D.mx4_empty(4, 5, dev), m)
    with bad(ValueError):
        D.mx4_linear(ctx, t, m, bias=torch.zeros(5, device=dev))
    with bad(ValueError):
        D.mx4_linear(ctx, t, m, out=torch.zeros(4, 5, device=dev))
    with bad(ValueError):
        D.mx4_linear(ctx, t, D.mx4_empty(4, 4, "cpu"))
    with bad(capi.LocalfoldError):
        D.mx4_linear(ctx, D.Mx4(4, 4, torch.zeros(4, 65, dtype=torch.uint8, device=dev).view(-1)[1:257].view(4, 64),
                                m.scales), m)
    with bad(ValueError):
        D.orthogonalize(ctx, t[0])
    with bad(ValueError):
        D.orthogonalize(ctx, t.t()[:, :2])
    with bad(TypeError):
        D.orthogonalize(ctx, t.double())
    with bad(ValueError):
        D.orthogonalize(ctx, torch.zeros(0, 4, device=dev))
    with bad(capi.LocalfoldError):
        D.orthogonalize(ctx, torch.zeros(0, 4, 4, device=dev))
    with bad(capi.LocalfoldError):
        D.orthogonalize(ctx, torch.zeros(16385, 1, device=dev))
    with bad(capi.LocalfoldError):
        D.orthogonalize(ctx, t, epsilon=-1.0)
    for co in ((math.nan, 0, 0), (100.0, 0.0, 0.0), (3.0, 5.0, 7.0)):
        with bad(capi.LocalfoldError):
            D.orthogonalize(ctx, t, coefficients=co)
    with bad(ValueError):
        D.muon_step(ctx, t, torch.zeros(4, 5, device=dev))
    with bad(TypeError):
        D.muon_step(ctx, t, t, t.half())
    with bad(ValueError):
        D.muon_step(ctx, t, t, momentum_out=t)
    with bad(capi.LocalfoldError):
        D.muon_step(ctx, t, t, rate=math.inf)
    with bad(capi.LocalfoldError):
        D.muon_step(ctx, torch.zeros(200, 300, device=dev), torch.zeros(200, 300, device=dev),
                    scratch=torch.zeros(16, dtype=torch.uint8, device=dev))
    # what Python does not reach
    lib, h = ctx.lib, ctx.handle
    pairs = capi.lf_relative_pairs(4, 4, pos.data_ptr(), pos.data_ptr(), pos.data_ptr(), None, 4, b.data_ptr())
    a = capi.lf_relative_position_args(C.pointer(pairs), 4, 0, table.data_ptr(), None, 0, None, torch.zeros(64, device=dev).data_ptr())
    assert lib.lf_relative_position(h, C.byref(a)) == capi.LF_ERR_INVALID and b"segments" in lib.lf_last_error()
    k = capi.lf_mx4_pack_args(4, 4, 0, t.data_ptr())
    assert lib.lf_mx4_pack(h, C.byref(k)) == capi.LF_ERR_INVALID and b"no output" in lib.lf_last_error()
    l = capi.lf_mx4_linear_args(4, None, 0, None, m._pointer, None, 0, 0, None, t.data_ptr())
    assert lib.lf_mx4_linear(h, C.byref(l)) == capi.LF_ERR_INVALID
    l = capi.lf_mx4_linear_args(4, None, 7, t.data_ptr(), m._pointer, None, 0, 0, None, t.data_ptr())
    assert lib.lf_mx4_linear(h, C.byref(l)) == capi.LF_ERR_INVALID and b"dtypes" in lib.lf_last_error()
    o = capi.lf_orthogonalize_args(1, 4, 4, 0, t.data_ptr(), t.data_ptr(), 5, None, 1e-7)
    assert lib.lf_orthogonalize(h, C.byref(o)) == capi.LF_ERR_INVALID and b"coefficients" in lib.lf_last_error()
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_muon_step_refuses_factors_past_f32(ctx):
    """rate scale and 1 - rate decay are what the kernels multiply with: as infinities they would make NaN of zeros."""
    from localfold_amd import capi, device as D
    t = torch.zeros(4, 4, device=ctx.device)
    w = torch.ones(4, 4, device=ctx.device)
    for args in (dict(rate=1e30, scale=1e30), dict(rate=-1e20, scale=1e20), dict(rate=1e30, decay=1e30)):
        with pytest.raises(capi.LocalfoldError, match="finite"):
            D.muon_step(ctx, w, t, **args)
    assert (w == 1).all()
    D.muon_step(ctx, w, t, rate=1e30, decay=-1e-30, scale=1e8)
    assert (w == 2).all()

@pytest.mark.gpu
def test_documented_step_runs(ctx):
    """The example of these operators, as it stands, on tensors of the names that it uses."""
    rng = np.random.default_rng(11)
    n, c, outputs = 24, 40, 72
    rows = n * n
    t = lambda *shape: torch.as_tensor(rng.normal(size=shape)).float().to(ctx.device)
    from localfold_amd import device as D
    chains = (torch.arange(n, device=ctx.device) > 9).to(torch.int32)
    v = dict(table=t(66, c), positions=torch.arange(n, dtype=torch.int32, device=ctx.device), chains=chains, bias=t(c),
             weight=t(outputs, c), b=t(outputs), rows=rows, outputs=outputs, dout=t(rows, outputs), db=t(outputs), dpair=t(n, n, c),
             dbias=t(c), momentum=torch.zeros(outputs, c, device=ctx.device))
    v["wt"], v["xt"] = D.mx4_empty(c, outputs, ctx.device), D.mx4_empty(c, rows, ctx.device)
    D.mx4_pack(ctx, v["weight"], transposed=v["wt"])
    D.mx4_pack(ctx, t(rows, c), transposed=v["xt"])
    (code,) = [code for _, code in documented_examples() if "muon_step" in code]
    exec(code, v)
    torch.cuda.synchronize()
    v["ctx"].close()
    p, s = np.arange(n, dtype=np.int32), chains.cpu().numpy()
    row = rows64(np.arange(-31, 33), p, p, s, s)
    want, mags = np.zeros((66, c)), np.zeros((66, c))
    np.add.at(want, row.ravel(), f64(v["dpair"]).reshape(-1, c))
    np.add.at(mags, row.ravel(), np.abs(f64(v["dpair"])).reshape(-1, c))
    close(v["dtable"], want, 2 * U * rows * mags, torch.float32)
    close(v["dbias"], want.sum(0), 2 * U * rows * mags.sum(0), torch.float32)
    assert v["pair"].shape == (n, n, c) and v["out"].shape == (n, n, outputs) and torch.equal(v["momentum"], v["dw"])


# Where a block does not take a whole matrix, momentum and weights pass through other kernels: blocks of 128 columns (smaller
# side 65 to 128), wide, tall and of odd widths; products of tiles of 64 and of 128 (40 matrices), tall with whole and cut
# groups of four rows, narrow.
STEPS = [(2, 128, 512), (3, 300, 70), (1, 101, 257), (2, 1001, 66), (1, 200, 300), (1, 301, 150), (2, 16, 700), (40, 390, 260), (1, 1500, 9)]


@pytest.mark.gpu
@pytest.mark.parametrize("wdt,gdt", [(torch.float32, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float16, torch.float16)])
@pytest.mark.parametrize("nesterov", [False, True])
@pytest.mark.parametrize("batch,rows,cols", STEPS)
def test_muon_step_of_larger_matrices(ctx, batch, rows, cols, wdt, gdt, nesterov):
    from localfold_amd import device as D
    rng = np.random.default_rng(rows * 1000 + cols)
    shape = batch, rows, cols
    g, w = gradients(rng, shape, gdt).to(ctx.device), torch.as_tensor(rng.normal(size=shape)).to(wdt).to(ctx.device)
    m = gradients(rng, shape, torch.float32).to(ctx.device)
    rate, decay, mu, scale = 0.25, 0.125, 0.9375, 3.0                   # exact in every type
    args = dict(rate=rate, decay=decay, momentum_factor=mu, nesterov=nesterov, scale=scale)
    for momentum in (m, None):
        out, mo = torch.empty_like(w), None if momentum is None else torch.empty_like(m)
        kept = [t.clone() for t in (w, g, m)]
        D.muon_step(ctx, w, g, momentum, out=out, momentum_out=mo, **args)
        assert all(torch.equal(a, b) for a, b in zip((w, g, m), kept))  # none of the inputs is written
        m64 = f64(g) if momentum is None else mu * f64(m) + f64(g)
        if momentum is not None:
            close(mo, m64, 4 * U * (np.abs(f64(m)) + np.abs(f64(g))), torch.float32, "momentum")
        u = m64 if momentum is None or not nesterov else f64(g) + mu * m64
        for b in sorted({0, batch // 2, batch - 1}):
            o, bound = schulz64(u[b], 5)
            want = (1 - rate * decay) * f64(w[b]) - rate * scale * o
            # u itself is off by a few U, which the steps' growth (4 a step at most) carries on
            bound += 8 * U * 4.0 ** 5
            store = (HALF[wdt] + 3 * U) * (np.linalg.norm(f64(w[b])) + rate * scale * (np.linalg.norm(o) + bound))
            assert np.linalg.norm(f64(out[b]) - want) <= rate * scale * bound + store, b
        w2, m2 = w.clone(), None if momentum is None else m.clone()
        assert D.muon_step(ctx, w2, g, m2, **args) is w2
        assert torch.equal(w2, out) and (momentum is None or torch.equal(m2, mo))


@pytest.mark.gpu
def test_muon_step_in_place_in_graphs(ctx):
    """Steps in place of both kinds that use scratch, captured with scratch of their own and replayed in turn, with eager
    ones between that move the context's workspace."""
    from localfold_amd import device as D
    rng = np.random.default_rng(12)
    cases = []
    for shape in ((3, 128, 512), (2, 300, 200)):
        w, m = torch.as_tensor(rng.normal(size=shape)).float().to(ctx.device), torch.zeros(shape, device=ctx.device)
        g = gradients(rng, shape, torch.float32).to(ctx.device)
        scratch = torch.empty(ctx.lib.lf_muon_scratch(*shape), dtype=torch.uint8, device=ctx.device)
        D.muon_step(ctx, w, g, m, decay=0.1, scratch=scratch)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        try:
            with torch.cuda.graph(graph):
                ctx.bind_stream()
                D.muon_step(ctx, w, g, m, decay=0.1, scratch=scratch)
        finally:
            ctx.bind_stream()
        cases.append((graph, w, g, m, w.clone(), m.clone(), scratch))
    for turn in range(4):
        for graph, w, g, m, w2, m2, _ in cases:
            g *= -0.75
            graph.replay()
            torch.cuda.synchronize()
            D.orthogonalize(ctx, torch.randn(4 * (turn + 1), 200, 256, device=ctx.device))
            D.muon_step(ctx, w2, g, m2, decay=0.1)
            torch.cuda.synchronize()
            assert torch.equal(w, w2) and torch.equal(m, m2), turn


@pytest.mark.gpu
def test_muon_steps_of_two_contexts_at_once(ctx):
    from localfold_amd import device as D
    other = D.Context(0)
    streams = [torch.cuda.Stream(ctx.device) for _ in range(2)]
    shapes = ((3, 128, 512), (2, 300, 200))
    state = [[(torch.as_tensor(rng.normal(size=s)).float().to(ctx.device), gradients(rng, s, torch.float32).to(ctx.device),
               torch.zeros(s, device=ctx.device)) for s in shapes] for rng in (np.random.default_rng(k) for k in (13, 14))]
    want = [[[t.clone() for t in part] for part in s] for s in state]
    for s in want:
        for _ in range(4):
            for w, g, m in s:
                D.muon_step(ctx, w, g, m, decay=0.1)
    torch.cuda.synchronize()
    try:
        for c, s in zip((ctx, other), streams):
            c.bind_stream(s)
        for _ in range(4):
            for k, c in enumerate((ctx, other)):
                with torch.cuda.stream(streams[k]):
                    for w, g, m in state[k]:
                        D.muon_step(c, w, g, m, decay=0.1)
        torch.cuda.synchronize()
    finally:
        ctx.bind_stream()
        other.close()
    for a, b in zip(state, want):
        assert all(torch.equal(p, q) for x, y in zip(a, b) for p, q in zip(x, y))


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("q,k,c,reach", [(3, 5, 4096, 2), (2, 40, 2051, 4), (70, 60, 2304, 1)])
def test_position_of_wide_rows(ctx, q, k, c, reach, dt):
    """Rows of more chunks of channels than a block has threads, and of 32 slices of channels in the gradient."""
    for segments in (False, True):
        test_position(ctx, q, k, c, reach, dt, segments)
        test_position_backward(ctx, q, k, c, reach, dt, segments)


def edges(dt):
    """Rows of 64 at the edges of a type: ties of every code and their neighbours, subnormals, the largest values."""
    big, small = torch.finfo(dt).max, torch.finfo(dt).smallest_normal * torch.finfo(dt).eps      # the smallest subnormal
    ties = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=dt)
    v = torch.zeros(12, 64, dtype=dt)
    for r, size in enumerate((1.0, 2.0 ** -10, 2.0 ** 10)):
        v[r, :8], v[r, 8:16], v[r, 32:40], v[r, 40:48] = (t * size for t in (ties, -ties, torch.nextafter(ties, ties * 0), -torch.nextafter(ties, ties * 0)))
    k = torch.arange(1, 65).double() * small
    v[3], v[4], v[5] = k.to(dt), -(k * 7).to(dt), (k.flip(0) * 31).to(dt)
    v[6, 0], v[6, 1], v[6, 32] = big, -big / 4, -big
    v[7] = small
    v[8, ::2] = torch.finfo(dt).smallest_normal
    v[8, 1::2] = -3 * small
    v[9, 5], v[9, 40] = math.inf, 1.0
    v[10, 63], v[10, 0] = math.nan, -1.0
    v[11] = -0.0
    return v


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
def test_mx4_edges_of_every_type(ctx, dt):
    """The same codes and bytes whichever way a matrix is packed, and products of them whether packed before or inside."""
    from localfold_amd import device as D
    v = edges(dt)
    x, want = v.to(ctx.device), mx64(f64(v))
    out, tr, alone = D.mx4_empty(12, 64, ctx.device), D.mx4_empty(12, 64, ctx.device), D.mx4_pack(ctx, x)
    D.mx4_pack(ctx, x, out=out, transposed=D.mx4_empty(64, 12, ctx.device))
    D.mx4_pack(ctx, x.t().contiguous(), transposed=tr)
    for name, m in (("alone", alone), ("both", out), ("transposed", tr)):
        got = values_of(m)[0][:, :64]
        assert np.array_equal(got, want, equal_nan=True), (name, np.argwhere(~((got == want) | np.isnan(want)))[:6].tolist())
    eye = torch.zeros(64, 64, device=ctx.device).fill_diagonal_(1.0)
    w = D.mx4_pack(ctx, eye)
    for rows in (12, 24, 12 * 3000):                 # few rows, two tiles of them, weights resident
        many = x.repeat(rows // 12, 1)
        got = f64(D.mx4_linear(ctx, many, w, dtype=torch.float32))
        with np.errstate(over="ignore"):
            # 0 times NaN is NaN: a group that holds one makes its whole row so
            full = np.where(np.isnan(want).any(1, keepdims=True), np.nan, want).astype(np.float32)
        assert np.array_equal(got[:12], full, equal_nan=True), (rows, np.argwhere(~((got[:12] == full) | np.isnan(full)))[:6].tolist())
        assert np.array_equal(got, np.tile(got[:12], (rows // 12, 1)), equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(3, 200, 40), (100, 200, 100), (6000, 200, 100), (600, 4096, 530), (8192, 640, 1024)])
def test_mx4_linear_far_exponents(ctx, rows, k, n):
    """Operands times powers of two that cancel or carry the product far: the same bits, shifted."""
    from localfold_amd import device as D
    rng = np.random.default_rng(rows + k)
    x, w = stream(rng, rows, k, torch.float32).to(ctx.device), stream(rng, n, k, torch.float32).to(ctx.device)
    base = D.mx4_linear(ctx, x, D.mx4_pack(ctx, w), dtype=torch.float32)
    for a, b in ((100, -100), (-100, 100), (110, -20), (-20, 110), (-40, -40), (40, 40), (-110, 120)):
        got = D.mx4_linear(ctx, x * 2.0 ** a, D.mx4_pack(ctx, w * 2.0 ** b), dtype=torch.float32)
        assert torch.equal(got, base * 2.0 ** (a + b)), (a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", [(2, 40, 70), (2, 128, 512), (1, 300, 200)])
def test_orthogonalize_far_below_epsilon(ctx, batch, rows, cols):
    """A norm far below epsilon: elements are kept to 2^-38 at the start and after each step, whatever the norm, and a
    difference grows by a = 3.4445 a step at most; beside that f32's relative errors, a 2^-20 a step with the roundings of P."""
    from localfold_amd import device as D
    u = np.random.default_rng(rows).normal(size=(batch, rows, cols))
    u /= np.linalg.norm(u, axis=(1, 2), keepdims=True)
    for size in (2.0 ** -8, 2.0 ** -20, 2.0 ** -45):
        x = torch.as_tensor(u * EPS * size).float()
        got = D.orthogonalize(ctx, x.to(ctx.device))
        for b in range(batch):
            want, _ = schulz64(f64(x[b]), 5)
            kept = sum(NS[0] ** k for k in range(6)) * math.sqrt(rows * cols) * 2.0 ** -38
            assert np.linalg.norm(f64(got[b]) - want) <= kept + 6 * 2.0 ** -20 * np.linalg.norm(want), (size, b)


@pytest.mark.gpu
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("q,k,c,reach", [(30, 33, 12, 2047), (400, 400, 128, 64)])
def test_position_of_large_tables(ctx, q, k, c, reach, dt):
    """4094 boundaries, of 4095 that may be given; and a table that LDS does not hold, of many pairs."""
    for segments in (False, True):
        test_position(ctx, q, k, c, reach, dt, segments)
        test_position_backward(ctx, q, k, c, reach, dt, segments)


@pytest.mark.gpu
def test_position_of_the_most_boundaries(ctx):
    from localfold_amd import device as D
    p = np.arange(-4200, 4200, 3).astype(np.int32)
    b = (2 * np.arange(4095) - 4095).astype(np.int32)
    zero = np.zeros(1, np.int32)
    row = rows64(b, p, zero)[:, 0]
    table = torch.arange(4096, dtype=torch.float32, device=ctx.device)[:, None].contiguous()
    got = D.relative_position(ctx, table, on(ctx, b), on(ctx, p), key_positions=on(ctx, zero))
    assert (f64(got)[:, 0, 0] == row).all()
    dt = D.relative_position_backward(ctx, torch.ones_like(got), on(ctx, b), on(ctx, p), key_positions=on(ctx, zero))
    assert (f64(dt)[:, 0] == np.bincount(row, minlength=4096)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", [(2, 40, 70), (3, 128, 512), (1, 300, 200)])
def test_orthogonalize_of_the_most_steps(ctx, batch, rows, cols):
    """32 steps, a triple each, that bring every singular value to one: what is left is the polar factor.

    A step keeps that factor; its rounding E, as schulz64 counts it, changes it by at most 2 |E| over the smallest singular
    value of the step's result."""
    from localfold_amd import device as D
    x = torch.as_tensor(np.random.default_rng(cols).normal(size=(batch, rows, cols))).float()
    co = [(1.5, -0.5, 0.0), (1.875, -1.25, 0.375)] * 16
    got = f64(D.orthogonalize(ctx, x.to(ctx.device), steps=32, coefficients=co))
    m, n = sorted((rows, cols))
    gamma = lambda k: 2.0 ** -21 + 3 * (k / 32 + 8) * 2 * U
    for i in range(batch):
        u, s, vt = np.linalg.svd(f64(x[i]), full_matrices=False)
        s = s / (np.linalg.norm(s) + EPS)
        bound = 2 * 4 * U / s.min()
        for a, b, c in co:
            f, p = np.linalg.norm(s), a + b * s ** 2 + c * s ** 4
            dp = (abs(b) + 2 * abs(c) * s.max() ** 2) * gamma(n) * f * f + gamma(m) * abs(c) * np.linalg.norm(s ** 2) ** 2 + 2.0 ** -21 * np.linalg.norm(p)
            e = s.max() * dp + gamma(m) * np.linalg.norm(p) * f
            s = p * s
            bound += 2 * (e + 2.0 ** -21 * np.linalg.norm(s)) / s.min()
        assert np.abs(s - 1).max() < 1e-12 and bound < 0.1 * math.sqrt(m)
        assert np.linalg.norm(got[i] - u @ vt) <= bound + U * math.sqrt(m)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,k,n", [(17000005, 128, 130), (2000001, 1100, 1080)])
def test_mx4_past_four_gigabytes(ctx, rows, k, n):
    """Activations and outputs past 2^32 bytes, by weights resident and streamed: rows at the end as in a call of their own."""
    from localfold_amd import device as D
    x = torch.empty(rows, k, dtype=torch.bfloat16, device=ctx.device).normal_()
    w = D.mx4_pack(ctx, torch.randn(n, k, device=ctx.device))
    out = D.mx4_linear(ctx, x, w)
    kept, t, sums = D.mx4_empty(rows, k, ctx.device), D.mx4_empty(k, rows, ctx.device), torch.empty(k, device=ctx.device)
    D.mx4_pack(ctx, x, out=kept, transposed=t, sums=sums)
    assert torch.equal(D.mx4_linear(ctx, kept, w), out)
    for r0 in (0, rows // 256 * 256 - 256 * 200):
        part = x[r0:r0 + 256 * 200 + 100].contiguous()
        m = part.shape[0]
        pk, pt = D.mx4_empty(m, k, ctx.device), D.mx4_empty(k, m, ctx.device)
        D.mx4_pack(ctx, part, out=pk, transposed=pt)
        assert torch.equal(D.mx4_linear(ctx, part, w), out[r0:r0 + m])
        assert torch.equal(pk.codes, kept.codes[r0:r0 + m]) and torch.equal(pk.scales[:, :m], kept.scales[:, r0:r0 + m])
        whole = m // 32 * 32                                # the part's last group of rows may be cut
        assert torch.equal(pt.codes[:, :whole // 2], t.codes[:, r0 // 2:(r0 + whole) // 2])
        assert torch.equal(pt.scales[:whole // 32, :k], t.scales[r0 // 32:(r0 + whole) // 32, :k])
    want, mags = torch.zeros(k, dtype=torch.float64, device=ctx.device), torch.zeros(k, dtype=torch.float64, device=ctx.device)
    for some in x.split(1000000):
        want += some.double().sum(0)
        mags += some.double().abs().sum(0)
    # 32 rows of a tile, then a run's tiles of 128 rows (2048 runs of all columns, the last one shorter), then doubles
    depth = 32 + 4 + math.ceil(rows / 128 / (2048 // -(-k // 128)))
    close(sums, f64(want), 2 * U * depth * f64(mags), torch.float32)


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", [(60000, 128, 300), (2800, 700, 1100)])
def test_orthogonalize_past_eight_gigabytes(ctx, batch, rows, cols):
    """More than 2^31 elements, a block a matrix and in products, written in place."""
    from localfold_amd import device as D
    x = torch.empty(batch, rows, cols, device=ctx.device).normal_()
    some = {b: x[b].clone() for b in (0, batch // 2, batch - 1)}
    D.orthogonalize(ctx, x, steps=2, out=x)
    for b, u in some.items():
        want, bound = schulz64(f64(u), 2)
        assert np.linalg.norm(f64(x[b]) - want) <= bound + U * np.linalg.norm(want), b


def test_muon_scratch_of_the_kinds():
    """Panels keep 192 KB for each 128 columns and 8 KB a matrix, blocks of their own nothing: panels where there are at least
    three of a matrix, and a CU for each of all of them."""
    from localfold_amd import capi
    lib = capi.load()
    for batch, rows, cols, panels in ((64, 128, 512, 4), (65, 128, 512, 0), (85, 70, 300, 3), (86, 300, 70, 0), (1, 128, 256, 0), (128, 256, 66, 0),
                                      (32, 128, 1024, 8), (3, 64, 512, 0), (1, 128, 385, 4)):
        need = lib.lf_muon_scratch(batch, rows, cols)
        assert need == (batch * (8192 + panels * 196608) if panels else 0), (batch, rows, cols)
    assert lib.lf_muon_scratch(33, 128, 1024) > 33 * 128 * 1024 * 16       # products: X and its transpose twice


@pytest.mark.gpu
@pytest.mark.parametrize("batch,rows,cols", [(64, 128, 512), (65, 128, 512), (85, 300, 70), (86, 70, 300), (1, 128, 256), (33, 128, 1024)])
def test_orthogonalize_on_both_sides_of_the_rule(ctx, batch, rows, cols):
    from localfold_amd import device as D
    x = gradients(np.random.default_rng(batch), (batch, rows, cols), torch.bfloat16).to(ctx.device)
    got = D.orthogonalize(ctx, x)
    for b in sorted({0, batch // 2, batch - 1}):
        want, bound = schulz64(f64(x[b]), 5)
        assert np.linalg.norm(f64(got[b]) - want) <= bound + HALF[torch.bfloat16] * (np.linalg.norm(want) + bound), b
