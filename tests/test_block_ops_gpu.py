"""Rotary positions and the residual norm on a B200, against their formulas in 64 bits.

Tolerances count roundings: u = 2^-24 is half a step of fp32, and an output of type t is off by at
most eps(t) / 2 of its value more."""

import threading

import pytest
import torch

from tests.conftest import pkg

pytestmark = pytest.mark.gpu

DEV = "cuda"
U = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def ops():
    return pkg("ops")


@pytest.fixture(autouse=True)
def no_device_error():
    """No wait of a kernel ran out."""
    yield
    pkg("device").Context.get(0).sync()


def randn(seed, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale + shift).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rel(got, ref):
    got, ref = got.double(), ref.double()
    return ((got - ref).norm() / ref.norm().clamp_min(1e-300)).item()


# ----------------------------------------------------------------------------- rotary

def rotary_ref(x, H, D, inv, pos, m, interleaved, inverse):
    """(y, |x0| + |x1| of each element's pair) in 64 bits."""
    R = 2 * inv.numel()
    x3 = x[:, :H * D].double().reshape(-1, H, D)
    ang = pos.double()[:, None, None] * inv
    c, s = ang.cos() * m, ang.sin() * m * (-1.0 if inverse else 1.0)
    a = x3[..., :R]
    x0, x1 = (a[..., 0::2], a[..., 1::2]) if interleaved else (a[..., :R // 2], a[..., R // 2:])
    parts = [x0 * c - x1 * s, x1 * c + x0 * s], [x0.abs() + x1.abs()] * 2
    put = (lambda p: torch.stack(p, -1).flatten(-2)) if interleaved else (lambda p: torch.cat(p, -1))
    y = torch.cat([put(parts[0]), x3[..., R:]], -1)
    mag = torch.cat([put(parts[1]), torch.zeros_like(x3[..., R:])], -1)
    return y.reshape(x.shape[0], -1), mag.reshape(x.shape[0], -1)


def check_rotary(got, ref, mag, m):
    # cos and sin: the fraction of a turn rounds once (relative 2^-24, at most pi 2^-24 in the angle),
    # the function 2 steps, m once: below 8 u each; two products and a sum: 3 u more; then the output
    y, tol = got.double(), 11 * U * m * mag + half_step(got.dtype) * ref.abs() * (1 + 1e-3)
    if got.dtype == torch.float16:
        tol = tol + 2.0 ** -25  # below 2^-14 its steps no longer shrink
    assert bool(((y - ref).abs() <= tol).all()), ((y - ref).abs() - tol).max().item()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,Hq,Hk,D,R", [(1, 1, 1, 64, 64), (77, 16, 8, 128, 128), (33, 9, 1, 128, 64),
                                             (5, 3, 2, 20, 12), (7, 2, 1, 7, 2), (130, 4, 0, 64, 20), (9, 8, 11, 80, 32)])
def test_rotary(ops, dtype, interleaved, rows, Hq, Hk, D, R):
    inv, m = ops.rotary_freqs(R, scaling="yarn", factor=4.0)
    g = torch.Generator(device=DEV).manual_seed(rows)
    pos = torch.randint(0, 2 ** 17, (rows,), generator=g, device=DEV, dtype=torch.int32)
    q = randn(1, rows, Hq * D, dtype=dtype)
    k = randn(2, rows, Hk * D, dtype=dtype) if Hk else None
    for inverse in (False, True):
        got = ops.rotary(q, k, inv, Hq=Hq, Hk=Hk, D=D, positions=pos, mscale=m, interleaved=interleaved, inverse=inverse)
        for x, y, H in ((q, got[0], Hq), (k, got[1], Hk)):
            if x is None:
                assert y is None
                continue
            check_rotary(y, *rotary_ref(x, H, D, inv, pos, m, interleaved, inverse), m)


def test_rotary_far_positions_and_their_sign(ops):
    """Angles hold at the ends of int32: in 64 bits 2^31 turns x frequency leave 2^-22 of a turn."""
    inv, _ = ops.rotary_freqs(64)
    pos = torch.tensor([2 ** 31 - 1, -2 ** 31, -1, 0, 10 ** 9], dtype=torch.int32, device=DEV)
    q = randn(3, 5, 64)
    y, _ = ops.rotary(q, None, inv, Hq=1, D=64, positions=pos)
    ref, mag = rotary_ref(q, 1, 64, inv, pos, 1.0, False, False)
    # the reference's own angle, 2^31 rounded to 53 bits, is off by up to 2^-22, and so may be ours
    assert bool(((y.double() - ref).abs() <= (11 * U + 2.0 ** -21) * mag + half_step(torch.float32) * ref.abs()).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_rotary_offset_items_strides_in_place(ops, dtype):
    inv, _ = ops.rotary_freqs(128, 1e6)
    rows, L, H, D = 66, 33, 4, 128
    wide = randn(4, rows, 3 * H * D + 8, dtype=dtype)
    before = wide.clone()
    q, k = wide[:, :H * D], wide[:, H * D:2 * H * D]
    pos = (1000 + torch.arange(rows, device=DEV) % L).to(torch.int32)
    refs = [rotary_ref(x.clone(), H, D, inv, pos, 1.0, False, False) for x in (q, k)]
    out = ops.rotary(q, k, inv, Hq=H, Hk=H, D=D, offset=1000, rows_per_item=L, out_q=q, out_k=k)
    assert out[0] is q and out[1] is k
    for x, (ref, mag) in zip((q, k), refs):
        check_rotary(x, ref, mag, 1.0)
    assert torch.equal(wide[:, 2 * H * D:], before[:, 2 * H * D:])  # neighbours are left as they were
    # a base that is not 16-byte aligned takes the elementwise form: the same bits
    odd = torch.empty(rows, H * D + 1, dtype=dtype, device=DEV)
    odd[:, 1:] = before[:, :H * D]
    assert torch.equal(ops.rotary(odd[:, 1:], None, inv, Hq=H, D=D, positions=pos)[0], q)


def test_rotary_in_place_of_a_part_leaves_the_rest(ops):
    inv, m = ops.rotary_freqs(32, scaling="yarn", factor=2.0)
    q = randn(5, 10, 2 * 64, dtype=torch.bfloat16)
    ref = ops.rotary(q, None, inv, Hq=2, D=64, mscale=m)[0]
    ops.rotary(q, None, inv, Hq=2, D=64, mscale=m, out_q=q)
    assert torch.equal(q, ref)


def test_rotary_inverse_undoes_and_is_the_gradient(ops):
    inv, m = ops.rotary_freqs(48, scaling="yarn", factor=8.0)
    q, w = randn(6, 50, 3 * 64), randn(7, 50, 3 * 64)
    kw = dict(Hq=3, D=64, mscale=m, interleaved=True, offset=12345)
    y = ops.rotary(q, None, inv, **kw)[0]
    gw = ops.rotary(w, None, inv, inverse=True, **kw)[0]
    # <w, J q> = <J^T w, q>
    a, b = (w.double() * y.double()).sum(), (gw.double() * q.double()).sum()
    assert abs(a - b) <= 30 * U * (w.double() * y.double()).abs().sum()
    back = ops.rotary(y, None, inv, inverse=True, **kw)[0].view(50, 3, 64).double()
    q3 = q.view(50, 3, 64).double()
    assert rel(back[..., :48], q3[..., :48] * m * m) < 30 * U
    assert torch.equal(back[..., 48:], q3[..., 48:])


def test_rotary_empty_and_long_strides(ops):
    inv, _ = ops.rotary_freqs(64)
    e = torch.empty(0, 64, device=DEV)
    assert ops.rotary(e, None, inv, Hq=1, D=64)[0].shape == (0, 64)
    # rows 2^31 + 64 elements apart: offsets past 32 bits
    ld = 2 ** 31 + 64
    buf = torch.empty(ld + 64, dtype=torch.float16, device=DEV)
    q = buf.as_strided((2, 64), (ld, 1))
    x = randn(8, 2, 64, dtype=torch.float16)
    q.copy_(x)
    ref = ops.rotary(x, None, inv, Hq=1, D=64, offset=5)[0]
    ops.rotary(q, None, inv, Hq=1, D=64, offset=5, out_q=q)
    assert torch.equal(q, ref)


def test_rotary_refusals_of_the_library(ops):
    err = pkg("device").AnimaError
    inv, _ = ops.rotary_freqs(64)
    q = randn(9, 4, 64)
    with pytest.raises(err, match="rotated of"):
        ops.rotary(q, None, inv, Hq=2, D=32)
    with pytest.raises(err, match="stride"):
        ops.rotary(q[:1].expand(4, 64), None, inv, Hq=1, D=64)


# ----------------------------------------------------------------------------- residual norm

def normalise(x, kind, eps):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    return x / (x.square().mean(-1, keepdim=True) + eps).sqrt()


def norm_ref(p, c):
    """x_out and h in 64 bits from 64-bit leaves p; c: post, pre, alpha, eps, L."""
    rows = p["y"].shape[0]
    item = torch.arange(rows, device=DEV) // c["L"]
    u = p["y"] if c["post"] is None else normalise(p["y"], c["post"], c["eps"])
    u = u * p["post_w"] if p.get("post_w") is not None else u
    u = u * p["gate"][item] if p.get("gate") is not None else u
    x = p["x"] + c["alpha"] * u
    return x, norm_h(x, p, c, item)


def norm_h(x, p, c, item):
    h = normalise(x, c["pre"], c["eps"])
    h = h * p["pre_w"] if p.get("pre_w") is not None else h
    h = h * (1 + p["scale"][item]) if p.get("scale") is not None else h
    return h + p["shift"][item] if p.get("shift") is not None else h


def make_norm(rows, C, L, post, pre, full, xd, yd, hd, seed=0):
    items = rows // L
    t = {"x": randn(seed + 1, rows, C, dtype=xd, scale=2.0, shift=0.5), "y": randn(seed + 2, rows, C, dtype=yd),
         "dh": randn(seed + 3, rows, C, dtype=hd), "dx_out": randn(seed + 4, rows, C, dtype=xd)}
    mods = randn(seed + 5, items, 3 * C, scale=0.3) if full else None
    for i, n in enumerate(("shift", "scale", "gate")):
        t[n] = mods[:, i * C:(i + 1) * C] if full else None
    t["post_w"] = randn(seed + 6, C, scale=0.1, shift=1.0) if post and full else None
    t["pre_w"] = randn(seed + 7, C, scale=0.1, shift=1.0) if full else None
    c = {"post": post, "pre": pre, "alpha": 0.75 if full else 1.0, "eps": 1e-6, "L": L}
    return t, c


PARAMS = ("gate", "post_w", "pre_w", "scale", "shift")


def kwargs(t, c):
    return dict(alpha=c["alpha"], post=c["post"], pre=c["pre"], eps=c["eps"], rows_per_item=c["L"],
                **{n: t[n] for n in PARAMS})


def grad_refs(t, c, dx_out=True):
    """The gradients by automatic differentiation of the formulas in 64 bits, around the stored x_out."""
    leaf = {n: t[n].double().detach().requires_grad_() for n in ("x", "y") + PARAMS if t[n] is not None}
    item = torch.arange(t["y"].shape[0], device=DEV) // c["L"]
    h = norm_h(leaf["x"], leaf, c, item)
    first = [n for n in ("x", "pre_w", "scale", "shift") if n in leaf]
    g = dict(zip(first, torch.autograd.grad((h * t["dh"].double()).sum(), [leaf[n] for n in first])))
    if dx_out:
        g["x"] = g["x"] + t["dx_out"].double()
    u, _ = norm_ref({**leaf, "x": torch.zeros_like(leaf["x"])}, c)
    second = [n for n in ("y", "gate", "post_w") if n in leaf]
    g |= dict(zip(second, torch.autograd.grad((u * g["x"]).sum(), [leaf[n] for n in second])))
    return g


def check_grads(got, ref, rows):
    # rows: about 20 roundings to fp32 on the way, sums over the columns among them; then the output's.
    # column sums: each adds up to `rows` terms, whose roundings grow as the root of their number
    for n in ("x", "y"):
        t = getattr(got, "d" + n)
        assert rel(t, ref[n]) <= half_step(t.dtype) + 64 * U, n
    for n in PARAMS:
        t = getattr(got, "d" + n)
        assert (t is None) == (n not in ref), n
        if t is not None:
            assert t.dtype == torch.float32 and rel(t, ref[n]) <= (64 + 4 * rows ** 0.5) * U, n


SIZES = [(1, 2048, 1), (77, 1024, 77), (6, 8, 3), (5, 7, 5), (4, 1, 2), (10, 1000, 5), (9, 333, 9), (12, 2047, 4),
         (6, 4096, 2), (7, 4095, 7), (300, 2048, 100), (257, 256, 257), (64, 40, 1)]


@pytest.mark.parametrize("rows,C,L", SIZES)
@pytest.mark.parametrize("post,pre", [(None, "layer"), ("rms", "rms"), ("layer", "layer")])
@pytest.mark.parametrize("full", [False, True])
def test_residual_norm_sizes(ops, rows, C, L, post, pre, full):
    if C == 1 and "layer" in (post, pre):
        pytest.skip("one column less its mean is nothing but rounding")
    t, c = make_norm(rows, C, L, post, pre, full, torch.float32, torch.float32, torch.float32)
    x, h = ops.residual_norm(t["x"], t["y"], **kwargs(t, c))
    rx, rh = norm_ref({n: (v.double() if v is not None else None) for n, v in t.items()}, c)
    assert rel(x, rx) <= 64 * U and rel(h, rh) <= 64 * U
    if C == 1:
        return  # a single column's rms norm is its sign: its gradient is nothing but rounding
    got = ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kwargs(t, c))
    check_grads(got, grad_refs(t, c), rows)


@pytest.mark.parametrize("xd", DTYPES)
@pytest.mark.parametrize("yd", DTYPES)
@pytest.mark.parametrize("hd", DTYPES)
@pytest.mark.parametrize("C", [1024, 333])
def test_residual_norm_types(ops, xd, yd, hd, C):
    t, c = make_norm(50, C, 25, "rms", "layer", True, xd, yd, hd, seed=10)
    x, h = ops.residual_norm(t["x"], t["y"], out_dtype=hd, **kwargs(t, c))
    rx, rh = norm_ref({n: (v.double() if v is not None else None) for n, v in t.items()}, c)
    assert (x.dtype, h.dtype) == (xd, hd)
    assert rel(x, rx) <= half_step(xd) + 64 * U and rel(h, rh) <= half_step(hd) + 64 * U
    got = ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kwargs(t, c))
    assert (got.dx.dtype, got.dy.dtype) == (xd, yd)
    check_grads(got, grad_refs(t, c), 50)


def test_residual_norm_backward_against_differences(ops):
    """The loss sum(h w) + sum(x_out v) moves as the gradients say (central differences, in the
    kernel's own forward): steps of 2^-6 leave 2^-12 of curvature and 2^-17 of rounding."""
    t, c = make_norm(8, 64, 4, "layer", "rms", True, torch.float32, torch.float32, torch.float32, seed=20)
    x_out, _ = ops.residual_norm(t["x"], t["y"], **kwargs(t, c))
    got = ops.residual_norm_backward(t["dh"], t["dx_out"], x_out, t["y"], **kwargs(t, c))

    def loss(**change):
        s = {**t, **change}
        x, h = ops.residual_norm(s["x"], s["y"], **kwargs(s, c))
        return ((h.double() * t["dh"].double()).sum() + (x.double() * t["dx_out"].double()).sum()).item()

    for n in ("x", "y") + PARAMS:
        d = randn(30, *t[n].shape)
        step = 2.0 ** -6
        slope = (loss(**{n: t[n] + step * d}) - loss(**{n: t[n] - step * d})) / (2 * step)
        want = (getattr(got, "d" + n).double() * d.double()).sum().item()
        size = (getattr(got, "d" + n).double().norm() * d.double().norm()).item()
        assert abs(slope - want) <= 2e-3 * size, n


def test_residual_norm_strides_in_place_and_neighbours(ops):
    t, c = make_norm(30, 256, 10, "rms", "rms", True, torch.bfloat16, torch.float16, torch.bfloat16, seed=40)
    kw = kwargs(t, c)
    x, h = ops.residual_norm(t["x"], t["y"], **kw)
    wide = torch.full((32, 272), 7.0, dtype=torch.bfloat16, device=DEV)
    xs, hs = wide[1:31, 8:264], torch.full((32, 264), 7.0, dtype=torch.bfloat16, device=DEV)
    xs.copy_(t["x"])
    ops.residual_norm(xs, t["y"], x_out=xs, h=hs[1:31, :256], **kw)
    assert torch.equal(xs, x) and torch.equal(hs[1:31, :256], h)
    assert bool((wide[[0, 31]] == 7).all() and (wide[:, :8] == 7).all() and (wide[:, 264:] == 7).all())
    assert bool((hs[[0, 31]] == 7).all() and (hs[:, 256:] == 7).all())
    ref = ops.residual_norm_backward(t["dh"], t["dx_out"], x, t["y"], **kw)
    g, y = t["dx_out"].clone(), t["y"].clone()
    got = ops.residual_norm_backward(t["dh"], g, x, y, dx=g, dy=y, **kw)
    assert got.dx is g and got.dy is y
    for a, b in zip(ref, got):
        assert torch.equal(a, b)
    none = ops.residual_norm_backward(t["dh"], None, x, t["y"], **kw)
    check_grads(none, grad_refs({**t, "x": x}, c, dx_out=False), 30)


def test_residual_norm_same_bits_and_rows_alone(ops):
    """The same inputs give the same bits, a row's result does not hang on its neighbours, and NaN in
    one row stays there (but for the column sums)."""
    t, c = make_norm(64, 1024, 32, "layer", "layer", True, torch.float32, torch.bfloat16, torch.bfloat16, seed=50)
    kw = kwargs(t, c)
    a, b = (ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kw) for _ in range(2))
    for u, v in zip(a, b):
        assert torch.equal(u, v)
    y = t["y"].clone()
    y[5] = float("nan")
    bad = ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], y, **kw)
    keep = torch.arange(64, device=DEV) != 5
    assert torch.equal(bad.dx[keep], a.dx[keep]) and torch.equal(bad.dy[keep], a.dy[keep])
    assert torch.equal(bad.dscale, a.dscale) and bool(bad.dgate[0].isnan().all()) and torch.equal(bad.dgate[1], a.dgate[1])
    x, h = ops.residual_norm(t["x"], y, **kw)
    x0, h0 = ops.residual_norm(t["x"], t["y"], **kw)
    assert torch.equal(x[keep], x0[keep]) and torch.equal(h[keep], h0[keep]) and bool(h[5].isnan().all())


def test_residual_norm_zero_rows_and_eps(ops):
    """A row of zeros normalises to zeros, with eps 0 only where no row is zero."""
    x, y = torch.zeros(3, 128, device=DEV), torch.zeros(3, 128, device=DEV)
    x_out, h = ops.residual_norm(x, y, post="rms", pre="rms")
    assert bool((h == 0).all() and (x_out == 0).all())
    t, c = make_norm(7, 96, 7, "rms", "rms", True, torch.float32, torch.float32, torch.float32, seed=60)
    c["eps"] = 0.0
    got = ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kwargs(t, c))
    check_grads(got, grad_refs(t, c), 7)
    e = torch.empty(0, 64, device=DEV)
    assert ops.residual_norm(e, e)[1].shape == (0, 64)
    g = ops.residual_norm_backward(e, e, e, e, pre_w=torch.ones(64, device=DEV))
    assert g.dx.shape == (0, 64) and bool((g.dpre_w == 0).all())


def test_residual_norm_large_mean(ops):
    """The variance is taken about the mean: rows of 1000 +- 1 keep their digits (x itself carries
    1000 u of rounding, so that much of 1 may be lost, not its square)."""
    t, c = make_norm(16, 2048, 16, None, "layer", False, torch.float32, torch.float32, torch.float32, seed=70)
    t["x"] = randn(71, 16, 2048, shift=1000.0)
    x, h = ops.residual_norm(t["x"], t["y"], **kwargs(t, c))
    _, rh = norm_ref({n: (v.double() if v is not None else None) for n, v in t.items()}, c)
    assert rel(h, rh) <= 2000 * U


def test_block_ops_captured_and_on_another_stream(ops):
    """Captured into a graph and replayed on new inputs, and on a side stream, the results are the
    same bits as eager ones; a graph's workspace is its own."""
    inv, m = ops.rotary_freqs(64, scaling="yarn", factor=2.0)
    t, c = make_norm(64, 512, 32, "rms", "layer", True, torch.float32, torch.bfloat16, torch.bfloat16, seed=80)
    q = randn(81, 64, 256, dtype=torch.bfloat16)

    def run():
        x, h = ops.residual_norm(t["x"], t["y"], out_dtype=torch.bfloat16, **kwargs(t, c))
        r = ops.rotary(q, None, inv, Hq=4, D=64, mscale=m)[0]
        return [x, h, r, *ops.residual_norm_backward(t["dh"], t["dx_out"], x, t["y"], **kwargs(t, c))]

    run()
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(run())
    for n in ("x", "y", "dh"):
        t[n].copy_(randn(82, *t[n].shape, dtype=t[n].dtype))
    want = run()
    s = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for g, st in zip(graphs, s):  # at the same time
        with torch.cuda.stream(st):
            g.replay()
    torch.cuda.synchronize()
    for got in outs:
        for a, b in zip(got, want):
            assert torch.equal(a, b)
    with torch.cuda.stream(s[0]):
        side = run()
    torch.cuda.synchronize()
    for a, b in zip(side, want):
        assert torch.equal(a, b)


# Blocks of several rows: as many as the ring has places and more, so that places are filled again, phases
# turn, column sums gather and the row sums' shared memory is used again and again. The last block of an item
# has fewer rows than the others.
MANY_ROWS = [(4593, 1024, 1531, "rms", "rms", torch.bfloat16, torch.bfloat16, torch.bfloat16),
             (16382, 512, 8191, "layer", "layer", torch.float32, torch.float32, torch.float32),
             (8191, 2048, 8191, None, "layer", torch.float32, torch.float16, torch.float16),
             (8190, 2048, 2730, "layer", "rms", torch.float32, torch.bfloat16, torch.bfloat16),
             (2503, 4096, 2503, "rms", "layer", torch.float32, torch.float32, torch.float32),  # a ring of two places
             (20001, 256, 6667, "rms", "layer", torch.bfloat16, torch.bfloat16, torch.float16)]


@pytest.mark.parametrize("rows,C,L,post,pre,xd,yd,hd", MANY_ROWS)
def test_residual_norm_blocks_of_many_rows(ops, rows, C, L, post, pre, xd, yd, hd):
    t, c = make_norm(rows, C, L, post, pre, True, xd, yd, hd, seed=90)
    kw = kwargs(t, c)

    def run():
        x, h = ops.residual_norm(t["x"], t["y"], out_dtype=hd, **kw)
        return [x, h, *(g for g in ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kw) if g is not None)]

    want = run()
    rx, rh = norm_ref({n: (v.double() if v is not None else None) for n, v in t.items()}, c)
    assert rel(want[0], rx) <= half_step(xd) + 64 * U and rel(want[1], rh) <= half_step(hd) + 64 * U
    got = ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kw)
    check_grads(got, grad_refs(t, c), rows)
    dx, dy = t["dx_out"].clone(), t["y"].clone()
    here = ops.residual_norm_backward(t["dh"], dx, t["x"], dy, dx=dx, dy=dy, **kw)
    for a, b in zip(got, here):
        assert (a is None and b is None) or torch.equal(a, b)
    for _ in range(200):
        for a, b in zip(want, run()):
            assert torch.equal(a, b)


def test_two_threads_on_streams_of_their_own(ops):
    """Both share the device's context. Each works on inputs that its own stream has just written, so a call
    on the other's stream would find the old ones."""
    inv, _ = ops.rotary_freqs(128)
    x = [randn(100 + i, 2048, 16 * 128, dtype=torch.bfloat16) for i in range(2)]
    want = [ops.rotary(t, None, inv, Hq=16, D=128)[0] for t in x]
    wrong, errors = [0, 0], []
    torch.cuda.synchronize()

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(200):
                    t = torch.zeros_like(x[i])
                    t.copy_(x[i])
                    wrong[i] += int(not torch.equal(ops.rotary(t, None, inv, Hq=16, D=128)[0], want[i]))
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and wrong == [0, 0]


@pytest.mark.parametrize("rows,C,L", [(65536, 8, 1), (70001, 33, 1), (131074, 64, 2)])
def test_residual_norm_of_many_items(ops, rows, C, L):
    """A modulation for each row or two, more of them than a grid axis has blocks, beside sums over all."""
    t, c = make_norm(rows, C, L, "rms", "rms", True, torch.float32, torch.float32, torch.float32, seed=110)
    x, h = ops.residual_norm(t["x"], t["y"], **kwargs(t, c))
    rx, rh = norm_ref({n: (v.double() if v is not None else None) for n, v in t.items()}, c)
    assert rel(x, rx) <= 64 * U and rel(h, rh) <= 64 * U
    got = ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kwargs(t, c))
    ref = grad_refs(t, c)
    check_grads(got, ref, rows)
    # each item for itself: some 20 roundings of every term, and the terms' own sums of magnitudes
    p = {n: v.double() for n, v in t.items() if v is not None}
    item = torch.arange(rows, device=DEV) // L
    r = 1 / (p["x"].square().mean(1, keepdim=True) + c["eps"]).sqrt()
    n, u = p["x"] * r, normalise(p["y"], "rms", c["eps"]) * p["post_w"]
    g = p["dh"] * (1 + p["scale"][item]) * p["pre_w"]
    G = p["dx_out"].abs() + r * (g.abs() + n.abs() * (g * n).abs().mean(1, keepdim=True))
    for name, mag in (("gate", c["alpha"] * G * u.abs()), ("scale", (p["dh"] * n * p["pre_w"]).abs()), ("shift", p["dh"].abs())):
        mag = mag.view(-1, L, C).sum(1)
        assert bool(((getattr(got, "d" + name).double() - ref[name]).abs() <= 64 * U * mag).all()), name


def test_residual_norm_rows_out_of_range(ops):
    """Infinities, NaN and squares past fp32 stay in their rows, forward and backward, in the forms for whole and
    for other widths alike: a row whose squares overflow has the norm 0 (its x_out stays), as 1 / sqrt(inf) says."""
    for C in (1024, 1000):
        t, c = make_norm(16, C, 16, None, "rms", False, torch.float32, torch.float32, torch.float32, seed=120)
        kw = kwargs(t, c)
        t["y"].zero_()
        x0, h0 = ops.residual_norm(t["x"], t["y"], **kw)
        g0 = ops.residual_norm_backward(t["dh"], t["dx_out"], t["x"], t["y"], **kw)
        x = t["x"].clone()
        x[3], x[7, 5], x[9, 11] = 1e25, float("inf"), float("nan")
        x1, h1 = ops.residual_norm(x, t["y"], **kw)
        g1 = ops.residual_norm_backward(t["dh"], t["dx_out"], x, t["y"], **kw)
        keep = torch.tensor([r not in (3, 7, 9) for r in range(16)], device=DEV)
        for a, b in ((x0, x1), (h0, h1), (g0.dx, g1.dx), (g0.dy, g1.dy)):
            assert torch.equal(a[keep], b[keep])
        assert bool((h1[3] == 0).all() and torch.equal(x1[3], x[3]) and torch.equal(g1.dx[3], t["dx_out"][3]))
        others = torch.arange(C, device=DEV) != 5
        assert bool(h1[7, 5].isnan() and (h1[7, others] == 0).all() and h1[9].isnan().all())
