"""Attention with its backward pass on a B200, against the formulas in 64 bits.

Tolerances are worst-case bounds, element by element, of the roundings that the kernels make. With h
half a step of the operands' type: P, dS and every output round once to that type (h of their value
each), and delta is taken from the rounded output (h of sum |dO O|). What is in fp32 (scores, exponents,
sums of up to a few thousand terms) stays below F = 2^-16 of the magnitudes that are summed."""

import ctypes
import math

import pytest
import torch

from tests.conftest import pkg

pytestmark = pytest.mark.gpu

DEV = "cuda"
F = 2.0 ** -16
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    return pkg("ops")


@pytest.fixture(autouse=True)
def no_device_error():
    """No wait of a kernel ran out."""
    yield
    pkg("device").Context.get(0).sync()


def randn(seed, *shape, dtype=FP, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(q, k, v, do, *, group=1, causal=False, lens=None, scale=None, dtype, out_dtype=None, grad_dtype=None):
    """q, do [B, H, Lq, D], k, v [B, Hk, Lk, D] in 64 bits: values and tolerances of out, lse, dq, dk, dv
    ([B, heads, L, D]; dk and dv of every item on its own)."""
    B, H, Lq, D = q.shape
    Lk = k.shape[2]
    scale = scale or 1 / math.sqrt(D)
    h = half_step(dtype)
    ho, hg = (half_step(t or dtype) for t in (out_dtype, grad_dtype))
    tiny = 2.0 ** -24 if dtype == HF else 0.0  # steps of fp16 below 2^-14 no longer shrink
    kk, vv = (t.repeat_interleave(group, 1) for t in (k, v))
    hidden = torch.zeros(B, 1, Lq, Lk, dtype=torch.bool, device=DEV)
    if causal:
        hidden |= torch.ones(Lq, Lk, dtype=torch.bool, device=DEV).triu(1)
    if lens is not None:
        hidden |= (torch.arange(Lk, device=DEV) >= lens.view(B, 1, 1, 1))
        gone = (torch.arange(Lk, device=DEV) >= lens.view(B, 1, 1))[..., None]
        kk, vv = kk.masked_fill(gone, 0.0), vv.masked_fill(gone, 0.0)
    s = (q @ kk.transpose(-1, -2) * scale).masked_fill(hidden, float("-inf"))
    lse = torch.logsumexp(s, -1)
    p = torch.where(torch.isfinite(lse)[..., None], torch.exp(s - lse[..., None]), torch.zeros_like(s))
    out = p @ vv
    dv = p.transpose(-1, -2) @ do
    dp = do @ vv.transpose(-1, -2)
    delta = (do * out).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    dq, dk = ds @ kk * scale, ds.transpose(-1, -2) @ q * scale
    # bounds. e_p: of P itself, from scores in fp32
    s_abs = (q.abs() @ kk.abs().transpose(-1, -2) * scale).masked_fill(hidden, 0.0)
    e_p = F + 2.0 ** -20 * s_abs
    e_out = ((h + e_p) * p + tiny * ~hidden) @ vv.abs() + ho * out.abs() + tiny
    e_delta = (do.abs() * (e_out + F * out.abs())).sum(-1, keepdim=True)
    dp_abs = do.abs() @ vv.abs().transpose(-1, -2)
    bound = 2 * do.norm(dim=-1).amax() * v.nan_to_num(0).norm(dim=-1).amax() if tiny else 0.0
    e_ds = (h + e_p) * ds.abs() + p * (e_delta + F * dp_abs + e_p * delta.abs()) + 2.0 ** -38 * bound
    e_ds = e_ds.masked_fill(hidden, 0.0)
    rows = lambda e, m, y: scale * (e @ m.abs()) + hg * y.abs() + tiny  # noqa: E731
    T = lambda t: t.transpose(-1, -2)  # noqa: E731
    tol = {"out": e_out, "lse": 2.0 ** -20 * (4 + s_abs.amax(-1) + lse.nan_to_num(0, 0, 0).abs()),
           "dq": rows(e_ds + F * ds.abs(), kk, dq), "dk": rows(T(e_ds + F * ds.abs()), q, dk),
           "dv": T((h + e_p) * p) @ do.abs() + hg * dv.abs() + tiny}
    val = {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    for n in ("dk", "dv"):  # shared heads
        for t in (val, tol):
            t[n] = t[n].view(B, H // group, group, Lk, D).sum(2)
    return val, tol


def check(got, val, tol, names=("out", "lse", "dq", "dk", "dv")):
    for n in names:
        g, r = got[n].double(), val[n]
        same = (g == r) | ((g - r).abs() <= tol[n])
        assert bool(same.all()), (n, (g - r).abs().nan_to_num(9e9).sub(tol[n]).max().item(), (~same).sum().item())


class Case:
    """Plain [B * L, heads * D] tensors of one problem, the call's arguments, and the reference's views."""

    def __init__(self, B, H, group, D, Lq, Lk, dtype, *, causal=False, lens=None, seed=0, gscale=1.0, sharp=1.0):
        self.B, self.H, self.Hk, self.D, self.Lq, self.Lk, self.dtype = B, H, H // group, D, Lq, Lk, dtype
        self.q = randn(seed + 1, B * Lq, H * D, dtype=dtype, scale=sharp)
        self.k = randn(seed + 2, B * Lk, self.Hk * D, dtype=dtype, scale=sharp)
        self.v = randn(seed + 3, B * Lk, self.Hk * D, dtype=dtype)
        self.do = randn(seed + 4, B * Lq, H * D, dtype=dtype, scale=gscale)
        self.lens = torch.tensor(lens, dtype=torch.int32, device=DEV) if lens is not None else None
        self.kw = dict(Lq=Lq, Lk=Lk, H=H, D=D, batch=B, group=group, causal=causal, key_len=self.lens,
                       q_bstride=Lq * H * D, k_bstride=Lk * self.Hk * D, v_bstride=Lk * self.Hk * D)
        self.ref_kw = dict(group=group, causal=causal, lens=self.lens, dtype=dtype)

    def heads(self, t, L):
        return t.view(self.B, L, -1, self.D).transpose(1, 2)

    def reference(self, **kw):
        a = [self.heads(t, L).double() for t, L in ((self.q, self.Lq), (self.k, self.Lk), (self.v, self.Lk), (self.do, self.Lq))]
        return reference(*a, **{**self.ref_kw, **kw})

    def run(self, ops, fwd={}, bwd={}):
        out, lse = ops.attention_lse(self.q, self.k, self.v, **self.kw, **fwd)
        dq, dk, dv = ops.attention_backward(self.do, self.q, self.k, self.v, out, lse, **self.kw, **bwd)
        return {"out": self.heads(out, self.Lq), "lse": lse, "dq": self.heads(dq, self.Lq),
                "dk": self.heads(dk, self.Lk), "dv": self.heads(dv, self.Lk)}


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (1, 77), (77, 1), (77, 77), (128, 128), (129, 257), (300, 64), (513, 1000),
                                   (64, 2048), (2048, 64), (255, 256)])
def test_lengths(ops, dtype, D, Lq, Lk):
    c = Case(1, 2, 1, D, Lq, Lk, dtype)
    check(c.run(ops), *c.reference())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lq,Lk", [(1, 1), (2, 2), (77, 77), (128, 128), (300, 300), (129, 500), (500, 129), (1025, 1025)])
def test_causal_shared_heads(ops, dtype, D, Lq, Lk):
    c = Case(2, 4, 2, D, Lq, Lk, dtype, causal=True)
    check(c.run(ops), *c.reference())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("causal,group,lens", [(True, 1, None), (True, 2, (1500,)), (False, 2, (1201,)), (True, 2, (130,))])
def test_few_units_are_split_along_their_walk(ops, dtype, D, causal, group, lens):
    """Two heads of 1500 tokens do not fill the SMs: the units are split and their parts joined, some of
    them without a block (a causal unit's first keys, keys past key_len)."""
    c = Case(1, 2, group, D, 1500, 1500, dtype, causal=causal, lens=lens)
    check(c.run(ops), *c.reference())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("Lq,Lk,lens", [(200, 333, (333, 129, 1, 0)), (130, 256, (128, 256, 500, -3)), (64, 700, (1, 640, 699, 513))])
def test_key_lengths(ops, dtype, D, causal, Lq, Lk, lens):
    c = Case(4, 4, 4, D, Lq, Lk, dtype, causal=causal, lens=lens)
    val, tol = c.reference()
    got = c.run(ops)
    check(got, val, tol)
    for b, n in enumerate(lens):  # nothing flows past them, and rows that see no key have lse = -inf
        n = max(0, min(n, Lk))
        assert bool((got["dk"][b, :, n:] == 0).all() and (got["dv"][b, :, n:] == 0).all())
        if n == 0:
            assert bool((got["out"][b] == 0).all() and (got["dq"][b] == 0).all() and got["lse"][b].eq(-math.inf).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -6e4])
def test_what_lies_behind_key_len_does_not_count(ops, dtype, D, bad):
    lens = (131, 200, 64)
    c = Case(3, 2, 1, D, 150, 260, dtype, lens=lens)
    ref = c.run(ops)
    if D == 128:  # attention() has the same output, as long as what it multiplies by 0 is finite
        assert torch.equal(ops.attention(c.q, c.k, c.v, **c.kw), ref["out"].transpose(1, 2).reshape(3 * 150, -1))
    for b, n in enumerate(lens):
        for t in (c.k, c.v):
            t.view(3, 260, -1)[b, n:] = bad
    got = c.run(ops)
    for n in ref:
        assert torch.equal(ref[n], got[n]), n


@pytest.mark.parametrize("dtype", [BF, HF])
def test_packed_gradients_strides_and_neighbours(ops, dtype):
    """q|k|v in one tensor, its gradient likewise, rows with a gap behind them; what is not a gradient
    stays as it was."""
    B, L, H, D = 2, 150, 4, 64
    C = H * D
    x = randn(1, B * L, 3 * C + 8, dtype=dtype)
    do = randn(2, B * L, C, dtype=dtype)
    ld = 3 * C + 8
    kw = dict(Lq=L, Lk=L, H=H, D=D, batch=B, ldq=ld, ldk=ld, ldv=ld, q_off=0, k_off=C, v_off=2 * C, q_bstride=L * ld,
              k_bstride=L * ld, v_bstride=L * ld)
    wide = torch.full((B * L, C + 16), 3.0, dtype=dtype, device=DEV)
    out, lse = ops.attention_lse(x, x, x, out=wide[:, 8:C + 8], **kw)
    dx = torch.full((B * L + 1, ld), 7.0, dtype=dtype, device=DEV)
    d = [dx[:B * L, i * C:(i + 1) * C] for i in range(3)]
    got = ops.attention_backward(do, x, x, x, out, lse, dq=d[0], dk=d[1], dv=d[2], **kw)
    assert all(a is b for a, b in zip(got, d))
    view = lambda t: t.reshape(B, L, H, D).transpose(1, 2)  # noqa: E731
    val, tol = reference(*(view(x[:, i * C:(i + 1) * C]).double() for i in range(3)), view(do).double(), dtype=dtype)
    check({"out": view(out), "lse": lse, "dq": view(d[0]), "dk": view(d[1]), "dv": view(d[2])}, val, tol)
    assert bool((dx[:, 3 * C:] == 7).all() and (dx[B * L] == 7).all())
    assert bool((wide[:, :8] == 3).all() and (wide[:, C + 8:] == 3).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("Lq,Lk", [(200, 130), (70, 600)])
def test_shared_kv_sums_over_the_batch(ops, dtype, Lq, Lk):
    """k_bstride = v_bstride = 0: all items read one K/V (and key_len[0]); its gradient is the sum."""
    B, H, D = 3, 2, 64
    c = Case(B, H, 1, D, Lq, Lk, dtype, lens=(Lk - 5,) * B)
    for t in (c.k, c.v):
        t.view(B, Lk, -1)[1:] = t.view(B, Lk, -1)[0]
    val, tol = c.reference()
    one = {"k": c.k[:Lk].contiguous(), "v": c.v[:Lk].contiguous()}
    kw = {**c.kw, "k_bstride": 0, "v_bstride": 0, "key_len": c.lens[:1]}
    out, lse = ops.attention_lse(c.q, one["k"], one["v"], **kw)
    dq, dk, dv = ops.attention_backward(c.do, c.q, one["k"], one["v"], out, lse, **kw)
    assert dk.shape == (Lk, H * D)
    check({"out": c.heads(out, Lq), "lse": lse, "dq": c.heads(dq, Lq)}, val, tol, ("out", "lse", "dq"))
    for n, g in (("dk", dk), ("dv", dv)):
        assert bool(((g.view(Lk, H, D).transpose(0, 1).double() - val[n].sum(0)).abs() <= tol[n].sum(0)).all()), n


@pytest.mark.parametrize("out_dtype", [None, FP])
@pytest.mark.parametrize("grad_dtype", [None, FP])
def test_fp32_output_and_gradients(ops, out_dtype, grad_dtype):
    c = Case(1, 2, 1, 128, 200, 1030, BF)
    got = c.run(ops, dict(out_dtype=out_dtype), dict(grad_dtype=grad_dtype))
    assert got["out"].dtype == (out_dtype or BF) and got["dq"].dtype == got["dk"].dtype == (grad_dtype or BF)
    check(got, *c.reference(out_dtype=out_dtype, grad_dtype=grad_dtype))


@pytest.mark.parametrize("gscale", [1e-6, 1e-3, 300.0])
def test_fp16_gradients_of_any_size(ops, gscale):
    """dS is moved into fp16's range by a power of two: gradients in fp32 keep their digits whatever
    the size of dout (whose own subnormals are exact inputs)."""
    c = Case(1, 2, 1, 64, 260, 2000, HF, gscale=gscale)
    got = c.run(ops, dict(out_dtype=FP), dict(grad_dtype=FP))
    val, _ = c.reference()
    for n in ("dq", "dk", "dv"):
        # |dP - delta| P near 2^-11 of the bound, 2^4 above fp16's subnormals: steps of 2^-11 each
        assert ((got[n].double() - val[n]).norm() / val[n].norm()).item() < 2 * half_step(HF), n


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scale_and_sharp_rows(ops, dtype):
    """Another softmax scale, and scores so far apart that most probabilities are 0 or 1."""
    c = Case(1, 2, 1, 64, 140, 300, dtype, sharp=3.0)
    c.kw["scale"] = 0.5
    check(c.run(ops), *c.reference(scale=0.5))


def test_against_differences(ops):
    """The loss sum(out w), out in fp32, moves as dq, dk and dv say. bf16 inputs leave whole steps to
    move by: an element of q, k or v changes by 1/8, the slope's error is cubic."""
    c = Case(1, 1, 1, 64, 40, 50, BF, seed=5)
    for n in "qkv":
        setattr(c, n, (getattr(c, n) * 8).round().div(8).clamp(-3, 3))  # so that +- 1/8 is exact in bf16
    got = c.run(ops, {}, dict(grad_dtype=FP))

    def loss():
        out, _ = ops.attention_lse(c.q, c.k, c.v, out_dtype=FP, **c.kw)
        return (out.double() * c.do.double()).sum().item()

    for n, L in (("q", 40), ("k", 50), ("v", 50)):
        t, keep = getattr(c, n), getattr(c, n).clone()
        d = (randn(9, *t.shape) > 0).to(BF) * 0.25 - 0.125
        t.copy_(keep + d)
        up = loss()
        t.copy_(keep - d)
        slope = (up - loss()) / 2
        t.copy_(keep)
        g = got["d" + n].transpose(1, 2).reshape(L, -1).double()
        # third-order term of a step of 1/8 in every element: scores move by up to 1/8 sqrt(64) / 8, a few
        # per cent of the slope's own size, which for random signs is |g| / 8
        assert abs(slope - (g * d.double()).sum().item()) <= 0.2 * g.norm().item() * 0.125 * 2, n


@pytest.mark.parametrize("causal", [False, True])
def test_same_bits_again(ops, causal):
    c = Case(1, 8, 2, 128, 1500, 1500, BF, causal=causal)
    a, b = c.run(ops), c.run(ops)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_long_self_attention_stream_k(ops):
    """4096 tokens of 16 heads, the key blocks spread over the SMs: the output has attention()'s bits,
    two heads are compared in full, and the workspace is the call's own."""
    c = Case(1, 16, 1, 128, 4096, 4096, HF)
    got = c.run(ops)
    assert torch.equal(ops.attention(c.q, c.k, c.v, **c.kw), got["out"].transpose(1, 2).reshape(4096, -1))
    for h in (0, 11):
        one = [c.heads(t, 4096)[:, h:h + 1].double() for t in (c.q, c.k, c.v, c.do)]
        val, tol = reference(*one, dtype=HF)
        check({n: t[:, h:h + 1] for n, t in got.items()}, val, tol)


def test_captured_replayed_and_two_at_once(ops):
    """Two graphs of the same step hold workspaces of their own: replayed at the same time on two
    streams, on inputs that came after the capture, both give the eager bits."""
    c = Case(2, 4, 2, 128, 700, 900, BF, lens=(900, 333))
    c.run(ops)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(c.run(ops))
    for n in ("q", "k", "v", "do"):
        getattr(c, n).copy_(randn(77, *getattr(c, n).shape, dtype=BF))
    c.lens.copy_(torch.tensor([640, 0], dtype=torch.int32))
    want = c.run(ops)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for g, s in zip(graphs, streams):
        with torch.cuda.stream(s):
            g.replay()
    torch.cuda.synchronize()
    for got in outs:
        for n in want:
            assert torch.equal(got[n], want[n]), n
    check(want, *c.reference())
    with torch.cuda.stream(streams[0]):
        side = c.run(ops)
    torch.cuda.synchronize()
    for n in want:
        assert torch.equal(side[n], want[n]), n


def test_offsets_past_32_bits(ops):
    """Items 2^31 + 1024 elements apart."""
    bs = 2 ** 31 + 1024
    H, D, L = 1, 64, 100
    c = Case(2, H, 1, D, L, L, BF)
    kw = {**c.kw, "q_bstride": bs, "k_bstride": bs, "v_bstride": bs, "ldq": 3 * D, "ldk": 3 * D, "ldv": 3 * D, "q_off": 0,
          "k_off": D, "v_off": 2 * D}
    far = torch.empty(bs + L * 3 * D, dtype=BF, device=DEV)
    for b in range(2):
        rows = far[b * bs:b * bs + L * 3 * D].view(L, 3 * D)
        for i, t in enumerate((c.q, c.k, c.v)):
            rows[:, i * D:(i + 1) * D] = t[b * L:(b + 1) * L]
    out, lse = ops.attention_lse(far, far, far, **kw)
    dq, dk, dv = ops.attention_backward(c.do, far, far, far, out, lse, **kw)
    want = c.run(ops)
    for n, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert torch.equal(c.heads(t, L), want[n]), n


def test_library_refusals(ops):
    err = pkg("device").AnimaError
    c = Case(1, 2, 1, 64, 32, 32, BF)
    odd = torch.empty(33 * 128 + 4, dtype=BF, device=DEV)[4:].as_strided((32, 128), (128, 1))
    with pytest.raises(err, match="aligned"):
        ops.attention_lse(odd, c.k, c.v, **c.kw)
    out, lse = ops.attention_lse(c.q, c.k, c.v, **c.kw)
    with pytest.raises(err, match="aligned"):
        ops.attention_backward(c.do, c.q, c.k, c.v, out, lse, dq=odd, **c.kw)


@pytest.mark.parametrize("B,H,Lq,Lk,lens,causal", [(2, 16, 4096, 512, (512, 325), False), (1, 16, 1024, 1024, None, False),
                                                    (1, 16, 1500, 1500, None, True)])
def test_many_passes(ops, B, H, Lq, Lk, lens, causal):
    """400 passes back to back: the same bits each time, and no wait runs out. (A q unit's dP runs a block
    ahead of its dS: a barrier that the math warps can pass twice before the issuing warp looks at it
    would stop a block once in some hundred thousand.)"""
    c = Case(B, H, 1, 128, Lq, Lk, BF, causal=causal, lens=lens)
    want = c.run(ops)
    for i in range(400):
        got = c.run(ops)
        if i % 100 == 99:
            for n in want:
                assert torch.equal(got[n], want[n]), n


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lq,Lk,causal", [(300, 5, False), (70, 128, False), (3, 3, True), (200, 200, True)])
def test_rows_of_few_keys_keep_their_digits(ops, dtype, D, Lq, Lk, causal):
    """Where a query block's keys lie in one key block, delta comes from the probabilities: against the
    64-bit gradients the error is that of rounding dS and the result once each (twice half a step, in
    the 2-norm), where a delta of the rounded output would add the rounding of sum |dO O|."""
    c = Case(1, 4, 2, D, Lq, Lk, dtype, causal=causal)
    got, (val, _) = c.run(ops), c.reference()
    rows = min(Lq, 128) if causal else Lq
    g, r = got["dq"][:, :, :rows].double(), val["dq"][:, :, :rows]
    assert ((g - r).norm() / r.norm()).item() <= 2 * half_step(dtype)


@pytest.mark.parametrize("grad_dtype", [BF, FP])
@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lq,Lk,causal", [(1, 33, False), (161, 95, False), (223, 223, True)])
def test_rows_behind_the_last_stay(ops, D, Lq, Lk, causal, grad_dtype):
    """Items of odd lengths lie end to end: a tile's rows past an item's end belong to the next item, or lie
    behind the last one, and its columns beside the heads'."""
    c = Case(3, 4, 2, D, Lq, Lk, BF, causal=causal, lens=[Lk, 0, max(1, Lk - 40)])
    bufs = [torch.full((3 * L + 130, n * D + 8), 7.0, dtype=grad_dtype, device=DEV) for L, n in ((Lq, 4), (Lk, 2), (Lk, 2))]
    d = [b[:, :b.shape[1] - 8] for b in bufs]
    out, lse = ops.attention_lse(c.q, c.k, c.v, **c.kw)
    ops.attention_backward(c.do, c.q, c.k, c.v, out, lse, dq=d[0], dk=d[1], dv=d[2], **c.kw)
    val, tol = c.reference(grad_dtype=grad_dtype)
    got = {n: c.heads(t[:3 * L].contiguous(), L) for n, t, L in zip(("dq", "dk", "dv"), d, (Lq, Lk, Lk))}
    check(got, val, tol, ("dq", "dk", "dv"))
    for b, L in zip(bufs, (Lq, Lk, Lk)):
        assert bool((b[3 * L:] == 7).all() and (b[:, -8:] == 7).all())


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("dtype,scale,sharp", [
    (HF, 2.0 ** -24, 1.0), (HF, 1e-7, 1.0), (HF, 1e-6, 1.0), (HF, 3e-5, 1.0), (HF, 2e-7, 700.0), (HF, 2.0 ** -24, 1500.0),
    (BF, 2.0 ** -100, 1.0), (BF, 1e-30, 1.0), (BF, 1e-7, 700.0)])
def test_small_scales(ops, D, dtype, scale, sharp):
    """lse / scale, which enters a product in 16-bit parts, is up to 10^8 times the scores' differences, and
    with large q and k as large as they are. Beside the bounds of each element, the 2-norm: P and dS round
    once (half a step each, random), delta and out are in fp32."""
    c = Case(2, 4, 2, D, 200, 300, dtype, lens=(300, 129), sharp=sharp)
    c.kw["scale"] = scale
    got = c.run(ops, dict(out_dtype=FP), dict(grad_dtype=FP))
    val, tol = c.reference(scale=scale, out_dtype=FP, grad_dtype=FP)
    check(got, val, tol)
    for n in ("dq", "dk", "dv"):
        assert ((got[n].double() - val[n]).norm() / val[n].norm()).item() < 2 * half_step(dtype), n


def test_the_library_refuses_scales(ops):
    dev = pkg("device")
    c = Case(1, 2, 1, 64, 32, 32, HF)
    ctx, need = dev.Context.get(0), ctypes.c_size_t()
    for scale, dtype in ((math.nan, BF), (math.inf, BF), (2.0 ** -25, HF), (2.0 ** -101, BF), (2.0 ** 65, HF)):
        g = dev.AttentionGradArgs()
        g.fwd.batch, g.fwd.heads, g.fwd.head_dim, g.fwd.Lq, g.fwd.Lk = 1, 2, 64, 32, 32
        g.fwd.dtype, g.fwd.scale = dev.DTYPE_CODE[dtype], scale
        with pytest.raises(dev.AnimaError, match="scale"):
            dev.check(ctx.lib.anima_attention_backward_workspace(ctx.h, ctypes.byref(g), ctypes.byref(need)))
    out, lse = ops.attention_lse(c.q, c.k, c.v, **c.kw, scale=2.0 ** -24)
    assert lse.isfinite().all()


@pytest.mark.parametrize("D", [128, 64])
@pytest.mark.parametrize("Lk,lens", [(2048, (2048, 1333)), (1030, (1030, 0)), (300, None)])
def test_long_causal_schedule(ops, D, Lk, lens):
    """More causal units than SMs, of eight query tiles' pairs a head: one CTA each with the longest first, or (few
    keys) a persistent grid. Both have the bits of each head alone, whose units are in neither."""
    B, H, L = 2, 16, 2048
    c = Case(B, H, 1, D, L, Lk, BF, causal=True, lens=lens)
    out, lse = ops.attention_lse(c.q, c.k, c.v, **c.kw)
    if D == 128:
        assert torch.equal(ops.attention(c.q, c.k, c.v, **c.kw), out)
    for b in range(B):
        for h in (0, 5, 15):
            q, k, v = (c.heads(t, n)[b, h].contiguous() for t, n in ((c.q, L), (c.k, Lk), (c.v, Lk)))
            o1, l1 = ops.attention_lse(q, k, v, Lq=L, Lk=Lk, H=1, D=D, causal=True,
                                       key_len=c.lens[b:b + 1] if lens else None)
            assert torch.equal(c.heads(out, L)[b, h], o1) and torch.equal(lse[b, h], l1[0, 0])
    one = [c.heads(t, n)[:, 3:4].double() for t, n in ((c.q, L), (c.k, Lk), (c.v, Lk), (c.do, L))]
    val, tol = reference(*one, causal=True, lens=c.lens, dtype=BF)
    check({"out": c.heads(out, L)[:, 3:4], "lse": lse[:, 3:4]}, val, tol, ("out", "lse"))


@pytest.mark.parametrize("dtype,D,causal", [(BF, 64, False), (HF, 64, True), (HF, 128, False)])
def test_more_items_than_a_grid_axis_has_blocks(ops, dtype, D, causal):
    """Windows of a few tokens, each an item of its own."""
    B, Lq, Lk = 66001, 3, 3 if causal else 5
    lens = [(i * 7) % (Lk + 1) for i in range(B)]
    c = Case(B, 1, 1, D, Lq, Lk, dtype, causal=causal, lens=lens)
    check(c.run(ops), *c.reference())


def test_more_items_share_keys_than_a_grid_axis_has_blocks(ops):
    B, Lq, Lk, D = 66001, 2, 5, 64
    c = Case(B, 1, 1, D, Lq, Lk, HF, gscale=0.03)
    for t in (c.k, c.v):
        t.view(B, Lk, -1)[1:] = t.view(B, Lk, -1)[0]
    val, tol = c.reference()
    k, v, kw = c.k[:Lk].contiguous(), c.v[:Lk].contiguous(), {**c.kw, "k_bstride": 0, "v_bstride": 0}
    out, lse = ops.attention_lse(c.q, k, v, **kw)
    dq, dk, dv = ops.attention_backward(c.do, c.q, k, v, out, lse, **kw)
    check({"out": c.heads(out, Lq), "lse": lse, "dq": c.heads(dq, Lq)}, val, tol, ("out", "lse", "dq"))
    for n, g in (("dk", dk), ("dv", dv)):
        r = val[n].sum(0)
        assert bool(((g.view(Lk, 1, D).transpose(0, 1).double() - r).abs() <= tol[n].sum(0) + half_step(HF) * r.abs()).all()), n
