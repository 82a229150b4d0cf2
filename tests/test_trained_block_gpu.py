"""One attention block as it is trained, forward and backward through the framework's operators: the gated
residual and adaLN norm before it, a q|k|v projection with a LoRA, rotary positions, causal attention with
shared k/v heads on a padded batch, the output projection, the gated residual and norm behind it. Every
gradient, the LoRA's among them, against automatic differentiation in 64 bits."""

import math

import pytest
import torch

from tests.conftest import pkg

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF = torch.bfloat16


def randn(seed, *shape, dtype=torch.float32, scale=1.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


B, L, C, H, HK, D, RANK = 2, 150, 256, 4, 2, 64, 8
LENS = (150, 97)
ROWS = B * L


def make():
    p = {"x": randn(1, ROWS, C), "y": randn(2, ROWS, C, dtype=BF), "mods1": randn(3, B, 3 * C, scale=0.3),
         "mods2": randn(4, B, 3 * C, scale=0.3), "w": randn(5, (H + 2 * HK) * D, C, dtype=BF, scale=C ** -0.5),
         "a": randn(6, RANK, C, dtype=BF, scale=C ** -0.5), "b": randn(7, (H + 2 * HK) * D, RANK, dtype=BF, scale=0.2),
         "wo": randn(8, C, H * D, dtype=BF, scale=C ** -0.5)}
    up = {"h": randn(9, ROWS, C, dtype=BF), "x": randn(10, ROWS, C)}
    live = (torch.arange(L, device=DEV) < torch.tensor(LENS, device=DEV)[:, None]).reshape(-1, 1)
    for n in up:  # nothing hangs on the padding
        up[n] = (up[n] * live).to(up[n].dtype)
    return p, up


def mods(m):
    return {n: m[:, i * C:(i + 1) * C] for i, n in enumerate(("shift", "scale", "gate"))}


def plan(ops):
    """What a program makes once: frequencies and key lengths on the device."""
    return ops.rotary_freqs(D, 1e6)[0], torch.tensor(LENS, dtype=torch.int32, device=DEV)


def block(ops, p, up, inv, lens):
    """(x, h) of the block's end and the gradients of all of p."""
    N, NK = H * D, HK * D
    attn = dict(Lq=L, Lk=L, H=H, D=D, batch=B, group=H // HK, causal=True, key_len=lens, q_bstride=L * N,
                k_bstride=L * NK, v_bstride=L * NK)
    rot = dict(Hq=H, Hk=HK, D=D, rows_per_item=L)
    n1, n2 = (dict(pre="layer", rows_per_item=L, **mods(p[m])) for m in ("mods1", "mods2"))
    x1, h = ops.residual_norm(p["x"], p["y"], out_dtype=BF, **n1)
    t = h @ p["a"].T
    qkv = h @ p["w"].T + t @ p["b"].T
    q, k = ops.rotary(qkv[:, :N], qkv[:, N:N + NK], inv, **rot)
    v = qkv[:, N + NK:].contiguous()
    o, lse = ops.attention_lse(q, k, v, **attn)
    y2 = o @ p["wo"].T
    x2, h2 = ops.residual_norm(x1, y2, out_dtype=BF, **n2)

    g2 = ops.residual_norm_backward(up["h"], up["x"], x2, y2, **n2)
    do = g2.dy @ p["wo"]
    dqkv = torch.empty_like(qkv)
    dq, dk, _ = ops.attention_backward(do, q, k, v, o, lse, dv=dqkv[:, N + NK:], **attn)
    ops.rotary(dq, dk, inv, inverse=True, out_q=dqkv[:, :N], out_k=dqkv[:, N:N + NK], **rot)
    dt = dqkv @ p["b"]
    g1 = ops.residual_norm_backward(dqkv @ p["w"] + dt @ p["a"], g2.dx, x1, p["y"], **n1)
    return (x2, h2), {"x": g1.dx, "y": g1.dy, "mods1": torch.cat([g1.dshift, g1.dscale, g1.dgate], 1),
                      "mods2": torch.cat([g2.dshift, g2.dscale, g2.dgate], 1), "w": dqkv.T @ h, "a": dt.T @ h,
                      "b": dqkv.T @ t, "wo": g2.dy.T @ o}


def reference(p, up):
    p = {n: t.double().requires_grad_() for n, t in p.items()}
    item = torch.arange(ROWS, device=DEV) // L

    def step(x, y, m):
        m = {n: t[item] for n, t in mods(m).items()}
        x = x + m["gate"] * y
        n = torch.nn.functional.layer_norm(x, (C,), eps=1e-6)
        return x, n * (1 + m["scale"]) + m["shift"]

    def turn(t, heads):
        t = t.view(B, L, heads, D)
        f = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=DEV) / D)
        ang = torch.arange(L, dtype=torch.float64, device=DEV)[:, None, None] * f
        a, b = t.chunk(2, -1)
        return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin()], -1).transpose(1, 2)

    x1, h = step(p["x"], p["y"], p["mods1"])
    qkv = h @ (p["w"] + p["b"] @ p["a"]).T
    N, NK = H * D, HK * D
    q, k = turn(qkv[:, :N], H), turn(qkv[:, N:N + NK], HK).repeat_interleave(H // HK, 1)
    v = qkv[:, N + NK:].view(B, L, HK, D).transpose(1, 2).repeat_interleave(H // HK, 1)
    j = torch.arange(L, device=DEV)
    hidden = (j[None] > j[:, None]) | (j >= torch.tensor(LENS, device=DEV)[:, None, None, None])
    s = (q @ k.transpose(-1, -2) / math.sqrt(D)).masked_fill(hidden, float("-inf"))
    o = (s.softmax(-1) @ v).transpose(1, 2).reshape(ROWS, N)
    x2, h2 = step(x1, o @ p["wo"].T, p["mods2"])
    loss = (h2 * up["h"].double()).sum() + (x2 * up["x"].double()).sum()
    return (x2.detach(), h2.detach()), dict(zip(p, torch.autograd.grad(loss, list(p.values()))))


def test_block_forward_and_backward():
    ops = pkg("ops")
    p, up = make()
    (x, h), grads = block(ops, p, up, *plan(ops))
    (rx, rh), want = reference(p, up)
    pkg("device").Context.get(0).sync()

    def rel(a, b):
        return ((a.double() - b).norm() / b.norm()).item()

    # bf16 roundings on the longest path: h, t, its product, their sum, q and k turned, P, the output, y2 and
    # h2 forward; dy, do, dS, dq, the turned gradient, dt, three sums behind it and the result backward; each
    # at most half a step of what it rounds, none larger than the gradient it becomes a part of
    half = torch.finfo(BF).eps / 2
    assert rel(x, rx) < 10 * half and rel(h, rh) < 10 * half
    for n in want:
        assert grads[n].shape == want[n].shape and rel(grads[n], want[n]) < 20 * half, (n, rel(grads[n], want[n]) / half)


def test_block_captured_while_an_eager_step_lives():
    """A captured step replays with the bits of an eager one, with the eager step's tensors still alive."""
    ops = pkg("ops")
    p, up = make()
    const = plan(ops)
    keep = block(ops, p, up, *const)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(ops, p, up, *const)
    p["x"].copy_(randn(20, ROWS, C))
    graph.replay()
    want = block(ops, p, up, *const)
    torch.cuda.synchronize()
    assert torch.equal(out[0][1], want[0][1]) and not torch.equal(out[0][1], keep[0][1])
    for n in want[1]:
        assert torch.equal(out[1][n], want[1][n]), n
