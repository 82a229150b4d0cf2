"""The operators of a trained transformer block, as cases to measure: attention with its backward
pass, rotary positions, and the gated residual between two norms, forward and backward.

`run` has each operator twice: as the framework's call (`own`), and in elementary torch operations
in 32 bits, rounded once at the end; `exact` has its definition in 64 bits.

Formulas. Attention of one head: S = scale Q K^T over the visible keys (j < key_len[b], and j <= i
where causal), lse = ln sum exp S, P = exp(S - lse), O = P V; a row that sees no key has O = 0 and
lse = -inf. Backward from dO: dV = P^T dO, dS = P (dO V^T - rowsum(dO O)), dQ = scale dS K,
dK = scale dS^T Q, with dK and dV summed over the q heads that share a k/v head. Rotary: the pair
(x0, x1) at position p and frequency f becomes mscale (x0 cos pf - x1 sin pf, x1 cos pf + x0 sin pf);
the inverse turns by -pf. Residual norm: x' = x + alpha gate[item] post(y),
h = pre(x') (1 + scale[item]) + shift[item].
"""

from __future__ import annotations

import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a 77-token prompt through one layer of the causal text encoder (16 q heads over 8): latency
        {"name": "attn_prompt", "op": "attention", "B": 1, "H": 16, "group": 2, "D": 128, "Lq": 77, "Lk": 77,
         "causal": True, "pad": 0, "dtype": "bf16", "packed": False},
        # the adapter's cross-attention in a padded batch of four prompts, odd lengths, 64-wide heads
        {"name": "attn_adapter", "op": "attention", "B": 4, "H": 16, "group": 1, "D": 64, "Lq": 413, "Lk": 509,
         "causal": False, "pad": 131, "dtype": "f16", "packed": False},
        # the DiT's cross-attention at 1024x1024 on two prompts of different length
        {"name": "attn_cross", "op": "attention", "B": 2, "H": 16, "group": 1, "D": 128, "Lq": 4096, "Lk": 512,
         "causal": False, "pad": 187, "dtype": "bf16", "packed": False},
        # the DiT's self-attention at 1024x1024: 4096 tokens, q|k|v in one tensor and so their gradients
        {"name": "attn_self", "op": "attention", "B": 1, "H": 16, "group": 1, "D": 128, "Lq": 4096, "Lk": 4096,
         "causal": False, "pad": 0, "dtype": "bf16", "packed": True},
        # a long causal sequence with shared k/v heads
        {"name": "attn_long", "op": "attention", "B": 1, "H": 16, "group": 2, "D": 128, "Lq": 8192, "Lk": 8192,
         "causal": True, "pad": 0, "dtype": "bf16", "packed": False},
        # q and k of a short prompt: latency
        {"name": "rotary_prompt", "op": "rotary", "B": 1, "L": 77, "Hq": 16, "Hk": 8, "D": 128, "R": 128,
         "inverse": False, "interleaved": False, "scaling": "none", "factor": 1.0, "offset": 0, "dtype": "bf16"},
        # the gradient through the rotation of an image batch's q and k (the inverse rotation)
        {"name": "rotary_image_grad", "op": "rotary", "B": 2, "L": 4096, "Hq": 16, "Hk": 16, "D": 128, "R": 128,
         "inverse": True, "interleaved": False, "scaling": "ntk", "factor": 4.0, "offset": 0, "dtype": "f16"},
        # far positions of a long context, half of each head turned, adjacent pairs, fp32
        {"name": "rotary_far", "op": "rotary", "B": 1, "L": 16381, "Hq": 16, "Hk": 8, "D": 128, "R": 64,
         "inverse": False, "interleaved": True, "scaling": "yarn", "factor": 16.0, "offset": 900001, "dtype": "f32"},
        # between two sublayers of a short prompt, rms norms with weights: latency
        {"name": "norm_prompt", "op": "norm", "B": 1, "L": 77, "C": 1024, "backward": False, "post": "rms",
         "pre": "rms", "gated": False, "alpha": 1.0, "x": "f32", "y": "f32", "h": "bf16"},
        # between two sublayers of the DiT at 1024x1024: gate, residual, the next adaLN norm
        {"name": "norm_image", "op": "norm", "B": 1, "L": 4096, "C": 2048, "backward": False, "post": "none",
         "pre": "layer", "gated": True, "alpha": 1.0, "x": "f32", "y": "f16", "h": "f16"},
        # its backward pass on a batch of four images
        {"name": "norm_image_grad", "op": "norm", "B": 4, "L": 4096, "C": 2048, "backward": True, "post": "none",
         "pre": "layer", "gated": True, "alpha": 1.0, "x": "f32", "y": "bf16", "h": "bf16"},
        # rms norms on both sides of the block, a residual scale, 16-bit residual stream, odd rows
        {"name": "norm_sandwich_grad", "op": "norm", "B": 3, "L": 1531, "C": 1024, "backward": True, "post": "rms",
         "pre": "rms", "gated": False, "alpha": 0.5, "x": "bf16", "y": "bf16", "h": "bf16"},
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rotary", "norm"])
    if op == "attention":
        H = rng.choice([8, 16, 24])
        group = rng.choice([1, 1, 2, 4])
        causal = rng.random() < 0.4
        # two keys or more: behind a single key the gradients of q and k are 0, and what is left is rounding
        Lq = _spread(rng, 2 if causal else 1, 5600)
        Lk = Lq if Lq > 1 and rng.random() < 0.5 else _spread(rng, 2, 5600)
        B = rng.choice([1, 1, 2, 3])
        if B * H * Lq * Lk > 16 * 5600 * 5600:
            B, H = 1, 16
        return {"op": op, "B": B, "H": H, "group": group, "D": rng.choice([64, 128]), "Lq": Lq, "Lk": Lk,
                "causal": causal, "pad": rng.choice([0, _spread(rng, 1, Lk)]), "dtype": rng.choice(["bf16", "f16"]),
                "packed": Lq == Lk and group == 1}
    if op == "rotary":
        D = rng.choice([64, 128])
        B, L = rng.choice([1, 2, 3]), _spread(rng, 1, 5400)
        return {"op": op, "B": B, "L": L, "Hq": rng.choice([8, 16]), "Hk": rng.choice([1, 8]), "D": D,
                "R": rng.choice([D, D // 2, 20]), "inverse": rng.random() < 0.4, "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "yarn"]), "factor": float(rng.choice([2, 8, 32])),
                "offset": rng.choice([0, _spread(rng, 1, 1000000)]), "dtype": rng.choice(["bf16", "f16", "f32"])}
    B, L = rng.choice([1, 2, 5]), _spread(rng, 1, 4096)
    x = rng.choice(["f32", "f32", "bf16"])
    return {"op": op, "B": B, "L": L, "C": rng.choice([256, 1000, 1024, 2048, _spread(rng, 64, 2048)]),
            "backward": rng.random() < 0.6, "post": rng.choice(["none", "rms", "layer"]),
            "pre": rng.choice(["rms", "layer"]), "gated": rng.random() < 0.6, "alpha": rng.choice([1.0, 0.5]), "x": x,
            "y": rng.choice(["bf16", "f16", x]), "h": rng.choice(["bf16", "f16", "f32"])}


def _key_len(c):
    """Visible keys of each item of the padded batch: the first has all, each next one `pad` fewer."""
    return [max(0, c["Lk"] - b * c["pad"]) for b in range(c["B"])]


def _frequencies(R, scaling, factor, device):
    """Inverse frequencies [R / 2] in 64 bits (theta 1e4, trained for 4096 positions) and the output factor."""
    theta, i2 = 10000.0, torch.arange(0, R, 2, dtype=torch.float64, device=device)
    if scaling == "ntk":
        theta = theta * factor ** (R / (R - 2.0)) if R > 2 else theta
    inv = theta ** (-i2 / R)
    if scaling == "linear":
        inv = inv / factor
    if scaling == "yarn":
        turns = 4096.0 * inv / (2.0 * math.pi)          # turns within the trained length
        keep = ((turns - 1.0) / (32.0 - 1.0)).clamp(0.0, 1.0)   # 1: fast dims stay, 0: slow dims are stretched
        inv = inv * keep + inv / factor * (1.0 - keep)
    return inv, (0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0)


def prepare(case, seed):
    dv = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dv).manual_seed(int(seed))

    def randn(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=g, device=dv) * scale + shift).to(dtype)

    c = dict(case)
    s = {"case": c}
    if c["op"] == "attention":
        dt = DT[c["dtype"]]
        B, H, D, Hk = c["B"], c["H"], c["D"], c["H"] // c["group"]
        # q and k leave a per-head norm, v a projection; the gradient is small
        if c["packed"]:
            s["qkv"] = randn(B * c["Lq"], 3 * H * D, dtype=dt)
        else:
            s["q"] = randn(B * c["Lq"], H * D, dtype=dt)
            s["k"], s["v"] = randn(B * c["Lk"], Hk * D, dtype=dt), randn(B * c["Lk"], Hk * D, dtype=dt)
        s["dout"] = randn(B * c["Lq"], H * D, dtype=dt, scale=1.0 / 16)
        s["key_len"] = torch.tensor(_key_len(c), dtype=torch.int32, device=dv) if c["pad"] else None
    elif c["op"] == "rotary":
        rows = c["B"] * c["L"]
        s["q"], s["k"] = (randn(rows, c[h] * c["D"], dtype=DT[c["dtype"]]) for h in ("Hq", "Hk"))
        # every item of the batch has its own first position
        first = c["offset"] + 17 * torch.arange(c["B"], dtype=torch.int32, device=dv)[:, None]
        s["positions"] = (first + torch.arange(c["L"], dtype=torch.int32, device=dv)).reshape(-1).contiguous()
        s["inv_freq"], s["mscale"] = _frequencies(c["R"], c["scaling"], c["factor"], dv)
    else:
        rows, C, B = c["B"] * c["L"], c["C"], c["B"]
        s["y"] = randn(rows, C, dtype=DT[c["y"]], scale=0.7)
        s["x"] = randn(rows, C, dtype=DT[c["x"]], scale=2.0, shift=0.25)   # the residual stream: x, or x' behind it
        s["post_w"] = randn(C, scale=0.1, shift=1.0) if c["post"] != "none" else None
        s["pre_w"] = randn(C, scale=0.1, shift=1.0) if c["pre"] == "rms" else None
        mods = randn(B, 3 * C, scale=0.3) if c["gated"] else None           # shift | scale | gate of each item
        s["shift"], s["scale"], s["gate"] = (mods[:, i * C:(i + 1) * C] if c["gated"] else None for i in range(3))
        if c["backward"]:
            s["dh"] = randn(rows, C, dtype=DT[c["h"]], scale=0.05)
            s["dx"] = randn(rows, C, dtype=DT[c["x"]], scale=0.05)
    return s


def run(state):
    return {"attention": _attention, "rotary": _rotary, "norm": _norm}[state["case"]["op"]](state)


# ------------------------------------------------------------------------------------ attention

def _split(s):
    """q, k, v as [B, H, L, D] views of the state's tensors, and dout."""
    c = s["case"]
    B, H, D = c["B"], c["H"], c["D"]
    if c["packed"]:
        q, k, v = s["qkv"].view(B, c["Lq"], 3, H, D).permute(2, 0, 3, 1, 4)
    else:
        q = s["q"].view(B, c["Lq"], H, D).transpose(1, 2)
        k, v = (s[n].view(B, c["Lk"], H // c["group"], D).transpose(1, 2) for n in ("k", "v"))
    return q, k, v, s["dout"].view(B, c["Lq"], H, D).transpose(1, 2)


def _attention(s):
    c = s["case"]
    B, H, D, Lq, Lk, group = c["B"], c["H"], c["D"], c["Lq"], c["Lk"], c["group"]
    Hk = H // group
    if own:
        ops = _ops()
        kw = dict(Lq=Lq, Lk=Lk, H=H, D=D, batch=B, key_len=s["key_len"], group=group, causal=c["causal"])
        if c["packed"]:
            x, C = s["qkv"], H * D
            q = k = v = x
            dx = torch.empty_like(x)
            kw |= dict(ldq=3 * C, ldk=3 * C, ldv=3 * C, q_off=0, k_off=C, v_off=2 * C, q_bstride=Lq * 3 * C,
                       k_bstride=Lk * 3 * C, v_bstride=Lk * 3 * C)
            grads = dict(dq=dx[:, :C], dk=dx[:, C:2 * C], dv=dx[:, 2 * C:])
        else:
            q, k, v, grads = s["q"], s["k"], s["v"], {}
            kw |= dict(q_bstride=Lq * H * D, k_bstride=Lk * Hk * D, v_bstride=Lk * Hk * D)
        out, lse = ops.attention_lse(q, k, v, **kw)
        dq, dk, dv = ops.attention_backward(s["dout"], q, k, v, out, lse, **kw, **grads)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}

    dt, scale = DT[c["dtype"]], 1.0 / math.sqrt(D)
    q, k, v, do = (t.float() for t in _split(s))
    q, do = (t.reshape(B, Hk, group, Lq, D) for t in (q, do))
    k, v = k[:, :, None], v[:, :, None]
    sc = (q @ k.transpose(-1, -2)) * scale
    i, j = torch.arange(Lq, device=q.device)[:, None], torch.arange(Lk, device=q.device)[None]
    hidden = (j > i) if c["causal"] else torch.zeros(Lq, Lk, dtype=torch.bool, device=q.device)
    hidden = hidden.expand(B, 1, 1, Lq, Lk)
    if s["key_len"] is not None:
        hidden = hidden | (j >= s["key_len"][:, None, None]).view(B, 1, 1, 1, Lk)
    sc = sc.masked_fill(hidden, float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isfinite(m), m, 0.0)
    sc = torch.exp(sc - m)                              # masked: exactly 0
    total = sc.sum(-1, keepdim=True)
    lse = (m + torch.log(total))[..., 0]
    p = sc / torch.where(total > 0, total, 1.0)
    out = p @ v
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = p * (do @ v.transpose(-1, -2) - (do * out).sum(-1, keepdim=True))
    dq = (ds @ k) * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2) * scale

    def rows(t):                                        # [B, heads, L, D] -> [B L, heads D]
        return t.transpose(1, 2).reshape(t.shape[0] * t.shape[2], -1).to(dt)

    out, dq = (rows(t.reshape(B, H, Lq, D)) for t in (out, dq))
    return {"out": out, "lse": lse.reshape(B, H, Lq), "dq": dq, "dk": rows(dk), "dv": rows(dv)}


def _attention_exact(s):
    c = s["case"]
    B, H, D, Lq, Lk, group = c["B"], c["H"], c["D"], c["Lq"], c["Lk"], c["group"]
    q, k, v, do = _split(s)
    f64 = dict(dtype=torch.float64, device=q.device)
    out, dq = torch.zeros(B, Lq, H, D, **f64), torch.zeros(B, Lq, H, D, **f64)
    dk, dv = torch.zeros(B, Lk, H // group, D, **f64), torch.zeros(B, Lk, H // group, D, **f64)
    lse = torch.full((B, H, Lq), float("-inf"), **f64)
    for b, n in enumerate(_key_len(c) if c["pad"] else [Lk] * B):
        if n == 0:
            continue
        for h in range(H):
            qh, kh, vh, dh = q[b, h].double(), k[b, h // group, :n].double(), v[b, h // group, :n].double(), do[b, h].double()
            sc = torch.mm(qh, kh.T) / D ** 0.5
            if c["causal"]:
                sc.masked_fill_(torch.ones(Lq, n, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
            lse[b, h] = torch.logsumexp(sc, 1)
            p = sc.sub_(lse[b, h][:, None]).exp_()
            out[b, :, h] = torch.mm(p, vh)
            dv[b, :n, h // group] += torch.mm(p.T, dh)
            ds = torch.mm(dh, vh.T).sub_((dh * out[b, :, h]).sum(1)[:, None]).mul_(p) / D ** 0.5
            dq[b, :, h] = torch.mm(ds, kh)
            dk[b, :n, h // group] += torch.mm(ds.T, qh)
    return {"out": out.view(B * Lq, -1), "lse": lse, "dq": dq.view(B * Lq, -1), "dk": dk.view(B * Lk, -1),
            "dv": dv.view(B * Lk, -1)}


# ------------------------------------------------------------------------------------ rotary

def _rotary(s):
    c = s["case"]
    if own:
        return _ops().rotary(s["q"], s["k"], s["inv_freq"], Hq=c["Hq"], Hk=c["Hk"], D=c["D"], positions=s["positions"],
                             mscale=s["mscale"], interleaved=c["interleaved"], inverse=c["inverse"])
    angle = s["positions"].double()[:, None, None] * s["inv_freq"]         # [rows, 1, R / 2], 64 bits
    cos, sin = (angle.cos() * s["mscale"]).float(), (angle.sin() * s["mscale"]).float()
    if c["inverse"]:
        sin = -sin

    def turn(x, H):
        R = c["R"]
        x3 = x.view(-1, H, c["D"]).float()
        a, rest = x3[..., :R], x3[..., R:]
        x0, x1 = (a[..., 0::2], a[..., 1::2]) if c["interleaved"] else (a[..., :R // 2], a[..., R // 2:])
        y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
        y = torch.stack([y0, y1], -1).flatten(-2) if c["interleaved"] else torch.cat([y0, y1], -1)
        return torch.cat([y, rest], -1).reshape(x.shape).to(x.dtype)

    return turn(s["q"], c["Hq"]), turn(s["k"], c["Hk"])


def _rotary_exact(s):
    c = s["case"]
    z = torch.polar(torch.full((1,), float(s["mscale"]), dtype=torch.float64, device=s["q"].device),
                    s["positions"].double()[:, None] * s["inv_freq"] * (-1.0 if c["inverse"] else 1.0))
    got = []
    for x, H in ((s["q"], c["Hq"]), (s["k"], c["Hk"])):
        y = x.double().view(-1, H, c["D"]).clone()
        n = c["R"] // 2
        at = [slice(0, c["R"], 2), slice(1, c["R"], 2)] if c["interleaved"] else [slice(0, n), slice(n, 2 * n)]
        w = torch.complex(y[..., at[0]].contiguous(), y[..., at[1]].contiguous()) * z[:, None]
        y[..., at[0]], y[..., at[1]] = w.real, w.imag
        got.append(y.view(x.shape))
    return tuple(got)


# ------------------------------------------------------------------------------------ residual norm

EPS = 1e-6


def _norm(s):
    c = s["case"]
    B, C = c["B"], c["C"]
    if own:
        ops = _ops()
        kw = dict(alpha=c["alpha"], gate=s["gate"], post=None if c["post"] == "none" else c["post"], post_w=s["post_w"],
                  pre=c["pre"], pre_w=s["pre_w"], scale=s["scale"], shift=s["shift"], eps=EPS, rows_per_item=c["L"])
        if not c["backward"]:
            return ops.residual_norm(s["x"], s["y"], out_dtype=DT[c["h"]], **kw)
        return [t for t in ops.residual_norm_backward(s["dh"], s["dx"], s["x"], s["y"], **kw) if t is not None]

    def per_item(m, one=0.0):                           # [B, C] -> [B, 1, C] against [B, L, C]
        return m[:, None] if m is not None else one

    def norm(t, kind):                                  # the normalised rows and 1 / deviation
        t = t - t.mean(-1, keepdim=True) if kind == "layer" else t
        r = torch.rsqrt((t * t).mean(-1, keepdim=True) + EPS)
        return t * r, r

    def back(g, n, r, kind):                            # the gradient through norm()
        g = g - g.mean(-1, keepdim=True) if kind == "layer" else g
        return (g - n * (g * n).mean(-1, keepdim=True)) * r

    x, y = s["x"].float().view(B, -1, C), s["y"].float().view(B, -1, C)
    gate = per_item(s["gate"], 1.0) * c["alpha"]
    post_w, pre_w = (1.0 if s[w] is None else s[w] for w in ("post_w", "pre_w"))
    m, rm = norm(y, c["post"]) if c["post"] != "none" else (y, None)
    if not c["backward"]:
        x = x + gate * (m * post_w)
        h = norm(x, c["pre"])[0] * pre_w * (1.0 + per_item(s["scale"])) + per_item(s["shift"])
        return x.view(-1, C).to(DT[c["x"]]), h.view(-1, C).to(DT[c["h"]])
    dh, dx = s["dh"].float().view(B, -1, C), s["dx"].float().view(B, -1, C)
    n, rn = norm(x, c["pre"])
    dx = dx + back(dh * (1.0 + per_item(s["scale"])) * pre_w, n, rn, c["pre"])
    du = dx * gate
    dy = back(du * post_w, m, rm, c["post"]) if rm is not None else du
    got = [dx.view(-1, C).to(DT[c["x"]]), dy.view(-1, C).to(DT[c["y"]])]
    if c["gated"]:
        got.append((dx * (m * post_w)).sum(1) * c["alpha"])
    if s["post_w"] is not None:
        got.append((du * m).sum((0, 1)))
    if s["pre_w"] is not None:
        got.append((dh * (1.0 + per_item(s["scale"])) * n).sum((0, 1)))
    if c["gated"]:
        got += [(dh * n * pre_w).sum(1), dh.sum(1)]
    return got


def _norm_exact(s):
    """The forward in 64 bits; the backward as derivatives of sum(h dh + x' dx) by automatic differentiation."""
    c = s["case"]
    C, item = c["C"], torch.arange(c["B"], device=s["y"].device).repeat_interleave(c["L"])
    leaf = {n: s[n].double().detach().requires_grad_(c["backward"])
            for n in ("x", "y", "gate", "post_w", "pre_w", "scale", "shift") if s[n] is not None}

    def normalise(t, kind):
        if kind == "layer":
            t = t - t.mean(1, keepdim=True)
        return t / (t.square().mean(1, keepdim=True) + EPS).sqrt()

    u = leaf["y"] if c["post"] == "none" else normalise(leaf["y"], c["post"]) * leaf["post_w"]
    if c["gated"]:
        u = leaf["gate"][item] * u
    u = c["alpha"] * u
    x = leaf["x"] if c["backward"] else leaf["x"] + u
    h = normalise(x, c["pre"])
    if "pre_w" in leaf:
        h = h * leaf["pre_w"]
    if c["gated"]:
        h = h * (1 + leaf["scale"][item]) + leaf["shift"][item]
    if not c["backward"]:
        return x, h
    # the state's x is x' itself: first its gradient, then that of x' = (what was) + u
    first = [n for n in ("x", "pre_w", "scale", "shift") if n in leaf]
    got = dict(zip(first, torch.autograd.grad((h * s["dh"].double()).sum(), [leaf[n] for n in first])))
    got["x"] = got["x"] + s["dx"].double()
    second = [n for n in ("y", "gate", "post_w") if n in leaf]
    got |= dict(zip(second, torch.autograd.grad((u * got["x"]).sum(), [leaf[n] for n in second])))
    return [got[n] for n in ("x", "y", "gate", "post_w", "pre_w", "scale", "shift") if n in got]


# ------------------------------------------------------------------------------------ all of them

def _ops():
    import importlib

    return importlib.import_module("anima-studio_b200.ops")


def _visible_pairs(c):
    """(query, key) pairs that the masks leave, of all items and one head."""
    pairs = 0
    for n in _key_len(c) if c["pad"] else [c["Lk"]] * c["B"]:
        m = min(n, c["Lq"])                             # causal: row i sees min(i + 1, n) keys
        pairs += m * (m + 1) // 2 + (c["Lq"] - m) * n if c["causal"] else c["Lq"] * n
    return pairs


def work(case):
    c = case
    if c["op"] == "attention":
        q, kv = c["B"] * c["Lq"] * c["H"] * c["D"], c["B"] * c["Lk"] * (c["H"] // c["group"]) * c["D"]
        # reads q, k, v, dout; writes out, lse, dq, dk, dv; two products forward, five backward
        return {"bytes": 2 * (4 * q + 4 * kv) + 4 * c["B"] * c["Lq"] * c["H"],
                "flops": 14 * _visible_pairs(c) * c["H"] * c["D"]}
    size = {"bf16": 2, "f16": 2, "f32": 4}
    if c["op"] == "rotary":
        rows = c["B"] * c["L"]
        n = rows * (c["Hq"] + c["Hk"])
        return {"bytes": 2 * n * c["D"] * size[c["dtype"]] + 4 * rows, "flops": 3 * n * c["R"]}
    n = c["B"] * c["L"] * c["C"]
    small = 4 * c["C"] * ((3 * c["B"] if c["gated"] else 0) + (c["post"] != "none") + (c["pre"] == "rms"))
    if not c["backward"]:
        return {"bytes": n * (2 * size[c["x"]] + size[c["y"]] + size[c["h"]]) + small, "flops": 12 * n}
    return {"bytes": n * (3 * size[c["x"]] + 2 * size[c["y"]] + size[c["h"]]) + 2 * small, "flops": 30 * n}


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _attention_exact, "rotary": _rotary_exact, "norm": _norm_exact}[case["op"]](s)
