"""The operator surface of the reference's app/gpu/ops.js, on the B200 kernels of libanima_b200.

Activations follow the reference's conventions (row-major, fp32 unless a fused path says
otherwise); names and argument meanings mirror ops.js, each function cites the line it stands in
for. Two B200-specific forms are added for the fused path the DiT uses:

  QuantRows   rotated + per-token quantized rows, x ~= scale * (hi + lo / 254) (lo optional);
              the "xr" input of a ConvRot linear in the reference (ops.js:48-54)
  layernorm_mod_quant / rotate_quant   produce QuantRows directly from the norm / the rotation

Everything runs on the current torch stream of the tensors' device; nothing falls back to the CPU.
"""

from __future__ import annotations

import ctypes as C
import math
from dataclasses import dataclass
from typing import NamedTuple

import torch

from . import device as dev
from .device import ctx_for, ptr


@dataclass
class QuantRows:
    """Per-token quantized rotated activations [rows, cols]: x ~= scale[:, None] * (hi + lo / 254)."""

    hi: torch.Tensor
    lo: torch.Tensor | None
    scale: torch.Tensor

    @property
    def rows(self):
        return self.hi.shape[0]

    @property
    def cols(self):
        return self.hi.shape[1]

    @staticmethod
    def empty(rows: int, cols: int, planes: int = 2, device=None) -> "QuantRows":
        hi = torch.empty(rows, cols, dtype=torch.int8, device=device)
        lo = torch.empty(rows, cols, dtype=torch.int8, device=device) if planes == 2 else None
        return QuantRows(hi, lo, torch.empty(rows, dtype=torch.float32, device=device))

    def c(self) -> dev.QAct:
        return dev.QAct(self.rows, self.cols, self.hi.stride(0), self.hi.data_ptr(),
                        self.lo.data_ptr() if self.lo is not None else 0, self.scale.data_ptr())

    def dequant(self) -> torch.Tensor:
        """fp32 rows this encodes (for tests and debugging)."""
        x = self.hi.float()
        if self.lo is not None:
            x = x + self.lo.float() / 254.0
        return x * self.scale[:, None]


def _dt(t: torch.Tensor) -> int:
    return dev.DTYPE_CODE[t.dtype]


def _contig_rows(t: torch.Tensor):
    if t.dim() != 2 or t.stride(1) != 1:
        raise dev.AnimaError(1, "expected a 2-D tensor with contiguous rows")


def _rows(fn: str, name: str, t: torch.Tensor, rows: int, cols: int, dtype=None, device=None, exact: bool = False) -> int:
    """Refuse what is not `rows` contiguous rows of at least (exact: just) `cols` columns of a kernel
    type, on device index `device`; returns the row stride. (Small calls are bound by the host: each
    attribute of a tensor is asked for once.)"""
    shape, st, dt = t.shape, t.stride(), t.dtype
    if len(shape) != 2 or shape[0] != rows or (shape[1] != cols if exact else shape[1] < cols):
        raise dev.AnimaError(1, f"{fn}: {name} is {tuple(shape)}, expected [{rows}, {cols}]")
    if rows > _MOST or cols > _MOST:
        raise dev.AnimaError(1, f"{fn}: {name} is [{rows}, {cols}], sizes end at 2^30")
    if st[1] != 1 and shape[1] > 1:
        raise dev.AnimaError(1, f"{fn}: {name} needs contiguous rows (strides {st})")
    if dt not in _FLOATS or (dtype is not None and dt is not dtype):
        raise dev.AnimaError(1, f"{fn}: {name} is {dt}" + (f", expected {dtype}" if dtype is not None else ""))
    if device is not None and t.get_device() != device:
        raise dev.AnimaError(1, f"{fn}: {name} is on {t.device}, expected device {device}")
    return st[0] if rows > 1 else shape[1]  # a single row's stride says nothing


_MOST = 2 ** 30  # sizes beyond are refused here: ctypes would cut a C int's upper bits off without a word
_FLOATS = frozenset((torch.float32, torch.bfloat16, torch.float16))


def _vector(fn: str, name: str, t: torch.Tensor, n: int, dtype, device: int):
    """Refuse what is not a dense vector of n elements of `dtype` on device index `device`."""
    shape = t.shape
    if len(shape) != 1 or shape[0] != n or t.dtype is not dtype or not t.is_contiguous() or t.get_device() != device:
        raise dev.AnimaError(1, f"{fn}: {name} has to be a dense {dtype} [{n}] on device {device}, is {t.dtype} "
                                f"{tuple(t.shape)} on {t.device}")


# ----------------------------------------------------------------------------- rotation / norms

def rotate(x: torch.Tensor) -> torch.Tensor:
    """ConvRot input rotation, y = x H per 256 features (ops.js:38-44)."""
    x2 = x.reshape(-1, x.shape[-1])
    y = torch.empty_like(x2, dtype=torch.float32)
    ctx_for(x).call("anima_rotate", ptr(x2), _dt(x2), x2.shape[0], x2.shape[1], x2.stride(0), ptr(y), dev.ANIMA_F32)
    return y.view(x.shape)


def rotate_quant(x: torch.Tensor, planes: int = 2, out: QuantRows | None = None, act: str | None = None) -> QuantRows:
    """rotate() fused with per-token quantization (input fp32/bf16/fp16 rows); act="gelu" applies
    the MLP activation first (for a layer1 GEMM that stored its pre-activation)."""
    _contig_rows(x)
    q = out or QuantRows.empty(x.shape[0], x.shape[1], planes, x.device)
    qa = q.c()
    if act:
        ctx_for(x).call("anima_act_rotate_quant", ptr(x), _dt(x), x.shape[0], x.shape[1], x.stride(0), dev.ACT[act],
                        C.byref(qa))
    else:
        ctx_for(x).call("anima_rotate_quant", ptr(x), _dt(x), x.shape[0], x.shape[1], x.stride(0), C.byref(qa))
    return q


def quant_rows(x: torch.Tensor, planes: int = 2, out: QuantRows | None = None) -> QuantRows:
    """Per-token quantization of already-rotated rows."""
    _contig_rows(x)
    q = out or QuantRows.empty(x.shape[0], x.shape[1], planes, x.device)
    qa = q.c()
    ctx_for(x).call("anima_quant_rows", ptr(x), _dt(x), x.shape[0], x.shape[1], x.stride(0), C.byref(qa))
    return q


def layernorm_mod(x: torch.Tensor, mod: torch.Tensor, shift_off: int, scale_off: int, cols: int,
                  rotate: bool = False, eps: float = 1e-6, out_dtype=torch.float32) -> torch.Tensor:
    """y = LN(x) * (1 + mod[scale_off:]) + mod[shift_off:] (+ ConvRot) (ops.js:129-137)."""
    rows = x.numel() // cols
    y = torch.empty(rows, cols, dtype=out_dtype, device=x.device)
    ctx_for(x).call("anima_layernorm_mod", ptr(x), rows, cols, ptr(mod), shift_off, scale_off, C.c_float(eps),
                    1 if rotate else 0, ptr(y), dev.DTYPE_CODE[out_dtype])
    return y


def layernorm_mod_quant(x: torch.Tensor, mod: torch.Tensor, shift_off: int, scale_off: int, cols: int,
                        planes: int = 2, eps: float = 1e-6, out: QuantRows | None = None) -> QuantRows:
    """layernorm_mod(rotate=True) fused with per-token quantization: the "xr" a ConvRot linear takes."""
    rows = x.numel() // cols
    q = out or QuantRows.empty(rows, cols, planes, x.device)
    qa = q.c()
    ctx_for(x).call("anima_layernorm_mod_quant", ptr(x), rows, cols, ptr(mod), shift_off, scale_off,
                    C.c_float(eps), C.byref(qa))
    return q


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, cols: int, eps: float = 1e-6, out=None,
            out_dtype=None) -> torch.Tensor:
    """y = x * rsqrt(mean(x^2) + eps) * w over rows of `cols` (ops.js:111-117)."""
    rows = x.numel() // cols
    y = out if out is not None else torch.empty(x.shape, dtype=out_dtype or x.dtype, device=x.device)
    ctx_for(x).call("anima_rmsnorm", ptr(x), _dt(x), rows, cols, ptr(weight), C.c_float(eps), ptr(y), _dt(y))
    return y


def qk_norm_rope(qkv: torch.Tensor, qn: torch.Tensor, kn: torch.Tensor, cs: torch.Tensor, L: int, H: int, D: int,
                 eps: float = 1e-6):
    """In-place per-head RMSNorm + RoPE on the q and k parts of qkv [L, 3 H D] (ops.js:140-145).
    cs: cos table [rows, D/2] followed by the sin table (rows = L or a divisor pattern)."""
    rows = cs.numel() // D
    ctx_for(qkv).call("anima_qk_norm_rope", ptr(qkv), _dt(qkv), L, H, D, qkv.stride(0), ptr(qn), ptr(kn), ptr(cs),
                      rows, C.c_float(eps))


def rope(x: torch.Tensor, cs: torch.Tensor, L: int, H: int, D: int, row_stride: int | None = None, col_off: int = 0):
    """In-place split-half RoPE on x viewed as [L, H, D] (ops.js:148-152)."""
    rows = cs.numel() // D
    ctx_for(x).call("anima_rope", ptr(x), _dt(x), L, H, D, row_stride or H * D, col_off, ptr(cs), rows)


def rotary_freqs(dim: int, theta: float = 10000.0, *, scaling: str | None = None, factor: float = 1.0,
                 original_len: int = 4096, beta_fast: float = 32.0, beta_slow: float = 1.0,
                 device="cuda") -> tuple[torch.Tensor, float]:
    """Inverse frequencies (fp64 [dim / 2]) and output factor for rotary(): theta^(-2i / dim), and for
    contexts `factor` times the trained original_len
      "linear"  every frequency divided by factor;
      "ntk"     theta raised to theta * factor^(dim / (dim - 2)): the slowest pair is stretched by
                factor, the fastest not at all;
      "yarn"    pairs that turn more than beta_fast times within original_len stay, those below
                beta_slow turns are divided by factor, a linear ramp over the turns between; outputs
                multiplied by 0.1 ln(factor) + 1.
    Made on the host: once, not inside a stream capture. No reference counterpart: its RoPE is a table of
    fixed theta (common.js:26-52)."""
    if dim < 2 or dim % 2 or not theta > 0 or not factor > 0:
        raise dev.AnimaError(1, f"rotary_freqs: dim {dim} (even, at least 2), theta {theta}, factor {factor}")
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise dev.AnimaError(1, f"rotary_freqs: scaling {scaling!r} (None, 'linear', 'ntk' or 'yarn')")
    if scaling == "ntk" and dim > 2:
        theta = theta * factor ** (dim / (dim - 2))
    inv = theta ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    mscale = 1.0
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        if not beta_fast > beta_slow or original_len <= 0:
            raise dev.AnimaError(1, f"rotary_freqs: beta_fast {beta_fast} has to exceed beta_slow {beta_slow}, "
                                    f"original_len {original_len} be positive")
        turns = original_len * inv / (2.0 * math.pi)
        keep = ((turns - beta_slow) / (beta_fast - beta_slow)).clamp(0.0, 1.0)
        inv = inv * keep + inv / factor * (1.0 - keep)
        mscale = 0.1 * math.log(factor) + 1.0
    return inv.to(device), mscale


def rotary(q: torch.Tensor, k: torch.Tensor | None, inv_freq: torch.Tensor, *, Hq: int, D: int, Hk: int = 0,
           positions: torch.Tensor | None = None, offset: int = 0, rows_per_item: int | None = None,
           mscale: float = 1.0, interleaved: bool = False, inverse: bool = False, out_q: torch.Tensor | None = None,
           out_k: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor | None]:
    """Rotary positions on q [rows, >= Hq D] and k [rows, >= Hk D] (or None) in one launch, angles from
    positions and frequencies (rope() is the table form). The first 2 len(inv_freq) dims of each head
    are turned and multiplied by mscale (rotary_freqs gives both), in pairs (i, i + R/2), or
    (2i, 2i + 1) when interleaved; the other dims are copied. Row r stands at positions[r] (int32), or
    at offset + r % rows_per_item (default: all rows are one item). inverse: the transposed rotation,
    for gradients. Returns (out_q, out_k), new tensors unless given; out_q may be q itself."""
    rows, dt, at, R = q.shape[0], q.dtype, q.get_device(), inv_freq.shape[0] * 2
    if R > _MOST:
        raise dev.AnimaError(1, f"rotary: {R} rotated dims")
    a = dev.RotaryArgs(dtype=dev.DTYPE_CODE.get(dt, -1), rows=rows, D=D, R=R, Hq=Hq, mscale=mscale, offset=offset,
                       rows_per_item=min(rows_per_item or rows, rows) or 1, interleaved=interleaved, inverse=inverse)
    a.ldq = _rows("rotary", "q", q, rows, Hq * D)
    if out_q is None:
        out_q, a.ldoq = torch.empty((rows, Hq * D), dtype=dt, device=q.device), Hq * D
    else:
        a.ldoq = _rows("rotary", "out_q", out_q, rows, Hq * D, dt, at)
    a.q, a.out_q, a.inv_freq = q.data_ptr(), out_q.data_ptr(), inv_freq.data_ptr()
    if k is not None:
        a.ldk, a.Hk = _rows("rotary", "k", k, rows, Hk * D, dt, at), Hk
        if out_k is None:
            out_k, a.ldok = torch.empty((rows, Hk * D), dtype=dt, device=q.device), Hk * D
        else:
            a.ldok = _rows("rotary", "out_k", out_k, rows, Hk * D, dt, at)
        a.k, a.out_k = k.data_ptr(), out_k.data_ptr()
    elif Hk or out_k is not None:
        raise dev.AnimaError(1, "rotary: Hk or out_k without k")
    _vector("rotary", "inv_freq", inv_freq, R // 2, torch.float64, at)
    if positions is not None:
        _vector("rotary", "positions", positions, rows, torch.int32, at)
        a.positions = positions.data_ptr()
    ctx_for(q).call("anima_rotary", C.byref(a))
    return out_q, out_k


NORM_KIND = {None: 0, "rms": 1, "layer": 2}


def _residual_norm_args(fn, x, y, alpha, gate, post, post_w, pre, pre_w, scale, shift, eps, rows_per_item):
    """The arguments that the forward and the backward share; x: the residual stream's tensor."""
    if post not in NORM_KIND or pre not in ("rms", "layer"):
        raise dev.AnimaError(1, f"{fn}: post {post!r} (None, 'rms' or 'layer'), pre {pre!r} ('rms' or 'layer')")
    if x.dim() != 2:
        raise dev.AnimaError(1, f"{fn}: x has to be a 2-D tensor of rows")
    (rows, cols), at = x.shape, x.get_device()
    L = rows_per_item or max(rows, 1)
    if L < 0 or rows % L:
        raise dev.AnimaError(1, f"{fn}: {rows} rows are not items of {L} rows")
    items = rows // L
    a = dev.ResidualNormArgs(rows=rows, cols=cols, rows_per_item=L, post=NORM_KIND[post], pre=NORM_KIND[pre], alpha=alpha,
                             eps=eps)
    a.ldy = _rows(fn, "y", y, rows, cols, None, at, exact=True)
    a.x_dtype, a.y_dtype, a.y = dev.DTYPE_CODE.get(x.dtype, -1), _dt(y), y.data_ptr()
    for name, m in (("gate", gate), ("scale", scale), ("shift", shift)):
        if m is None:
            continue
        if m.dim() == 1:
            _vector(fn, name, m, cols, torch.float32, at)
            if items > 1:
                raise dev.AnimaError(1, f"{fn}: {name} [{cols}] for {items} items of rows (a [items, cols] tensor)")
            ld = cols
        else:
            ld = _rows(fn, name, m, items, cols, torch.float32, at, exact=True)
        setattr(a, name, m.data_ptr())
        setattr(a, "ld_" + name, ld)
    if post_w is not None:
        _vector(fn, "post_w", post_w, cols, torch.float32, at)
        a.post_w = post_w.data_ptr()
    if pre_w is not None:
        _vector(fn, "pre_w", pre_w, cols, torch.float32, at)
        a.pre_w = pre_w.data_ptr()
    return a, rows, cols, at


def residual_norm(x: torch.Tensor, y: torch.Tensor, *, alpha: float = 1.0, gate: torch.Tensor | None = None,
                  post: str | None = None, post_w: torch.Tensor | None = None, pre: str = "layer",
                  pre_w: torch.Tensor | None = None, scale: torch.Tensor | None = None,
                  shift: torch.Tensor | None = None, eps: float = 1e-6, rows_per_item: int | None = None, out_dtype=None,
                  x_out: torch.Tensor | None = None, h: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """The step from one sublayer to the next in one pass: u = post(y) * post_w, x_out = x + alpha *
    gate * u, h = pre(x_out) * pre_w * (1 + scale) + shift; returns (x_out, h). x, y [rows, cols], each
    fp32, bf16 or fp16; post: None, "rms" or "layer"; pre: "rms" or "layer"; gate, scale, shift: fp32
    [items, cols] (rows may be strided: slices of a modulation tensor) or [cols] for one item, row r
    taking those of item r // rows_per_item; post_w, pre_w: fp32 [cols]. h has out_dtype (default
    x's). x_out may be x itself. The reference runs the gate and the adaLN norm apart (dit.js:261-314)."""
    fn = "residual_norm"
    a, rows, cols, at = _residual_norm_args(fn, x, y, alpha, gate, post, post_w, pre, pre_w, scale, shift, eps,
                                            rows_per_item)
    dt, a.ldx = x.dtype, _rows(fn, "x", x, rows, cols)
    if x_out is None:
        x_out, a.ldx_out = torch.empty((rows, cols), dtype=dt, device=x.device), cols
    else:
        a.ldx_out = _rows(fn, "x_out", x_out, rows, cols, dt, at, exact=True)
    if h is None:
        h, a.ldh = torch.empty((rows, cols), dtype=out_dtype or dt, device=x.device), cols
        if h.dtype not in _FLOATS:
            raise dev.AnimaError(1, f"{fn}: out_dtype {out_dtype}")
    elif out_dtype not in (None, h.dtype):
        raise dev.AnimaError(1, f"{fn}: h is {h.dtype}, out_dtype {out_dtype}")
    else:
        a.ldh = _rows(fn, "h", h, rows, cols, None, at, exact=True)
    a.h_dtype, a.x, a.x_out, a.h = _dt(h), x.data_ptr(), x_out.data_ptr(), h.data_ptr()
    ctx_for(x).call("anima_residual_norm", C.byref(a))
    return x_out, h


class ResidualNormGrads(NamedTuple):
    """Gradients of residual_norm's inputs; None where the parameter is None. dgate, dscale and dshift
    have one row per item (the caller sums them where it gave several items one vector)."""

    dx: torch.Tensor
    dy: torch.Tensor
    dgate: torch.Tensor | None
    dpost_w: torch.Tensor | None
    dpre_w: torch.Tensor | None
    dscale: torch.Tensor | None
    dshift: torch.Tensor | None


def residual_norm_backward(dh: torch.Tensor, dx_out: torch.Tensor | None, x_out: torch.Tensor, y: torch.Tensor, *,
                           alpha: float = 1.0, gate: torch.Tensor | None = None, post: str | None = None,
                           post_w: torch.Tensor | None = None, pre: str = "layer", pre_w: torch.Tensor | None = None,
                           scale: torch.Tensor | None = None, shift: torch.Tensor | None = None, eps: float = 1e-6,
                           rows_per_item: int | None = None, dx: torch.Tensor | None = None,
                           dy: torch.Tensor | None = None) -> ResidualNormGrads:
    """The backward pass of residual_norm: dh is the gradient of h, dx_out the gradient that reaches
    x_out from behind (None: none), x_out and y are as the forward left and had them, the rest are the
    forward's arguments. dx (x's type) may be dx_out itself, dy (y's type) y itself. Statistics are
    computed again in fp32 from y and the stored x_out; column sums are in fp32 and of fixed order."""
    fn = "residual_norm_backward"
    a, rows, cols, at = _residual_norm_args(fn, x_out, y, alpha, gate, post, post_w, pre, pre_w, scale, shift, eps,
                                            rows_per_item)
    dt, dv = x_out.dtype, x_out.device
    a.ldx_out, a.lddh = _rows(fn, "x_out", x_out, rows, cols), _rows(fn, "dh", dh, rows, cols, None, at, exact=True)
    if dx is None:
        dx, a.lddx = torch.empty((rows, cols), dtype=dt, device=dv), cols
    else:
        a.lddx = _rows(fn, "dx", dx, rows, cols, dt, at, exact=True)
    if dy is None:
        dy, a.lddy = torch.empty((rows, cols), dtype=y.dtype, device=dv), cols
    else:
        a.lddy = _rows(fn, "dy", dy, rows, cols, y.dtype, at, exact=True)
    a.h_dtype, a.x_out, a.dh, a.dx, a.dy = _dt(dh), x_out.data_ptr(), dh.data_ptr(), dx.data_ptr(), dy.data_ptr()
    if dx_out is not None:
        a.lddx_out, a.dx_out = _rows(fn, "dx_out", dx_out, rows, cols, dt, at, exact=True), dx_out.data_ptr()
    grads = {}
    for name, t in (("dgate", gate), ("dpost_w", post_w), ("dpre_w", pre_w), ("dscale", scale), ("dshift", shift)):
        g = None
        if t is not None:
            g = (torch.empty if rows else torch.zeros)(t.shape, dtype=torch.float32, device=dv)
            setattr(a, name, g.data_ptr())
        grads[name] = g
    ctx = ctx_for(x_out)
    need = C.c_size_t()
    dev.check(ctx.lib.anima_residual_norm_backward_workspace(ctx.h, C.byref(a), C.byref(need)))
    if need.value:
        ws = torch.empty(need.value, dtype=torch.uint8, device=dv)
        a.workspace, a.workspace_bytes = ws.data_ptr(), need.value
    ctx.call("anima_residual_norm_backward", C.byref(a), kernels=2 if need.value else 1)
    return ResidualNormGrads(dx, dy, **grads)


def elementwise(op: str, a: torch.Tensor, b: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """silu | copy | add | silu_mul over fp32 elements (ops.js:154-160)."""
    code = {"copy": 0, "add": 1, "silu": 2, "silu_mul": 3}[op]
    y = out if out is not None else torch.empty_like(a)
    n = min(y.numel(), a.numel())
    ctx_for(a).call("anima_elementwise", code, ptr(a), ptr(b), ptr(y), n)
    return y


def conv3x3(x: torch.Tensor, W, h: int, w: int, up: bool = False, into: torch.Tensor | None = None) -> torch.Tensor:
    """NHWC 3x3 convolution, pad 1, of x [h w, cin] with W (bf16 OHWI as [N, 9 cin], + bias); up:
    nearest 2x upsample first; into: out += conv (ops.js:97-109, conv3x3 / conv3x3Into)."""
    H, Wd = (2 * h, 2 * w) if up else (h, w)
    out = into if into is not None else torch.empty(H * Wd, W.N, dtype=torch.float32, device=x.device)
    wc = W.c()
    ctx_for(x).call("anima_conv3x3", ptr(x), h, w, W.K // 9, C.byref(wc), 1 if up else 0, ptr(out),
                    1 if into is not None else 0)
    return out


def channel_norm(x: torch.Tensor, gamma: torch.Tensor, cols: int, silu: bool) -> torch.Tensor:
    """The Wan VAE's RMS_norm over channels, then SiLU (ops.js:120-126)."""
    y = torch.empty_like(x)
    ctx_for(x).call("anima_channel_norm", ptr(x), x.numel() // cols, cols, ptr(gamma), 1 if silu else 0, ptr(y))
    return y


def zero(t: torch.Tensor):
    """ops.zero (ops.js:89-93)."""
    ctx_for(t).call("anima_zero", ptr(t), t.numel() * t.element_size())


# ----------------------------------------------------------------------------- linears

def linear(x, W, *, out: torch.Tensor | None = None, resid: bool = False, gate: torch.Tensor | None = None,
           g_off: int = 0, act: str | None = None, add: torch.Tensor | None = None, out_dtype=torch.float32,
           mode: str = "store", qk=None, rope_cs: torch.Tensor | None = None, n_q: int = 0, eps: float = 1e-6,
           planes: int = 2, name: str | None = None, peer=None) -> torch.Tensor:
    """y = x @ W^T (+ bias) (+ add) (act); or out += gate[g_off + n] * y when resid (ops.js:48-66).

    x: QuantRows (rotated, quantized) for ConvRot weights, or an fp32 tensor (rotated and quantized
    here, like ops.linear rotating when no xr is given). LoRA side paths attached to W are added
    before the activation, as the reference does (ops.js:55-57).
    mode: "store" | "qkv" (per-head RMSNorm + RoPE on q/k heads, qk = (qn, kn)) |
          "head_norm" (per-head RMSNorm with qk[0]).
    peer (mode "qkv"): {"kv": [device addresses of every rank's gathered k|v buffer], "row0", "rows",
          "item_rows"}: the k|v columns go to those buffers over NVLink instead of to `out`
          (sharding.KVExchange; anima_linear_opts.peer_*).
    """
    from . import lora as lora_mod

    if W.kind in ("bf16", "f32"):
        return matmul(x, W, act=act, out=out, resid=resid, gate=gate, g_off=g_off)
    if not isinstance(x, QuantRows):
        x = rotate_quant(x.reshape(-1, W.K).contiguous(), planes)
    M = x.rows
    o = dev.LinearOpts()
    keep = None
    if W.lora:
        if lora_mod.PATH == "fused":
            keep = lora_mod.lora_epilogue(x, W, o)   # T B^T inside the GEMM epilogue (None: entries it
        if keep is None:                             # cannot take, which get an added delta)
            delta = lora_mod.lora_delta_tc(x, W) if lora_mod.PATH == "delta" else lora_mod.lora_delta(x, W)
            add = delta if add is None else add + delta
    if out is None:
        if resid:
            raise dev.AnimaError(1, "resid=True needs out")
        out = torch.empty(M, W.N, dtype=out_dtype, device=x.hi.device)
    o.act = dev.ACT[act]
    o.add = add.data_ptr() if add is not None else 0
    o.ld_add = add.stride(0) if add is not None else 0
    o.out_mode = dev.OUT_RESID if resid else {"store": dev.OUT_STORE, "qkv": dev.OUT_QKV_NORM_ROPE,
                                              "head_norm": dev.OUT_HEAD_NORM}[mode]
    o.out_dtype = _dt(out)
    o.out = out.data_ptr()
    o.ldo = out.stride(0)
    o.gate = gate.data_ptr() if gate is not None else 0
    o.gate_off = g_off
    if qk is not None:
        o.norm_q = qk[0].data_ptr()
        o.norm_k = qk[1].data_ptr() if len(qk) > 1 and qk[1] is not None else 0
    if rope_cs is not None:
        o.rope = rope_cs.data_ptr()
        o.rope_rows = rope_cs.numel() // 128
    o.n_q = n_q
    o.eps = eps
    if peer is not None:
        o.peer_count = len(peer["kv"])
        for r, a in enumerate(peer["kv"]):
            o.peer_kv[r] = a
        o.peer_row0, o.peer_rows, o.peer_item_rows = peer["row0"], peer["rows"], peer["item_rows"]
    qa = x.c()
    w = W.c()
    ctx_for(x.hi).call("anima_linear", C.byref(qa), C.byref(w), C.byref(o), tag=name, work=2.0 * M * W.N * W.K,
                       kernels=2 if W.kind == "w4" else 1)  # w4: the decode, then the GEMM
    del keep
    return out


def matmul(x: torch.Tensor, W, *, act: str | None = None, out: torch.Tensor | None = None, resid: bool = False,
           gate: torch.Tensor | None = None, g_off: int = 0, alpha: float = 1.0) -> torch.Tensor:
    """runMatmul for bf16/f32 weights (ops.js:14-33): small SIMT GEMM, fp32 accumulate."""
    x2 = x.reshape(-1, x.shape[-1])
    M, K = x2.shape
    if out is None:
        if resid:
            raise dev.AnimaError(1, "resid=True needs out")
        out = torch.empty(M, W.N, dtype=torch.float32, device=x.device)
    w = W.c()
    ctx_for(x).call("anima_matmul", M, W.N, K, C.c_float(alpha), ptr(x2), x2.stride(0), C.byref(w), dev.ACT[act],
                    ptr(out), out.stride(0), 1 if resid else 0, ptr(gate), g_off)
    return out


# ----------------------------------------------------------------------------- attention

def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, Lq: int, Lk: int, H: int, D: int = 128,
              ldq: int | None = None, ldk: int | None = None, ldv: int | None = None, q_off: int = 0,
              k_off: int = 0, v_off: int = 0, batch: int = 1, q_bstride: int = 0, k_bstride: int = 0,
              v_bstride: int = 0, key_len: torch.Tensor | None = None, out: torch.Tensor | None = None,
              out_dtype=None, o_bstride: int | None = None, scale: float | None = None,
              name: str | None = None, noalloc: bool = False, group: int = 1, causal: bool = False) -> torch.Tensor:
    """Non-causal multi-head attention (ops.js:166-208): q [.., ldq] with head h at q_off + h D,
    k/v likewise; output [batch * Lq, H D]. q/k/v are bf16 or fp16; key_len (int32 [batch]) masks
    keys past each item's text length. noalloc: the entry point whose stream-K workspace is the
    library's static device array (no allocation; calls must not overlap). group: q heads per k/v
    head (GQA); causal: query i sees keys j <= i; with either, or D = 64, or fp32 q/k/v, the
    text-model kernel runs (ops.js:166-208 takes the same `group` and `causal`)."""
    ldq = ldq or H * D
    ldk = ldk or (H // max(group, 1)) * D
    ldv = ldv or (H // max(group, 1)) * D
    if out is None:
        out = torch.empty(batch * Lq, H * D, dtype=out_dtype or q.dtype, device=q.device)
    a = dev.AttentionArgs()
    a.batch, a.heads, a.head_dim, a.Lq, a.Lk = batch, H, D, Lq, Lk
    a.dtype = _dt(q)
    a.q, a.ldq, a.q_bstride, a.q_off = q.data_ptr(), ldq, q_bstride, q_off
    a.k, a.ldk, a.k_bstride, a.k_off = k.data_ptr(), ldk, k_bstride, k_off
    a.v, a.ldv, a.v_bstride, a.v_off = v.data_ptr(), ldv, v_bstride, v_off
    a.out, a.ldo = out.data_ptr(), out.stride(0)
    a.o_bstride = o_bstride if o_bstride is not None else Lq * out.stride(0)
    a.out_dtype = _dt(out)
    a.key_len = key_len.data_ptr() if key_len is not None else 0
    a.scale = scale if scale is not None else 1.0 / math.sqrt(D)
    a.group, a.causal = int(group), 1 if causal else 0
    ctx_for(q).call("anima_attention_noalloc" if noalloc else "anima_attention", C.byref(a), tag=name,
                    work=4.0 * batch * Lq * Lk * D * H)
    return out


def _reach(fn: str, name: str, t: torch.Tensor, off: int, items: int, bstride: int, rows: int, ld: int, cols: int):
    """Refuse strides that lead past the end of t's memory (or before its start)."""
    if off < 0 or ld < off + cols or (items > 1 and bstride < 0):
        raise dev.AnimaError(1, f"{fn}: {name}'s row stride {ld} is below its {off} + {cols} columns, or its batch "
                                f"stride {bstride} negative")
    need = off + (items - 1) * bstride + (rows - 1) * ld + cols
    if t.is_contiguous() and need <= t.numel():
        return
    have = t.untyped_storage().nbytes() // t.element_size() - t.storage_offset()
    if t.is_contiguous() or need > have:
        raise dev.AnimaError(1, f"{fn}: {name} has {t.numel()} elements ({have} behind its start), its sizes and strides "
                                f"reach {need}")


def _train_args(fn, q, k, v, Lq, Lk, H, D, ldq, ldk, ldv, q_off, k_off, v_off, batch, q_bstride, k_bstride, v_bstride,
                key_len, out, o_bstride, scale, group, causal):
    """The checked arguments that attention_lse and attention_backward share; returns them with the
    number of k/v items (1 where the batch shares one K/V) and the k/v columns."""
    if Lq <= 0 or Lk <= 0 or H <= 0 or batch <= 0 or group <= 0 or H % group:
        raise dev.AnimaError(1, f"{fn}: batch {batch}, {Lq} queries, {Lk} keys, {H} heads in groups of {group}")
    if max(Lq, Lk, H, batch, q_off, k_off, v_off) > _MOST:
        raise dev.AnimaError(1, f"{fn}: sizes and column offsets end at 2^30 (batch {batch}, {Lq} queries, {Lk} keys, {H} "
                                f"heads, columns {q_off}, {k_off}, {v_off})")
    if D not in (64, 128):
        raise dev.AnimaError(1, f"{fn}: head_dim {D} (64 or 128)")
    if q.dtype not in (torch.bfloat16, torch.float16):
        raise dev.AnimaError(1, f"{fn}: q, k and v are bf16 or fp16, not {q.dtype}")
    if scale is not None and not (2.0 ** -24 if q.dtype is torch.float16 else 2.0 ** -100) <= scale <= 2.0 ** 64:
        raise dev.AnimaError(1, f"{fn}: scale {scale} (2^-24 in fp16, 2^-100 in bf16, to 2^64)")
    C, Ck, dt, at = H * D, H // group * D, q.dtype, q.get_device()
    kv_items = 1 if batch > 1 and k_bstride == 0 and v_bstride == 0 else batch
    ldq, ldk, ldv = ldq or C, ldk or Ck, ldv or Ck
    for n, t, ld, off, items, bs, L, cols in (("q", q, ldq, q_off, batch, q_bstride, Lq, C),
                                              ("k", k, ldk, k_off, kv_items, k_bstride, Lk, Ck),
                                              ("v", v, ldv, v_off, kv_items, v_bstride, Lk, Ck)):
        if t.dtype is not dt or t.get_device() != at:
            raise dev.AnimaError(1, f"{fn}: {n} is {t.dtype} on {t.device}, q {q.dtype} on {q.device}")
        if items > 1 and bs <= 0:
            raise dev.AnimaError(1, f"{fn}: {n}_bstride {bs} with {batch} items (k and v may both have 0: shared)")
        _reach(fn, n, t, off, items, bs, L, ld, cols)
    a = dev.AttentionArgs(batch, H, D, Lq, Lk, dev.DTYPE_CODE[dt], q.data_ptr(), ldq, q_bstride, q_off, k.data_ptr(), ldk,
                          k_bstride, k_off, v.data_ptr(), ldv, v_bstride, v_off)
    a.scale, a.group, a.causal = scale or 0.0, group, bool(causal)
    if key_len is not None:
        _vector(fn, "key_len", key_len, key_len.numel(), torch.int32, at)
        if key_len.numel() < kv_items:
            raise dev.AnimaError(1, f"{fn}: {key_len.numel()} key lengths for {kv_items} k/v items")
        a.key_len = key_len.data_ptr()
    if out is not None:
        a.ldo, a.o_bstride = _grad_out(fn, "out", out, batch, Lq, C, o_bstride, at)
        a.out, a.out_dtype = out.data_ptr(), _dt(out)
    return a, kv_items, Ck


def _grad_out(fn, name, t, items, L, cols, bstride, device, dtype=None) -> tuple[int, int]:
    """Check a 2-D [items * L, >= cols] tensor (rows of item b from b * bstride on where that is given)
    and return its row and batch strides."""
    shape, st, dt = t.shape, t.stride(), t.dtype
    if len(shape) != 2 or st[1] != 1 or t.get_device() != device or dt not in _FLOATS or (dtype is not None and dt is not dtype):
        raise dev.AnimaError(1, f"{fn}: {name} has to be 2-D with contiguous rows" +
                                (f", {dtype}" if dtype is not None else "") + f", on device {device}; is {t.dtype} "
                                f"{tuple(t.shape)} on {t.device}")
    ld = st[0] if shape[0] > 1 else shape[1]
    if bstride is None:
        if shape[0] < items * L or shape[1] < cols or ld < cols:
            raise dev.AnimaError(1, f"{fn}: {name} is {tuple(t.shape)}, expected [{items * L}, {cols}]")
        return ld, L * ld
    _reach(fn, name, t, 0, items, bstride, L, ld, cols)
    return ld, bstride


def attention_lse(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, *, Lq: int, Lk: int, H: int, D: int = 128,
                  ldq: int | None = None, ldk: int | None = None, ldv: int | None = None, q_off: int = 0,
                  k_off: int = 0, v_off: int = 0, batch: int = 1, q_bstride: int = 0, k_bstride: int = 0,
                  v_bstride: int = 0, key_len: torch.Tensor | None = None, out: torch.Tensor | None = None,
                  out_dtype=None, o_bstride: int | None = None, scale: float | None = None, group: int = 1,
                  causal: bool = False, name: str | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """attention() for training: the same arguments (bf16 or fp16 q/k/v, D 64 or 128), and beside the
    output [batch * Lq, H D] the row statistics lse [batch, H, Lq] that attention_backward needs: ln of
    each query's sum of exponentials, -inf (with an output of zeros) where it sees no key. scale: 2^-24
    (bf16: 2^-100) to 2^64; in fp16 |q.k| below 2^30 before it. k and v may hold anything, NaN included, past key_len. Its workspace comes from torch's allocator, so calls on
    several streams and captured graphs share nothing."""
    fn = "attention_lse"
    if out is None:
        out = torch.empty(batch * Lq, H * D, dtype=out_dtype or q.dtype, device=q.device)
    a, _, _ = _train_args(fn, q, k, v, Lq, Lk, H, D, ldq, ldk, ldv, q_off, k_off, v_off, batch, q_bstride, k_bstride,
                          v_bstride, key_len, out, o_bstride, scale, group, causal)
    lse = torch.empty(batch, H, Lq, dtype=torch.float32, device=q.device)
    ctx = ctx_for(q)
    need = C.c_size_t()
    dev.check(ctx.lib.anima_attention_lse_workspace(ctx.h, C.byref(a), C.byref(need)))
    ws = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
    ctx.call("anima_attention_lse", C.byref(a), lse.data_ptr(), ws.data_ptr() if need.value else None, need, tag=name, work=4.0 * batch * Lq * Lk * D * H)
    return out, lse


def attention_backward(dout: torch.Tensor, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor,
                       lse: torch.Tensor, *, Lq: int, Lk: int, H: int, D: int = 128, ldq: int | None = None,
                       ldk: int | None = None, ldv: int | None = None, q_off: int = 0, k_off: int = 0, v_off: int = 0,
                       batch: int = 1, q_bstride: int = 0, k_bstride: int = 0, v_bstride: int = 0,
                       key_len: torch.Tensor | None = None, o_bstride: int | None = None, scale: float | None = None,
                       group: int = 1, causal: bool = False, do_bstride: int | None = None,
                       dq: torch.Tensor | None = None, dk: torch.Tensor | None = None, dv: torch.Tensor | None = None,
                       grad_dtype=None, name: str | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The gradients (dq, dk, dv) of attention_lse's q, k and v for the gradient dout [batch * Lq, H D] of
    its output; out and lse are what it returned, the rest its arguments. Probabilities are recomputed. dq
    is [batch * Lq, H D], dk and dv [items * Lk, (H / group) D]: a shared k/v head sums over its q heads,
    and where the batch shares one K/V (k_bstride = v_bstride = 0) there is one item, the sum over all.
    Given dq, dk, dv may be slices of one tensor; new ones have grad_dtype (q's type or fp32). Keys past
    key_len get zeros. The same inputs give the same bits."""
    fn = "attention_backward"
    if out.dim() != 2 or dout.dim() != 2:
        raise dev.AnimaError(1, f"{fn}: out and dout are 2-D [batch * Lq, H D]")
    a, kv_items, Ck = _train_args(fn, q, k, v, Lq, Lk, H, D, ldq, ldk, ldv, q_off, k_off, v_off, batch, q_bstride,
                                  k_bstride, v_bstride, key_len, out, o_bstride, scale, group, causal)
    at, device, Cq = q.get_device(), q.device, H * D
    if lse.dtype is not torch.float32 or lse.shape != (batch, H, Lq) or not lse.is_contiguous() or lse.get_device() != at:
        raise dev.AnimaError(1, f"{fn}: lse has to be a dense fp32 [{batch}, {H}, {Lq}] on {device}")
    gt = grad_dtype or q.dtype
    for t in (dv, dk, dq):
        if t is not None:
            gt = t.dtype
    if gt not in (torch.float32, q.dtype) or grad_dtype not in (None, gt):
        raise dev.AnimaError(1, f"{fn}: gradients are {gt}, have to be {q.dtype} or fp32 (grad_dtype {grad_dtype})")
    g = dev.AttentionGradArgs()
    g.fwd, g.lse, g.dout, g.grad_dtype = a, lse.data_ptr(), dout.data_ptr(), dev.DTYPE_CODE[gt]
    g.lddo, g.do_bstride = _grad_out(fn, "dout", dout, batch, Lq, Cq, do_bstride, at, q.dtype)
    if dq is None:
        dq, g.lddq, g.dq_bstride = torch.empty((batch * Lq, Cq), dtype=gt, device=device), Cq, Lq * Cq
    else:
        g.lddq, g.dq_bstride = _grad_out(fn, "dq", dq, batch, Lq, Cq, None, at, gt)
    if dk is None:
        dk, g.lddk, g.dk_bstride = torch.empty((kv_items * Lk, Ck), dtype=gt, device=device), Ck, Lk * Ck
    else:
        g.lddk, g.dk_bstride = _grad_out(fn, "dk", dk, kv_items, Lk, Ck, None, at, gt)
    if dv is None:
        dv, g.lddv, g.dv_bstride = torch.empty((kv_items * Lk, Ck), dtype=gt, device=device), Ck, Lk * Ck
    else:
        g.lddv, g.dv_bstride = _grad_out(fn, "dv", dv, kv_items, Lk, Ck, None, at, gt)
    g.dq, g.dk, g.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
    ctx = ctx_for(q)
    need = C.c_size_t()
    dev.check(ctx.lib.anima_attention_backward_workspace(ctx.h, C.byref(g), C.byref(need)))
    ws = torch.empty(need.value, dtype=torch.uint8, device=device)
    g.workspace, g.workspace_bytes = ws.data_ptr(), need.value
    ctx.call("anima_attention_backward", C.byref(g), tag=name, work=10.0 * batch * Lq * Lk * D * H,
             kernels=2 + (q.dtype is torch.float16) + (bool(causal) or Lk <= 128))  # (and the join of split units)
    return dq, dk, dv


# ----------------------------------------------------------------------------- model glue

def patchify(latent: torch.Tensor) -> torch.Tensor:
    """[B, 16, h, w] -> [B (h/2)(w/2), 68] with the zero mask channel (dit.js:55-65)."""
    B, _, h, w = latent.shape
    out = torch.empty(B * (h // 2) * (w // 2), 68, dtype=torch.float32, device=latent.device)
    ctx_for(latent).call("anima_patchify", ptr(latent), B, h, w, ptr(out))
    return out


def unpatchify(o: torch.Tensor, B: int, h: int, w: int) -> torch.Tensor:
    """[B (h/2)(w/2), 64] -> [B, 16, h, w] (dit.js:68-78)."""
    out = torch.empty(B, 16, h, w, dtype=torch.float32, device=o.device)
    ctx_for(o).call("anima_unpatchify", ptr(o), B, h, w, ptr(out))
    return out


def timestep_embedding(sigmas: torch.Tensor) -> torch.Tensor:
    """[S] sigmas -> [S, 2048] sinusoidal embeddings (dit.js:41-51)."""
    out = torch.empty(sigmas.numel(), 2048, dtype=torch.float32, device=sigmas.device)
    ctx_for(sigmas).call("anima_timestep_embedding", ptr(sigmas), sigmas.numel(), ptr(out))
    return out


def euler_step(x: torch.Tensor, v: torch.Tensor, sigma: float, sigma_next: float, v_uncond=None, cfg: float = 1.0,
               den_out: torch.Tensor | None = None):
    """In place: CFG combine, x0 = x - sigma v, Euler step (pipeline.js:260-269, samplers.js:109-117)."""
    ctx_for(x).call("anima_euler_step", ptr(x), ptr(v), ptr(v_uncond), C.c_float(cfg), C.c_float(sigma),
                    C.c_float(sigma_next), x.numel(), ptr(den_out))
    return x


def lincomb(out: torch.Tensor, *terms) -> torch.Tensor:
    """out = sum of c * t over up to four (c, t) pairs of fp32 tensors with out's element count; out
    may be one of the t (the samplers' axpby, samplers.js:97-101)."""
    if not 1 <= len(terms) <= 4:
        raise ValueError("lincomb takes one to four (coefficient, tensor) terms")
    xs = [C.c_void_p(0)] * 4
    cs = (C.c_float * 4)(0.0, 0.0, 0.0, 0.0)
    for k, (c, t) in enumerate(terms):
        if t.dtype != torch.float32 or t.numel() != out.numel() or not t.is_contiguous():
            raise dev.AnimaError(1, "lincomb: terms must be contiguous fp32 tensors of out's size")
        xs[k] = ptr(t)
        cs[k] = float(c)
    ctx_for(out).call("anima_lincomb", ptr(out), out.numel(), *xs, cs)
    return out


def unpack_w4(packed: torch.Tensor, s_rel: torch.Tensor, codebook: torch.Tensor, N: int, K: int) -> torch.Tensor:
    """4-bit codes -> int8-grid values [N, K], bit-exact with tools/quant.py:179-180."""
    out = torch.empty(N, K, dtype=torch.int8, device=packed.device)
    ctx_for(packed).call("anima_unpack_w4", ptr(packed), ptr(s_rel), ptr(codebook), N, K, ptr(out))
    return out
