"""CPU tests of the trained block's operators: frequencies, refusals, the C structs' layout."""

import ctypes
import math
import os
import shutil
import subprocess
import threading

import pytest
import torch

from tests.conftest import ROOT, pkg


@pytest.fixture(scope="module")
def ops():
    return pkg("ops")


@pytest.fixture(scope="module")
def err():
    return pkg("device").AnimaError


def test_structs_match_the_c_header(tmp_path):
    dev = pkg("device")
    structs = {"anima_rotary_args": dev.RotaryArgs, "anima_residual_norm_args": dev.ResidualNormArgs,
               "anima_attention_grad_args": dev.AttentionGradArgs}
    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "anima_b200.h"', "int main(void) {"]
    for cname, cls in structs.items():
        lines.append(f'  printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'  printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, *_ in cls._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["  return 0;", "}"]) + "\n")
    subprocess.run([cc, "-std=c11", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split("\n")
    got = {(a, b): int(c) for a, b, c in (ln.split() for ln in out if ln)}
    for cname, cls in structs.items():
        assert got[(cname, "sizeof")] == ctypes.sizeof(cls), cname
        for f, *_ in cls._fields_:
            assert got[(cname, f)] == getattr(cls, f).offset, (cname, f)


# ----------------------------------------------------------------------------- frequencies

def test_rotary_freqs(ops):
    plain, m = ops.rotary_freqs(128, 1e6, device="cpu")
    assert m == 1.0 and plain.dtype == torch.float64
    for i in (0, 1, 63):
        assert math.isclose(plain[i].item(), 1e6 ** (-2 * i / 128), rel_tol=1e-14)
    lin, _ = ops.rotary_freqs(128, 1e6, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(lin, plain / 4)
    ntk, _ = ops.rotary_freqs(128, 1e6, scaling="ntk", factor=4.0, device="cpu")
    assert ntk[0] == 1.0 and math.isclose((plain[63] / ntk[63]).item(), 4.0, rel_tol=1e-12)
    yarn, m = ops.rotary_freqs(128, 1e4, scaling="yarn", factor=8.0, original_len=4096, device="cpu")
    plain, _ = ops.rotary_freqs(128, 1e4, device="cpu")
    assert math.isclose(m, 0.1 * math.log(8.0) + 1.0)
    turns = 4096 * plain / (2 * math.pi)
    assert torch.equal(yarn[turns >= 32], plain[turns >= 32])
    torch.testing.assert_close(yarn[turns <= 1], plain[turns <= 1] / 8, rtol=1e-14, atol=0)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and bool(((yarn < plain) & (yarn > plain / 8))[mid].all())


@pytest.mark.parametrize("kw", [dict(dim=0), dict(dim=7), dict(dim=8, theta=0.0), dict(dim=8, factor=-1.0),
                                dict(dim=8, scaling="cubic"), dict(dim=8, scaling="yarn", beta_fast=1.0),
                                dict(dim=8, scaling="yarn", original_len=0)])
def test_rotary_freqs_refuses(ops, err, kw):
    with pytest.raises(err):
        ops.rotary_freqs(device="cpu", **kw)


# ----------------------------------------------------------------------------- refusals

def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


@pytest.mark.parametrize("change", [
    dict(q=t(5, 63)), dict(q=t(320)), dict(q=t(64, 5).T), dict(q=t(5, 64, dtype=torch.float64)),
    dict(k=t(4, 32)), dict(k=t(5, 31)), dict(k=t(5, 32, dtype=torch.bfloat16)), dict(k=None),
    dict(positions=t(5, dtype=torch.int64)), dict(positions=t(4, dtype=torch.int32)),
    dict(positions=torch.zeros(10, dtype=torch.int32)[::2]), dict(inv_freq=t(8)),
    dict(inv_freq=t(2, 4, dtype=torch.float64)), dict(out_q=t(5, 64, dtype=torch.float16)), dict(out_q=t(6, 64)),
    dict(out_k=t(5, 16)),
])
def test_rotary_refuses(ops, err, change):
    kw = dict(q=t(5, 64), k=t(5, 32), inv_freq=t(8, dtype=torch.float64), Hq=4, Hk=2, D=16)
    with pytest.raises(err) as e:
        ops.rotary(**{**kw, **change})
    assert e.value.status == 1


def test_no_cpu_path(ops, err):
    with pytest.raises(err) as e:
        ops.rotary(t(5, 64), t(5, 32), t(8, dtype=torch.float64), Hq=4, Hk=2, D=16)
    assert e.value.status == -1
    with pytest.raises(err) as e:
        ops.residual_norm(t(6, 16), t(6, 16))
    assert e.value.status == -1


NORM_BAD = [
    dict(y=t(5, 16)), dict(y=t(6, 15)), dict(y=t(16, 6).T), dict(y=t(6, 16, dtype=torch.float64)), dict(post="max"),
    dict(pre=None), dict(gate=t(16)), dict(gate=t(3, 16)), dict(scale=t(2, 15)), dict(shift=t(2, 16, dtype=torch.float16)),
    dict(pre_w=t(15)), dict(post_w=t(2, 8), post="rms"),
]


@pytest.mark.parametrize("change", NORM_BAD + [dict(x=t(6, 16, 1)), dict(x_out=t(6, 16, dtype=torch.float16)),
                                               dict(h=t(5, 16)), dict(h=t(6, 16), out_dtype=torch.float16)])
def test_residual_norm_refuses(ops, err, change):
    kw = dict(x=t(6, 16), y=t(6, 16), rows_per_item=3, gate=t(2, 16))
    with pytest.raises(err) as e:
        ops.residual_norm(**{**kw, **change})
    assert e.value.status == 1


@pytest.mark.parametrize("change", NORM_BAD + [dict(dh=t(6, 15)), dict(dx_out=t(6, 16, dtype=torch.float16)),
                                               dict(dx=t(5, 16)), dict(dy=t(6, 16, dtype=torch.bfloat16))])
def test_residual_norm_backward_refuses(ops, err, change):
    kw = dict(dh=t(6, 16), dx_out=t(6, 16), x_out=t(6, 16), y=t(6, 16), rows_per_item=3, gate=t(2, 16))
    with pytest.raises(err) as e:
        ops.residual_norm_backward(**{**kw, **change})
    assert e.value.status == 1


ATTN_BAD = [
    dict(Lq=0), dict(Lk=0), dict(H=3, group=2), dict(H=0), dict(batch=0), dict(D=96), dict(q=t(20, 128)),
    dict(k=t(24, 64, dtype=torch.float16)), dict(q=t(19, 128, dtype=torch.bfloat16)), dict(k=t(23, 64, dtype=torch.bfloat16)),
    dict(ldq=64), dict(ldk=32), dict(q_off=-8), dict(q_off=8), dict(v_off=64), dict(k_bstride=0), dict(v_bstride=-64),
    dict(q_bstride=11 * 128), dict(key_len=t(2)), dict(key_len=t(1, dtype=torch.int32)), dict(scale=-1.0), dict(scale=0.0),
    dict(scale=float("nan")),
]


def attn_kw():
    b = dict(dtype=torch.bfloat16)
    return dict(q=t(20, 128, **b), k=t(24, 64, **b), v=t(24, 64, **b), Lq=10, Lk=12, H=2, D=64, group=2, batch=2,
                q_bstride=1280, k_bstride=768, v_bstride=768)


@pytest.mark.parametrize("change", ATTN_BAD + [dict(out=t(19, 128)), dict(out=t(20, 127)), dict(out=t(20, 256).T)])
def test_attention_lse_refuses(ops, err, change):
    with pytest.raises(err) as e:
        ops.attention_lse(**{**attn_kw(), **change})
    assert e.value.status == 1


@pytest.mark.parametrize("change", ATTN_BAD + [
    dict(out=t(19, 128)), dict(dout=t(20, 128)), dict(dout=t(19, 128, dtype=torch.bfloat16)), dict(lse=t(2, 2, 9)),
    dict(lse=t(2, 2, 10, dtype=torch.float64)), dict(lse=t(2, 10, 2).transpose(1, 2)), dict(dq=t(20, 127)),
    dict(dk=t(24, 64), dv=t(24, 64, dtype=torch.bfloat16)), dict(dk=t(23, 64)), dict(dq=t(20, 128, dtype=torch.float16)),
    dict(grad_dtype=torch.float16), dict(dq=t(20, 128), grad_dtype=torch.bfloat16), dict(dout=t(2, 10, 128, dtype=torch.bfloat16)),
])
def test_attention_backward_refuses(ops, err, change):
    b = dict(dtype=torch.bfloat16)
    kw = dict(dout=t(20, 128, **b), out=t(20, 128, **b), lse=t(2, 2, 10), **attn_kw())
    with pytest.raises(err) as e:
        ops.attention_backward(**{**kw, **change})
    assert e.value.status == 1


# ----------------------------------------------------------------------------- the context's stream

class StreamLib:
    """A stand-in for the library: which stream each call would have run on."""

    def __init__(self):
        self.bound, self.ran, self.at_bind = None, [], None

    def anima_ctx_set_stream(self, h, stream):
        self.bound = getattr(stream, "value", stream)
        if self.at_bind:
            self.at_bind(self.bound)
        return 0

    def anima_zero(self, h, name):
        self.ran.append((name, self.bound))
        return 0


@pytest.fixture
def shared_context(monkeypatch):
    dev = pkg("device")
    ctx = dev.Context.__new__(dev.Context)
    ctx.lib, ctx.device, ctx.h, ctx.lock = StreamLib(), 0, None, threading.RLock()
    here = threading.local()
    monkeypatch.setattr(dev, "_raw_stream", lambda device: here.stream)
    return ctx, here


def test_threads_that_share_a_context_keep_their_streams(shared_context):
    """Another thread's call in the middle of one (between the binding of its stream and what follows)
    moves neither that call nor the thread's later ones to the other's stream."""
    ctx, here = shared_context
    done = threading.Event()

    def other():
        here.stream = 22
        ctx.call("anima_zero", "b")
        done.set()

    def in_the_middle(stream):
        if stream == 11:
            ctx.lib.at_bind = None
            threading.Thread(target=other, daemon=True).start()
            done.wait(0.5)  # as far as it gets

    ctx.lib.at_bind = in_the_middle
    here.stream = 11
    ctx.call("anima_zero", "a")
    assert done.wait(10)
    for i in range(3):
        ctx.call("anima_zero", "a")
    assert sorted(set(ctx.lib.ran)) == [("a", 11), ("b", 22)]


def test_a_stream_set_behind_the_context_does_not_stay(shared_context):
    """A host that calls anima_ctx_set_stream itself: the next operator is on torch's current stream again."""
    ctx, here = shared_context
    here.stream = 11
    ctx.call("anima_zero", "a")
    ctx.lib.anima_ctx_set_stream(ctx.h, 99)
    ctx.call("anima_zero", "a")
    assert ctx.lib.ran == [("a", 11), ("a", 11)]


# ----------------------------------------------------------------------------- ranges

@pytest.mark.parametrize("dtype,scale", [(torch.float16, 2.0 ** -25), (torch.float16, 1e-9), (torch.bfloat16, 2.0 ** -101),
                                         (torch.bfloat16, 1e-46), (torch.float16, 2.0 ** 65), (torch.bfloat16, 1e39),
                                         (torch.bfloat16, math.inf)])
def test_attention_refuses_scales_out_of_range(ops, err, dtype, scale):
    """1e-46 is 0 in the kernels' fp32, which stands for the default, and 1e39 is infinite."""
    kw = {n: (v.to(dtype) if isinstance(v, torch.Tensor) else v) for n, v in attn_kw().items()}
    with pytest.raises(err, match="scale"):
        ops.attention_lse(**kw, scale=scale)
    with pytest.raises(err, match="scale"):
        ops.attention_backward(t(20, 128, dtype=dtype), out=t(20, 128, dtype=dtype), lse=t(2, 2, 10), **kw, scale=scale)


FAR = 2 ** 32  # a C int would keep the rest: 5 rows of 2^32 + 5


def far(rows, cols, dtype=torch.float32):
    return torch.empty(rows, cols, dtype=dtype, device="meta")


@pytest.mark.parametrize("rows,cols", [(FAR + 5, 64), (2 ** 30 + 1, 64), (5, FAR + 64)])
def test_sizes_that_a_c_int_cuts_off_are_refused(ops, err, rows, cols):
    inv = torch.empty(8, dtype=torch.float64, device="meta")
    x = far(rows, cols)
    for call in (lambda: ops.rotary(x, None, inv, Hq=1, D=cols), lambda: ops.residual_norm(x, x),
                 lambda: ops.residual_norm_backward(x, x, x, x)):
        with pytest.raises(err) as e:
            call()
        assert e.value.status == 1
    with pytest.raises(err) as e:
        ops.rotary(far(4, 64), None, torch.empty(FAR // 2 + 8, dtype=torch.float64, device="meta"), Hq=1, D=64)
    assert e.value.status == 1


@pytest.mark.parametrize("change", [dict(Lq=FAR + 10), dict(Lk=FAR + 12), dict(batch=FAR + 2), dict(H=FAR + 2),
                                    dict(q_off=FAR), dict(k_off=FAR), dict(v_off=FAR + 8), dict(H=FAR + 2, group=FAR + 2)])
def test_attention_sizes_that_a_c_int_cuts_off_are_refused(ops, err, change):
    kw = {n: (far(2 ** 34, 128, torch.bfloat16) if isinstance(v, torch.Tensor) else v) for n, v in attn_kw().items()}
    kw |= dict(q_bstride=8, k_bstride=8, v_bstride=8, ldq=2 ** 33, ldk=2 ** 33, ldv=2 ** 33)
    with pytest.raises(err) as e:
        ops.attention_lse(**{**kw, **change}, out=far(2 ** 37, 128, torch.bfloat16))
    assert e.value.status == 1 and "2^30" in str(e.value)


def test_rows_per_item_past_a_c_int(ops, monkeypatch):
    """More rows an item than there are: one item, as the longest count that is kept whole says."""
    dev, seen = pkg("device"), []

    class Fake:
        def call(self, name, args, **kw):
            seen.append(args._obj.rows_per_item)

    monkeypatch.setattr(ops, "ctx_for", lambda t: Fake())
    inv = t(8, dtype=torch.float64)
    for n in (None, 3, 6, FAR + 2, 2 ** 31):
        ops.rotary(t(6, 16), None, inv, Hq=1, D=16, rows_per_item=n)
    assert seen == [6, 3, 6, 6, 6]
    for n in (4, FAR + 2, -3):
        with pytest.raises(dev.AnimaError) as e:
            ops.residual_norm(t(6, 16), t(6, 16), rows_per_item=n)
        assert e.value.status == 1
