"""Refusals of the serving operators, checked without a GPU: every bad call ends on the host before a launch."""
import ctypes

import pytest
import torch

import comfy_kitchen as ck
from comfy_kitchen import _native
from comfy_kitchen.backends import cuda as backend

BF16 = torch.bfloat16


def _lora(**change):
    args = dict(y=torch.zeros(4, 16, dtype=BF16), x=torch.zeros(4, 24, dtype=BF16), a=torch.zeros(2, 8, 24, dtype=BF16),
                b=torch.zeros(2, 16, 8, dtype=BF16), adapter_ids=torch.zeros(4, dtype=torch.int32), scales=torch.ones(2), out=None)
    args.update(change)
    return args


@pytest.mark.parametrize("change,what", [
    (dict(b=torch.zeros(3, 16, 8, dtype=BF16)), "do not match"),
    (dict(b=torch.zeros(2, 16, 16, dtype=BF16)), "do not match"),
    (dict(x=torch.zeros(4, 32, dtype=BF16)), "columns"),
    (dict(y=torch.zeros(5, 16, dtype=BF16)), "y must be"),
    (dict(y=torch.zeros(4, 16)), "one dtype"),
    (dict(a=torch.zeros(2, 4, 24, dtype=BF16), b=torch.zeros(2, 16, 4, dtype=BF16)), "multiples of 8"),
    (dict(a=torch.zeros(2, 264, 24, dtype=BF16), b=torch.zeros(2, 16, 264, dtype=BF16)), "at most 256"),
    (dict(a=torch.zeros(0, 8, 24, dtype=BF16), b=torch.zeros(0, 16, 8, dtype=BF16), scales=None), "of 0 adapters"),
    (dict(adapter_ids=torch.zeros(4)), "int32 or int64"),
    (dict(adapter_ids=torch.zeros(2, dtype=torch.int32)), "adapter_ids"),
    (dict(adapter_ids=torch.zeros(4, 1, dtype=torch.int32)), "adapter_ids"),
    (dict(scales=torch.ones(3)), "scales"),
    (dict(scales=torch.ones(2, dtype=torch.float64)), "scales"),
    (dict(out=torch.zeros(4, 8, dtype=BF16)), "out must"),
    (dict(out=torch.zeros(16, 4, dtype=BF16).t()), "out must"),
    (dict(out=torch.zeros(4 * 16 + 1, dtype=BF16)[1:].view(4, 16)), "out must"),
])
def test_lora_refusals(change, what):
    with pytest.raises(ValueError, match=what):
        backend.lora_add(**_lora(**change))


@pytest.mark.parametrize("change,what", [
    (dict(residual=torch.zeros(3, 64, dtype=BF16)), "same shape"),
    (dict(residual=torch.zeros(2, 64, dtype=torch.float16)), "residual has"),
    (dict(x=torch.zeros(2, 48, dtype=BF16), residual=torch.zeros(2, 48, dtype=BF16)), "divisible by 32"),
    (dict(x=torch.zeros(2, 0, dtype=BF16), residual=torch.zeros(2, 0, dtype=BF16)), "positive"),
    (dict(weight=torch.zeros(32, dtype=BF16)), "weight"),
    (dict(sum_out=torch.zeros(2, 64)), "sum_out"),
    (dict(sum_out=torch.zeros(64, 2, dtype=BF16).t()), "sum_out"),
])
def test_norm_refusals(change, what):
    args = dict(x=torch.zeros(2, 64, dtype=BF16), residual=torch.zeros(2, 64, dtype=BF16), weight=None)
    args.update(change)
    with pytest.raises(ValueError, match=what):
        backend.add_rmsnorm_quantize_mxfp8(**args)


def test_norm_fp8_refusals():
    x = torch.zeros(2, 64, dtype=BF16)
    with pytest.raises(ValueError, match="output_type"):
        backend.add_rmsnorm_quantize_fp8(x, x, None, torch.ones(1), output_type=torch.float16)
    with pytest.raises(ValueError, match="scalar"):
        backend.add_rmsnorm_quantize_fp8(x, x, None, torch.ones(2))


@pytest.mark.parametrize("change,what", [
    (dict(tokens_dim=3), "tokens_dim"),
    (dict(xq=torch.zeros(1, 2, 8)), "four dimensions"),
    (dict(xk=torch.zeros(1, 2, 6, 8)), "agree"),
    (dict(xk=torch.zeros(1, 2, 5, 8, dtype=BF16)), "agree"),
    (dict(axes_dim=(3, 5)), "axes_dim"),
    (dict(axes_dim=(8, 2)), "axes_dim"),
    (dict(axes_dim=()), "axes_dim"),
    (dict(axes_dim=(8, 0)), "axes_dim"),
    (dict(freqs=torch.zeros(3, dtype=torch.float64)), "freqs"),
    (dict(freqs=torch.zeros(4)), "freqs"),
    (dict(positions=torch.zeros(4, 2)), "positions"),
    (dict(positions=torch.zeros(2, 5, 2)), "positions"),
    (dict(positions=torch.zeros(5, 3)), "positions"),
    (dict(positions=torch.zeros(5, 2, dtype=torch.int16)), "positions"),
])
def test_rope_refusals(change, what):
    args = dict(xq=torch.zeros(1, 2, 5, 8), xk=torch.zeros(1, 1, 5, 8), positions=torch.zeros(5, 2), freqs=torch.zeros(4, dtype=torch.float64), axes_dim=(4, 4))
    args.update(change)
    with pytest.raises(ValueError, match=what):
        backend.apply_rope_axes(**args)


def test_no_gradient_is_dropped_in_silence():
    leaf = lambda *s: torch.zeros(*s, dtype=BF16, requires_grad=True)  # noqa: E731
    with pytest.raises(RuntimeError, match="no backward"):
        backend.lora_add(**_lora(a=leaf(2, 8, 24)))
    with pytest.raises(RuntimeError, match="no backward"):
        backend.add_rmsnorm_quantize_mxfp8(leaf(2, 64), torch.zeros(2, 64, dtype=BF16))
    with pytest.raises(RuntimeError, match="no backward"):
        backend.apply_rope_axes1(leaf(1, 1, 2, 8), torch.zeros(2, 1), torch.zeros(4, dtype=torch.float64), (8,))
    with pytest.raises(RuntimeError, match="no backward"):     # (nor is a leaf written to)
        backend.lora_add(**_lora(out=leaf(3, 16)))
    with pytest.raises(RuntimeError, match="no backward"):
        backend.add_rmsnorm_quantize_mxfp8(torch.zeros(2, 64, dtype=BF16), torch.zeros(2, 64, dtype=BF16), sum_out=leaf(2, 64))


def test_cpu_tensors_find_no_backend():
    x = torch.zeros(2, 64, dtype=BF16)
    with pytest.raises(ck.NoCapableBackendError):
        ck.add_rmsnorm_quantize_mxfp8(x, x)
    with pytest.raises(ck.NoCapableBackendError):
        ck.add_rmsnorm_quantize_fp8(x, x, None, torch.ones(1), sum_out=x)
    with pytest.raises(ck.NoCapableBackendError):
        ck.lora_add(*list(_lora().values())[:6])
    with pytest.raises(ck.NoCapableBackendError):
        ck.apply_rope_axes1(torch.zeros(1, 1, 2, 8), torch.zeros(2, 1), torch.zeros(4, dtype=torch.float64), (8,))


def test_adapters_of_a_layer():
    from comfy_kitchen.linear import MXFP8Linear, NVFP4Linear

    for layer in (NVFP4Linear(24, 16, bias=False), MXFP8Linear(24, 16)):
        a, b = torch.zeros(2, 8, 24, dtype=BF16), torch.zeros(2, 16, 8, dtype=BF16)
        layer.set_adapters(a, b, torch.ones(2))
        assert layer.adapter_a.shape == a.shape and not any("adapter" in k for k in torch.nn.Module.state_dict(layer))
        for bad in ((a, None), (a, b[:1]), (a, b.transpose(1, 2)), (a, b.float()), (a, b, torch.ones(3)), (a, b, torch.ones(2).double())):
            with pytest.raises(ValueError):
                layer.set_adapters(*bad)
        layer.set_adapters(None)
        with pytest.raises(ValueError, match="set_adapters"):
            layer._add_adapters(torch.zeros(1, 16, dtype=BF16), torch.zeros(1, 24, dtype=BF16), torch.zeros(1, dtype=torch.int32))
        y = torch.zeros(1, 16)
        assert layer._add_adapters(y, None, None) is y


def test_frequency_table():
    f = ck.rope_axes_freqs((4, 8), 100.0, device="cpu")
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 100.0 ** -0.5, 1.0, 100.0 ** -0.25, 100.0 ** -0.5, 100.0 ** -0.75], dtype=torch.float64))


# ---- the C entry points: bad arguments are answered with a status, nothing is launched (pointers are never read)

P = 0x10000   # an aligned address that is not looked at


def _refused(name, *args):
    with pytest.raises(RuntimeError, match=r"status -[1-5]"):
        _native.call(name, *args)


def test_native_norm_refusals():
    def call(x=P, res=P, w=0, scale=0, s=P, y=0, q=P, sf=P, n=2, d=64, xs=64, rs=64, eps=1e-6, t=2, rt=2, ot=5):
        _refused("launch_add_rmsnorm_quantize_kernel", x, res, w, scale, s, y, q, sf, n, d, xs, rs, eps, t, rt, ot, None)

    for bad in (dict(x=0), dict(res=0), dict(s=0), dict(q=0), dict(sf=0), dict(n=0), dict(n=-1), dict(d=0), dict(d=48), dict(xs=63), dict(rs=0), dict(t=5),
                dict(rt=1), dict(ot=6), dict(ot=2), dict(sf=P + 2), dict(res=P, s=P, rs=128), dict(n=1 << 40)):
        call(**bad)


def test_native_rope_refusals():
    strides = (ctypes.c_int64 * 11)(*([8] * 11))

    def call(q=P, k=0, pos=P, f=P, oq=P, ok=0, st=strides, b=1, n=2, hq=1, hk=0, d=8, axes=(4,), count=None, t=2, pt=0):
        pairs = (ctypes.c_int32 * max(1, len(axes)))(*axes)
        _refused("launch_apply_rope_axes_kernel", q, k, pos, f, oq, ok, st, b, n, hq, hk, d, pairs, len(axes) if count is None else count, t, pt, False, False, False, None)

    for bad in (dict(q=0), dict(pos=0), dict(f=0), dict(oq=0), dict(k=P), dict(k=P, ok=P), dict(hk=1), dict(b=0), dict(n=0), dict(hq=0), dict(hq=70000), dict(d=7),
                dict(axes=(5,)), dict(axes=(0,)), dict(axes=(2, 3)), dict(count=0), dict(axes=(1,) * 9, d=32), dict(t=5), dict(pt=4), dict(pt=-1), dict(b=1 << 20), dict(n=1 << 60, d=64), dict(b=512, n=1 << 40, d=65536)):
        call(**bad)


def test_native_lora_refusals():
    def call(y=P, x=P, a=P, b=P, ids=P, out=P, ws=P, rows=4000, k=24, n=16, r=8, count=2, ys=16, xs=24, os=16, per=1, t=2):
        _refused("launch_lora_add_kernel", y, x, a, b, ids, 0, out, ws, rows, k, n, r, count, ys, xs, os, per, t, False, None)

    for bad in (dict(y=0), dict(x=0), dict(a=0), dict(b=0), dict(ids=0), dict(out=0), dict(rows=0), dict(rows=1 << 40), dict(k=0), dict(k=20), dict(n=12), dict(r=0), dict(r=4),
                dict(r=264), dict(count=0), dict(ys=8), dict(xs=16), dict(os=8), dict(per=0), dict(t=0), dict(y=P + 2), dict(x=P + 8), dict(a=P + 4), dict(xs=25), dict(out=P + 6), dict(ws=0), dict(ws=P + 8)):
        call(**bad)
