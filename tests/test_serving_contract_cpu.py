"""What the serving operators promise beyond their refusals of shapes and types, checked without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

import comfy_kitchen as ck
from comfy_kitchen import _native
from comfy_kitchen.backends import cuda as backend

BF16 = torch.bfloat16


def _zeros(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype)


def _calls():
    """(entry point, its arguments by name), one small valid call of each."""
    lora = dict(y=_zeros(4, 16), x=_zeros(4, 24), a=_zeros(2, 8, 24), b=_zeros(2, 16, 8), adapter_ids=torch.zeros(4, dtype=torch.int32), scales=torch.ones(2))
    norm = dict(x=_zeros(2, 64), residual=_zeros(2, 64), weight=_zeros(64))
    rope = dict(positions=torch.zeros(3, 1), freqs=torch.zeros(4, dtype=torch.float64), axes_dim=(8,))
    return {
        "lora_add": (backend.lora_add, lora),
        "mxfp8": (backend.add_rmsnorm_quantize_mxfp8, norm),
        "fp8": (backend.add_rmsnorm_quantize_fp8, dict(norm, scale=torch.ones(1))),
        "rope": (backend.apply_rope_axes, dict(rope, xq=_zeros(1, 2, 3, 8), xk=_zeros(1, 1, 3, 8))),
        "rope1": (backend.apply_rope_axes1, dict(rope, x=_zeros(1, 2, 3, 8))),
    }


TRACKED = [("lora_add", n) for n in ("y", "x", "a", "b", "scales")] + [(k, n) for k in ("mxfp8", "fp8") for n in ("x", "residual", "weight")] + [
    ("fp8", "scale"), ("rope", "xq"), ("rope", "xk"), ("rope", "freqs"), ("rope", "positions"), ("rope1", "x"), ("rope1", "freqs")]


@pytest.mark.parametrize("kind", ["leaf", "parameter", "result", "tangent"])
@pytest.mark.parametrize("name,argument", TRACKED)
def test_no_derivative_is_dropped_in_silence(name, argument, kind):
    """Trainable adapters and norm weights are parameters: they are refused as any other tensor that wants a gradient is."""
    entry, args = _calls()[name]
    t = args[argument]
    if kind == "tangent":
        with forward_ad.dual_level(), torch.no_grad():      # (forward mode goes on under no_grad)
            args[argument] = forward_ad.make_dual(t, torch.ones_like(t))
            with pytest.raises(RuntimeError, match="forward-mode"):
                entry(**args)
        return
    args[argument] = {"leaf": lambda: t.requires_grad_(), "parameter": lambda: torch.nn.Parameter(t), "result": lambda: t.requires_grad_() * 1}[kind]()
    with pytest.raises(RuntimeError, match="no backward"):
        entry(**args)


def test_dual_level_takes_what_has_no_tangent():
    """Inside a dual level a call without tangents gets as far as it does outside: to the device."""
    entry, args = _calls()["rope1"]
    args["positions"] = torch.zeros(3, 1, dtype=torch.int64)
    with forward_ad.dual_level():
        with pytest.raises(Exception) as e:
            entry(**args)
    assert "forward-mode" not in str(e.value) and "backward" not in str(e.value)


# ---- a layer with adapters


def _plain_lora(y, x, a, b, adapter_ids, scales=None):
    """lora_add on the CPU, with its question about gradients."""
    backend._no_grad("lora_add", y, x, a, b, scales)
    f = torch.ones(a.shape[0]) if scales is None else scales
    more = [f[i] * (x[t].double() @ a[i].double().T) @ b[i].double().T for t, i in enumerate(adapter_ids.tolist())]
    return (y.double() + torch.stack(more)).to(y.dtype)


@pytest.fixture
def layer(monkeypatch):
    """An NVFP4Linear as it is built by default, with a plain weight in the quantized one's place and its adapters."""
    from comfy_kitchen.linear import NVFP4Linear, QuantizedTensor

    monkeypatch.setattr(QuantizedTensor, "from_float", staticmethod(lambda x, *args, **kwargs: x))
    monkeypatch.setattr(ck, "lora_add", _plain_lora)
    g = torch.Generator().manual_seed(1)
    layer = NVFP4Linear(24, 16)
    layer.weight = torch.nn.Parameter(torch.randn(16, 24, generator=g).to(BF16), requires_grad=False)
    layer.bias.data.normal_(generator=g)
    layer.set_adapters(torch.randn(2, 8, 24, generator=g).to(BF16), torch.randn(2, 16, 8, generator=g).to(BF16))
    return layer


def test_layer_with_its_default_bias_takes_adapters(layer):
    """The bias wants a gradient, so the projection does: it passes through the adapters' sum as it is."""
    g = torch.Generator().manual_seed(2)
    x, ids, grad = torch.randn(3, 24, generator=g).to(BF16), torch.tensor([1, 0, 1]), torch.randn(3, 16, generator=g).to(BF16)
    base = layer(x)
    assert base.requires_grad
    got = layer(x, ids)
    assert torch.equal(got, _plain_lora(base.detach(), x, layer.adapter_a, layer.adapter_b, ids))
    want, = torch.autograd.grad(base, layer.bias, grad)
    have, = torch.autograd.grad(got, layer.bias, grad)
    assert torch.equal(have, want)
    with torch.no_grad():
        assert torch.equal(layer(x, ids), got) and not layer(x, ids).requires_grad


def test_layer_does_not_drop_the_input_gradient(layer):
    with pytest.raises(RuntimeError, match="no backward"):
        layer(torch.zeros(1, 24, dtype=BF16, requires_grad=True), torch.tensor([1]))


def test_adapters_given_as_parameters_stay_out_of_the_state(layer):
    """Scales as well as a and b: buffers that no state dict or optimizer sees."""
    layer.set_adapters(torch.nn.Parameter(_zeros(2, 8, 24)), torch.nn.Parameter(_zeros(2, 16, 8)), torch.nn.Parameter(torch.ones(2)))
    assert sorted(n for n, _ in layer.named_parameters()) == ["bias", "weight"]
    assert not any("adapter" in k for k in torch.nn.Module.state_dict(layer))
    assert not any(t.requires_grad for t in (layer.adapter_a, layer.adapter_b, layer.adapter_scales))
    assert layer(_zeros(1, 24), torch.tensor([1])).shape == (1, 16)
    layer.set_adapters(None)
    assert layer.adapter_scales is None


# ---- outputs that overlap inputs: asked of the C entry points, where addresses and strides are known (nothing is launched
# for a refusal, and no pointer is read)

P = 1 << 24
FAR = 1 << 40    # where the arguments lie that are not in question, each FAR from the next


def _status(name, *args):
    lib = _native.load()
    return getattr(lib, name)(*args), lib.ck_last_error().decode()


def _lora_status(rows=4, y=1, x=2, out=7, ys=16, xs=24, os=16, per=1, **at):
    """4 rows, 24 -> 16, rank 8, two adapters; a number below 100 stands for a place of its own."""
    a, b, ids, scales = (at.get(n, i * FAR) for n, i in (("a", 3), ("b", 4), ("ids", 5), ("scales", 6)))
    place = lambda v: v * FAR if v < 100 else v  # noqa: E731
    return _status("launch_lora_add_kernel", place(y), place(x), a, b, ids, scales, place(out), 0, rows, 24, 16, 8, 2, ys, xs, os, per, 2, False, None)


OVERLAPS = [
    dict(y=P, out=P + 32),                          # a row on
    dict(y=P + 32, out=P),
    dict(y=P, out=P + 16),                          # half a row on
    dict(y=P, out=P, os=24),                        # the same address, rows further apart
    dict(y=P, ys=48, out=P + 16, os=48),            # columns that meet, of one buffer
    dict(x=P, out=P),                               # rows of another width: not the same rows
    dict(x=P, out=P + 48),
    dict(x=P, xs=40, out=P + 64, os=40),            # out's row reaches the next one of x
    dict(x=P + 64, xs=40, out=P, os=40),
    dict(a=P, out=P + 2 * 8 * 24 * 2 - 16),         # the end of the adapters
    dict(b=P, out=P - 16),
    dict(ids=P + 112, out=P),                       # the last of four rows
    dict(scales=P + 4, out=P),
    dict(y=P, ys=64, out=P + 16, os=32),            # rows of two spacings
]


@pytest.mark.parametrize("change", OVERLAPS)
def test_lora_output_over_an_input_is_refused(change):
    code, why = _lora_status(**change)
    assert code == -5 and "overlap" in why, (code, why)


def _norm_status(d=64, n=4, xs=64, rs=64, t=2, rt=2, mx=True, x=1, res=2, w=3, scale=4, s=5, y=6, q=7, sf=8):
    place = lambda v: v * FAR if v < 100 else v  # noqa: E731
    return _status("launch_add_rmsnorm_quantize_kernel", place(x), place(res), place(w), 0 if mx else place(scale), place(s), place(y), place(q),
                   place(sf) if mx else 0, n, d, xs, rs, 1e-6, t, rt, 5, None)


@pytest.mark.parametrize("change", [
    dict(s=P + 128, res=P), dict(s=P, res=P + 128), dict(s=P, res=P, rs=128), dict(s=P, x=P, rt=0), dict(s=P, x=P + 32), dict(s=P, x=P, xs=128),
    dict(s=P, w=P + 64), dict(mx=False, s=P, scale=P + 4), dict(s=P, y=P), dict(s=P, q=P + 384), dict(q=P, sf=P + 64), dict(y=P, x=P + 128), dict(q=P, x=P),
    dict(s=P, sf=P + 256),
])
def test_norm_output_over_an_input_is_refused(change):
    code, why = _norm_status(**change)
    assert code in (-2, -5) and ("overlap" in why or "in place" in why), (code, why)


# ---- outputs that the caller gives


@pytest.fixture
def no_launch(monkeypatch):
    monkeypatch.setattr(backend, "_launch", lambda *args: None)


def _given(name):
    """An entry point called with an output of the caller's, and that output: one of its inputs' place, as in place."""
    entry, args = _calls()[name]
    out = args["y" if name == "lora_add" else "residual"]
    return lambda: entry(**args, **{"out" if name == "lora_add" else "sum_out": out}), out


@pytest.mark.parametrize("name", ["lora_add", "mxfp8", "fp8"])
def test_autograd_sees_what_is_written(no_launch, name):
    """A tensor that a backward pass needs and that is overwritten makes that pass fail, as for torch's own operators."""
    call, out = _given(name)
    factor = torch.ones_like(out, requires_grad=True)
    product = (out * factor).sum()
    with torch.no_grad():
        call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        product.backward()
    with torch.inference_mode():        # (no versions there)
        call, out = _given(name)
        call()


@pytest.mark.parametrize("same", [True, False])
def test_given_outputs_under_a_fake_mode(same):
    """The in-place forms are traceable, like those that return new tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        (_, lora), (_, norm) = _calls()["lora_add"], _calls()["mxfp8"]
        out = lora["y"] if same else torch.empty_like(lora["y"])
        assert ck.lora_add(**lora, out=out) is out
        sum_out = norm["residual"] if same else torch.empty_like(norm["residual"])
        for keep in (False, True):
            q, s, h, *y = ck.add_rmsnorm_quantize_mxfp8(**norm, return_norm=keep, sum_out=sum_out)
            assert q.shape == (2, 64) and s.shape == (128, 4) and h is sum_out and [t.shape for t in y] == [norm["x"].shape] * keep
            q, h, *y = ck.add_rmsnorm_quantize_fp8(**norm, scale=torch.ones(1), return_norm=keep, sum_out=sum_out)
            assert q.shape == (2, 64) and q.dtype == torch.float8_e4m3fn and h is sum_out and [t.shape for t in y] == [norm["x"].shape] * keep


# ---- the registry's answers


def test_a_validation_result_cannot_be_changed():
    """One answer serves every call that is in order: a caller that could write to it would change all later ones."""
    import dataclasses

    from comfy_kitchen.constraints import FunctionConstraints, validate_function_call

    good = validate_function_call(FunctionConstraints(), {})
    for field, value in (("success", False), ("failed_param", "x"), ("failure_reason", "y")):
        with pytest.raises(dataclasses.FrozenInstanceError):
            setattr(good, field, value)
    assert validate_function_call(FunctionConstraints(), {}).success


@pytest.mark.parametrize("name,argument", [("lora_add", "a"), ("lora_add", "x"), ("mxfp8", "weight"), ("fp8", "weight"), ("fp8", "scale")])
def test_no_derivative_is_dropped_by_a_traced_write(name, argument):
    """An op that only writes to an argument returns nothing that could ask for a gradient later: the call itself is refused."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    entry = {"lora_add": ck.lora_add, "mxfp8": ck.add_rmsnorm_quantize_mxfp8, "fp8": ck.add_rmsnorm_quantize_fp8}[name]

    def call(args):
        given = torch.empty_like(args["y" if name == "lora_add" else "residual"])
        return entry(**args, **{"out" if name == "lora_add" else "sum_out": given})

    args = _calls()[name][1]
    args[argument] = torch.nn.Parameter(args[argument])
    with pytest.raises(RuntimeError, match="no backward"):
        torch.compile(call, backend="aot_eager")(args)
    torch._dynamo.reset()
    with FakeTensorMode():
        args = _calls()[name][1]
        args[argument] = torch.nn.Parameter(args[argument])
        with pytest.raises(RuntimeError, match="no backward"):
            call(args)
        with torch.no_grad():
            call(args)
