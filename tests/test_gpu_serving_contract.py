"""What the serving operators promise beyond their results on whole, separate, finite tensors."""
import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ck():
    import comfy_kitchen

    return comfy_kitchen


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(g, *shape, dtype=BF16, scale=1.0):
    return (scale * torch.randn(shape, generator=g, device="cuda")).to(dtype)


def _layers(ck, k, n, bias):
    """An NVFP4Linear and an MXFP8Linear of the same weight, with a bias that wants a gradient (as it does by default)."""
    from comfy_kitchen.linear import MXFP8Linear, NVFP4Linear

    g = _gen(12)
    plain = torch.nn.Linear(k, n, bias=bias, device="cuda", dtype=BF16)
    plain.weight.data.copy_(_randn(g, n, k, scale=k ** -0.5))
    ts = plain.weight.data.float().abs().max().reshape(1) / (6 * 448)
    q, sf = ck.quantize_nvfp4(plain.weight.data, ts)
    state = {"weight": q, "weight_scale": sf.view(torch.uint8), "weight_scale_2": ts}
    if bias:
        plain.bias.data.copy_(_randn(g, n))
        state["bias"] = plain.bias.data
    nv = NVFP4Linear(k, n, bias=bias, device="cuda")
    nv.load_state_dict(state, strict=False)
    return nv, MXFP8Linear.from_linear(plain)


def test_layers_with_a_bias_take_adapters(ck):
    k, n, rows = 256, 384, 70
    g = _gen(1)
    a, b = _randn(g, 3, 16, k, scale=0.06), _randn(g, 3, n, 16, scale=0.1)
    x, ids = _randn(g, rows, k), torch.arange(rows, device="cuda") % 4
    for layer in _layers(ck, k, n, True):
        layer.set_adapters(a, b)
        base = layer(x)
        got = layer(x, ids)
        assert got.requires_grad == base.requires_grad
        assert torch.equal(got.detach(), ck.lora_add(base.detach(), x, a, b, ids))
        if got.requires_grad:
            grad = _randn(g, rows, n)
            want, = torch.autograd.grad(base, layer.bias, grad)
            have, = torch.autograd.grad(got, layer.bias, grad)
            assert torch.equal(have, want)
        with torch.no_grad():
            assert torch.equal(layer(x, ids), got.detach())
