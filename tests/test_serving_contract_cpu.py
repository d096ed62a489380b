"""What the serving operators promise beyond their refusals of shapes and types, checked without a GPU."""
import pytest
import torch
from torch.autograd import forward_ad

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
