"""Derivatives that the dense operators do not have are refused instead of dropped."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from fast_b200.ops import fused

BF = torch.bfloat16


def _calls(device):
    def t(*shape, dtype=BF):
        return torch.ones(*shape, device=device, dtype=dtype)

    x, w, b, r, nw = t(4, 64), t(256, 64), t(256), t(4, 256), t(64)
    logits, idx = t(4, 8, dtype=torch.float32), torch.zeros(4, 2, device=device, dtype=torch.int32)
    q, scales = t(4, 128, dtype=torch.uint8), t(4, 1, dtype=torch.float32)
    return {
        "linear x": (x, lambda v: fused.linear(v, w)), "linear weight": (w, lambda v: fused.linear(x, v)), "linear bias": (b, lambda v: fused.linear(x, w, bias=v, activation="gelu")),
        "linear residual": (r, lambda v: fused.linear(x, w, residual=v)), "swiglu": (x, lambda v: fused.linear(v, w, activation="swiglu")),
        "norm x": (x, lambda v: fused.add_rms_norm(v, nw).y), "norm weight": (nw, lambda v: fused.add_rms_norm(x, v).y), "norm residual": (x, lambda v: fused.add_rms_norm(x, nw, residual=v).y),
        "balance": (logits, lambda v: fused.balance_loss(v, idx)[0]), "dequantise": (scales, lambda v: fused.dequantise_rows(q, v)),
    }


NAMES = sorted(_calls("cpu"))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused(name, grad):
    """Before anything is looked at but the tangent, so a tensor of the host shows it."""
    at, call = _calls("cpu")[name]
    with fwad.dual_level(), torch.set_grad_enabled(grad):
        dual = fwad.make_dual(at.clone().requires_grad_(grad), torch.ones_like(at))
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            call(dual)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_a_tangent_is_refused_on_the_device_and_values_are_not(name):
    at, call = _calls("cuda")[name]
    want = call(at)
    with fwad.dual_level():
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            call(fwad.make_dual(at, torch.ones_like(at)))
        assert torch.equal(call(at), want) and torch.equal(call(fwad.unpack_dual(fwad.make_dual(at, torch.ones_like(at))).primal), want)


@pytest.mark.gpu
def test_scales_that_require_a_gradient_are_refused():
    at, call = _calls("cuda")["dequantise"]
    with pytest.raises(RuntimeError, match="no gradient"):
        call(at.clone().requires_grad_())
    with torch.no_grad():
        assert torch.equal(call(at.clone().requires_grad_()), call(at))
