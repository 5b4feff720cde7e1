"""Layer norm under torch's other ways to differentiate: forward mode and function transforms."""

import pytest
import torch
from torch.autograd import forward_ad

from packbalance_b200.ops.layernorm import add_layernorm, layernorm

pytestmark = pytest.mark.gpu
dev = "cuda"


def _tensors(n=64):
    gen = torch.Generator(device=dev).manual_seed(0)
    x, w, b = (torch.randn(*s, generator=gen, device=dev) for s in ((6, n), (n,), (n,)))
    return x, torch.randn(6, n, generator=gen, device=dev).bfloat16(), w, b


@pytest.mark.parametrize("which", ["x", "weight", "bias"])
@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("mode", [True, False])
def test_forward_mode_is_refused(which, grad, mode):
    """A tangent that would be lost is an error, whether or not a backward pass is recorded."""
    x, _, w, b = _tensors()
    if grad:
        w.requires_grad_()
    with forward_ad.dual_level(), torch.set_grad_enabled(mode):
        t = {"x": x, "weight": w, "bias": b}
        t[which] = forward_ad.make_dual(t[which].detach(), torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            layernorm(t["x"], t["weight"], t["bias"])


@pytest.mark.parametrize("which", ["x", "delta", "weight", "bias"])
def test_forward_mode_of_the_sum_is_refused(which):
    x, delta, w, b = _tensors()
    with forward_ad.dual_level():
        t = {"x": x, "delta": delta, "weight": w, "bias": b}
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(RuntimeError, match="forward-mode"):
            add_layernorm(t["x"], t["delta"], t["weight"], t["bias"])


def test_function_transforms_are_refused_or_right():
    """Through torch.func nothing is silently wrong: an error, or the derivative."""
    x, _, w, b = _tensors()
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda t: layernorm(t, w, b), (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda t: layernorm(t, w, b))(x.expand(3, 6, 64))
