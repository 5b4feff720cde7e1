"""Layer-norm results as other torch operations meet them: forward-mode derivatives, in-place use."""

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


@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64), (64,)])
def test_results_change_in_place(shape):
    x, delta, w, b = _tensors()
    n = x.numel() if len(shape) > 1 else 64
    x, delta = x.flatten()[:n].view(shape), delta.flatten()[:n].view(shape)
    gen = torch.Generator(device=dev).manual_seed(1)
    dy = torch.randn(shape, generator=gen, device=dev)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(layernorm(*leaves), leaves, 2 * dy)
    y = layernorm(*leaves)
    assert y.shape == x.shape and not y._is_view()
    y.mul_(2.0)
    y.add_(1.0)
    for got, expect in zip(torch.autograd.grad(y, leaves, dy), want):
        assert torch.equal(got, expect)
    leaves = [t.clone().requires_grad_() for t in (x, delta, w, b)]
    total, normed = add_layernorm(*leaves)
    want = torch.autograd.grad((total, normed), leaves, (dy, 2 * dy.bfloat16()))
    total, normed = add_layernorm(*leaves)
    assert total.shape == normed.shape == x.shape and not total._is_view() and not normed._is_view()
    normed.mul_(2.0)
    for got, expect in zip(torch.autograd.grad((total, normed), leaves, (dy, dy.bfloat16())), want):
        assert torch.equal(got, expect)
    # the sum is what the backward pass reads: changing it is allowed, a backward pass after it an error
    total, normed = add_layernorm(*leaves)
    total.add_(1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(normed, leaves, dy.bfloat16())
    with torch.no_grad():
        total, normed = add_layernorm(*leaves)
        total.add_(1.0)
        normed.add_(1.0)


def test_graphs_of_the_sum_are_freed():
    """The node keeps its own output: no reference cycle holds the activations."""
    x, delta, w, b = (t.repeat(1000, 1) if t.dim() == 2 else t for t in _tensors(512))
    w.requires_grad_()
    add_layernorm(x, delta, w, b)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(4):
        add_layernorm(x, delta, w, b)
    assert torch.cuda.memory_allocated() <= before


@pytest.mark.parametrize("shape", [(6, 64), (2, 3, 64), (64,)])
def test_rmsnorm_results_change_in_place(shape):
    from packbalance_b200.ops.rmsnorm import rmsnorm

    x, _, w, _ = _tensors()
    x = x.flatten()[: 384 if len(shape) > 1 else 64].view(shape)
    leaves = [t.clone().requires_grad_() for t in (x, w)]
    want = torch.autograd.grad(rmsnorm(*leaves, 1e-5), leaves, 2 * torch.ones_like(x))
    y = rmsnorm(*leaves, 1e-5)
    y.mul_(2.0)
    assert y.shape == x.shape
    for got, expect in zip(torch.autograd.grad(y, leaves, torch.ones_like(x)), want):
        assert torch.equal(got, expect)
