"""Layer normalisation: the CPU path against its definition, and what the entry points refuse."""

import pytest
import torch

from packbalance_b200.ops.layernorm import add_layernorm, layernorm


def _definition(x, w, b, eps):
    mean = x.sum(-1, keepdim=True) / x.shape[-1]
    var = ((x - mean) ** 2).sum(-1, keepdim=True) / x.shape[-1]
    y = (x - mean) / torch.sqrt(var + eps) * w
    return y if b is None else y + b


@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (2, 5, 33), (0, 8)])
@pytest.mark.parametrize("with_bias", [True, False])
def test_cpu_matches_definition_with_gradients(shape, with_bias) -> None:
    gen = torch.Generator().manual_seed(1)
    n = shape[-1]
    x, w, b, dy = (torch.randn(*s, generator=gen) for s in (shape, (n,), (n,), shape))
    leaves = [t.clone().requires_grad_() for t in ((x, w, b) if with_bias else (x, w))]
    exact = [t.double().requires_grad_() for t in ((x, w, b) if with_bias else (x, w))]
    y = layernorm(leaves[0], leaves[1], leaves[2] if with_bias else None, 1e-2)
    ref = _definition(exact[0], exact[1], exact[2] if with_bias else None, 1e-2)
    torch.testing.assert_close(y.double(), ref, atol=1e-5, rtol=1e-5)
    for got, want in zip(torch.autograd.grad(y, leaves, dy), torch.autograd.grad(ref, exact, dy.double())):
        torch.testing.assert_close(got.double(), want, atol=1e-4, rtol=1e-4)


def test_gradient_of_the_definition_by_differences() -> None:
    """dL/dx of the formula the kernels use, against central differences in 64 bits."""
    gen = torch.Generator().manual_seed(2)
    x, w, b, dy = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((2, 9), (9,), (9,), (2, 9)))
    mean = x.mean(-1, keepdim=True)
    r = 1 / torch.sqrt(((x - mean) ** 2).mean(-1, keepdim=True) + 1e-2)
    xh, g = (x - mean) * r, dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    h = 1e-5
    for i in range(2):
        for j in range(9):
            e = torch.zeros_like(x)
            e[i, j] = h
            diff = ((_definition(x + e, w, b, 1e-2) - _definition(x - e, w, b, 1e-2)) * dy).sum() / (2 * h)
            assert abs(diff - dx[i, j]) < 1e-7


def test_add_layernorm_cpu() -> None:
    gen = torch.Generator().manual_seed(3)
    x, delta = torch.randn(4, 10, generator=gen), torch.randn(4, 10, generator=gen).bfloat16()
    w, b = torch.randn(10, generator=gen), torch.randn(10, generator=gen)
    total, y = add_layernorm(x, delta, w, b, 1e-5)
    assert total.dtype == torch.float32 and y.dtype == torch.bfloat16
    assert torch.equal(total, x + delta.float())
    torch.testing.assert_close(y.double(), _definition(total.double(), w.double(), b.double(), 1e-5),
                               atol=1e-5, rtol=2**-8)


@pytest.mark.parametrize("call,message", [
    (lambda: layernorm(torch.ones(2, 4, dtype=torch.float64), torch.ones(4)), "fp32 or bf16"),
    (lambda: layernorm(torch.ones(2, 4, dtype=torch.float16), torch.ones(4)), "fp32 or bf16"),
    (lambda: layernorm(torch.ones(2, 4), torch.ones(5)), "weight must have shape"),
    (lambda: layernorm(torch.ones(2, 4), torch.ones(1, 4)), "weight must have shape"),
    (lambda: layernorm(torch.ones(2, 4), torch.ones(4), torch.ones(3)), "bias must have shape"),
    (lambda: layernorm(torch.ones(2, 0), torch.ones(0)), "non-empty last dimension"),
    (lambda: layernorm(torch.tensor(1.0), torch.ones(1)), "non-empty last dimension"),
    (lambda: add_layernorm(torch.ones(2, 4), torch.ones(2, 4), torch.ones(4)), "bf16 delta"),
    (lambda: add_layernorm(torch.ones(2, 4), torch.ones(1, 4).bfloat16(), torch.ones(4)), "same shape"),
    (lambda: add_layernorm(torch.ones(2, 4).bfloat16(), torch.ones(2, 4).bfloat16(), torch.ones(4)), "fp32 x"),
])
def test_refusals(call, message) -> None:
    with pytest.raises(ValueError, match=message):
        call()
