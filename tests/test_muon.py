"""Newton-Schulz orthogonalisation and the Muon update: the CPU path against the definition in
64 bits, and what the entry points refuse."""

import math

import pytest
import torch

from packbalance_b200.ops.muon import COEFFICIENTS, orthogonalize, muon_update_


def exact_newton_schulz(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Per matrix, in 64 bits, through the singular values: every step maps s to
    a s + b s^3 + c s^5 and leaves the singular vectors alone."""
    a, b, c = coefficients
    w, s, v = torch.linalg.svd(u.double(), full_matrices=False)
    s = s / (s.square().sum(-1, keepdim=True).sqrt() + eps)
    for _ in range(steps):
        s = a * s + b * s**3 + c * s**5
    return (w * s.unsqueeze(-2)) @ v


@pytest.mark.parametrize("shape", [(1, 1), (1, 9), (9, 1), (6, 6), (5, 12), (12, 5), (3, 2, 4, 7)])
def test_cpu_matches_singular_value_map(shape) -> None:
    x = torch.randn(*shape, generator=torch.Generator().manual_seed(0))
    y = orthogonalize(x)
    assert y.dtype == torch.bfloat16 and y.shape == x.shape
    torch.testing.assert_close(y.double(), exact_newton_schulz(x), atol=1e-4, rtol=2**-8 + 1e-3)


def test_cpu_singular_values_end_near_one() -> None:
    x = torch.randn(16, 40, generator=torch.Generator().manual_seed(1))
    s = torch.linalg.svdvals(orthogonalize(x).double())
    assert 0.6 < float(s.min()) and float(s.max()) < 1.3


@pytest.mark.parametrize("nesterov", [True, False])
@pytest.mark.parametrize("clip", [False, True])
def test_cpu_update_matches_definition(nesterov, clip) -> None:
    gen = torch.Generator().manual_seed(2)
    shapes = [(6, 8), (2, 10, 4), (6, 8)]
    p, g, m = ([torch.randn(*s, generator=gen) for s in shapes] for _ in range(3))
    sh = [t.bfloat16() for t in p]
    p0, m0 = [t.double() for t in p], [t.double() for t in m]
    norm = torch.tensor(8.0) if clip else None
    muon_update_(p, g, m, lr=0.1, momentum=0.9, nesterov=nesterov, weight_decay=0.2, shadows=sh, grad_norm=norm,
                 max_norm=2.0)
    for k in range(3):
        gk = g[k].double() * (2.0 / (8.0 + 1e-6) if clip else 1.0)
        mk = 0.9 * m0[k] + 0.1 * gk
        u = 0.1 * gk + 0.9 * mk if nesterov else mk
        want = p0[k] * (1 - 0.1 * 0.2) - 0.1 * 0.2 * math.sqrt(max(p[k].shape[-2:])) * exact_newton_schulz(u)
        torch.testing.assert_close(m[k].double(), mk, atol=1e-6, rtol=1e-5)
        torch.testing.assert_close(p[k].double(), want, atol=1e-5, rtol=1e-4)
        assert torch.equal(sh[k], p[k].bfloat16())


def test_cpu_nonfinite_norm_changes_nothing() -> None:
    p, g, m = torch.ones(3, 4), torch.ones(3, 4), torch.ones(3, 4)
    for bad in (math.inf, math.nan):
        muon_update_([p], [g], [m], lr=1.0, grad_norm=torch.tensor(bad), max_norm=1.0)
    assert torch.equal(p, torch.ones(3, 4)) and torch.equal(m, torch.ones(3, 4))


def _one():
    return torch.ones(3, 4)


@pytest.mark.parametrize("call,message", [
    (lambda: orthogonalize(torch.ones(4)), "two dimensions"),
    (lambda: orthogonalize(torch.ones(4, 4).double()), "fp32 or bf16"),
    (lambda: orthogonalize(torch.ones(4, 4).half()), "fp32 or bf16"),
    (lambda: orthogonalize(_one(), steps=0), "steps"),
    (lambda: orthogonalize(_one(), steps=101), "steps"),
    (lambda: orthogonalize(_one(), coefficients=(1.0, 2.0)), "three coefficients"),
    (lambda: muon_update_([_one()], [], [_one()], lr=0.1), "0 grads"),
    (lambda: muon_update_([_one()], [_one()], [_one()], lr=0.1, shadows=[]), "0 shadows"),
    (lambda: muon_update_([torch.ones(4)], [torch.ones(4)], [torch.ones(4)], lr=0.1), "rows, cols"),
    (lambda: muon_update_([_one()], [torch.ones(4, 3)], [_one()], lr=0.1), "one shape"),
    (lambda: muon_update_([_one()], [_one().double()], [_one()], lr=0.1), "fp32"),
    (lambda: muon_update_([torch.ones(4, 3).t()], [_one()], [_one()], lr=0.1), "contiguous"),
])
def test_refusals(call, message) -> None:
    with pytest.raises(ValueError, match=message):
        call()


_flat = torch.zeros(64)


def _at(i, j):
    return _flat[i:j].view(-1, 4)


@pytest.mark.parametrize("p,g,m,shadows,message", [
    ([_at(0, 12), _at(0, 12)], [_one(), _one()], [_one(), _one()], None, "listed twice"),
    ([_at(0, 12), _at(8, 20)], [_one(), _one()], [_one(), _one()], None, "listed twice"),
    ([_at(0, 12)], [_one()], [_at(8, 20)], None, "listed twice"),
    ([_at(0, 12), _at(12, 24)], [_one(), _at(0, 12)], [_one(), _one()], None, "gradients must not overlap"),
    ([_at(0, 12), _at(16, 28)], [_one(), _at(8, 20)], [_one(), _one()], None, "gradients must not overlap"),
    ([_one()], [_at(0, 12)], [_at(0, 12)], None, "gradients must not overlap"),
    ([_at(0, 12)], [_one()], [_one()], [_at(0, 12)], "bf16"),
    ([_at(0, 12)], [_one()], [_one()], [torch.zeros(3, 3).bfloat16()], "size"),
    ([_at(0, 12)], [_one()], [_one()], [torch.zeros(12)[4:10].view(torch.bfloat16).view(4, 3).t()], "contiguous"),
])
def test_cpu_update_refuses_what_the_native_one_refuses(p, g, m, shadows, message) -> None:
    before = _flat.clone()
    with pytest.raises(ValueError, match=message):
        muon_update_(p, g, m, lr=0.1, shadows=shadows)
    assert torch.equal(_flat, before)


def test_cpu_update_of_neighbours_and_of_a_transposed_gradient() -> None:
    """Parameters, momenta and gradients back to back in one buffer touch but do not overlap; a
    transposed view of a parameter as gradient is read before anything is written."""
    buf = torch.randn(48, generator=torch.Generator().manual_seed(5))
    p, m, g = ([buf[k : k + 8].view(2, 4), buf[k + 8 : k + 16].view(4, 2)] for k in (0, 16, 32))
    want = [t.clone() for t in p], [t.clone() for t in m]
    muon_update_(want[0], [t.clone() for t in g], want[1], lr=0.1)
    muon_update_(p, g, m, lr=0.1)
    for got, expect in zip(p + m, want[0] + want[1]):
        assert torch.equal(got, expect)
    q = [torch.ones(2, 4), torch.randn(4, 2, generator=torch.Generator().manual_seed(6))]
    n = [torch.zeros(2, 4), torch.zeros(4, 2)]
    r, s = [t.clone() for t in q], [t.clone() for t in n]
    muon_update_(r, [torch.ones(2, 4), r[0].clone().t()], s, lr=0.1)
    muon_update_(q, [torch.ones(2, 4), q[0].t()], n, lr=0.1)
    for got, expect in zip(q + n, r + s):
        assert torch.equal(got, expect)


def test_empty_lists_and_empty_matrices() -> None:
    muon_update_([], [], [], lr=0.1)
    assert orthogonalize(torch.ones(0, 3, 4)).shape == (0, 3, 4)
