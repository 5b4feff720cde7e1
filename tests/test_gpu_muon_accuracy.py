"""Accuracy of the fp16 Newton-Schulz iteration on matrices with few dominant directions.

Bounds, from a simulation of the kernels' number formats (X, A, P and the carried rounding error of X
in fp16 at their scales, exact products) against 64 bits, made before the kernels ran: over Gaussian
matrices and sums of rank 1, 2 and 4 plus noise of 3e-3 to 1e-5 the iterate is off by at most 3.7e-3
of its Frobenius norm from 64 rows on (Gaussian 1.9e-3) and by at most 5.2e-3 for 33 to 63 rows, where
fewer roundings average out.  WIDE and FEW are those with the margin of 300 samples per case.  The
update of zero parameters at unit step length returns the iterate unrounded; orthogonalize rounds it
to bf16, at most 2^-8 of each element and independent of the iterate's error: the squares add up."""

import math

import pytest
import torch

from packbalance_b200.ops import _native
from packbalance_b200.ops.muon import COEFFICIENTS, muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
dev = "cuda"
WIDE, FEW = 4e-3, 5.5e-3


def _exact(u, steps=5):
    a, b, c = COEFFICIENTS
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + 1e-7)
    if x.shape[-2] > x.shape[-1]:
        return _exact(u.transpose(-2, -1), steps).transpose(-2, -1)
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def _low_rank(batch, m, n, rank, noise, seed):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    return rand(batch, m, rank) @ rand(batch, rank, n) / rank**0.5 + noise * rand(batch, m, n)


def _off(got, want):
    return float((torch.linalg.matrix_norm(got.double() - want) / torch.linalg.matrix_norm(want)).max())


@pytest.mark.parametrize("rank,noise", [(1, 1e-3), (1, 3e-4), (1, 1e-5), (2, 3e-4), (4, 1e-4), (16, 1e-3)])
@pytest.mark.parametrize("batch,m,n", [(8, 64, 64), (4, 64, 200), (4, 128, 128), (4, 256, 768), (4, 768, 256),
                                       (3, 512, 1408), (2, 768, 768), (20, 33, 40), (20, 45, 200)])
def test_one_to_sixteen_dominant_directions(batch, m, n, rank, noise):
    u = _low_rank(batch, m, n, rank, noise, seed=m + rank)
    want = _exact(u)
    bound = WIDE if min(m, n) >= 64 else FEW
    p, mom = torch.zeros_like(u), torch.zeros_like(u)
    # momentum 0 without Nesterov: the direction is the gradient, p = -orthogonalised u
    muon_update_([p], [u], [mom], lr=1.0 / (0.2 * math.sqrt(max(m, n))), momentum=0.0, nesterov=False, weight_decay=0.0)
    _native.check_status()
    assert torch.equal(mom, u)
    off = _off(-p, want)
    print(f"{batch}x{m}x{n} rank {rank} + {noise}: {off:.2e}")
    assert off <= bound
    assert _off(orthogonalize(u), want) <= math.hypot(bound, 2.0**-8)


@pytest.mark.parametrize("scale", [1e-9, 1e-11, 1e-13])
@pytest.mark.parametrize("m,n", [(64, 200), (256, 768), (1024, 1024)])
def test_matrices_far_smaller_than_eps(m, n, scale):
    """Down to |x|_F = 1e-6 eps the carried rounding errors hold what fp16 loses (simulated: 2.1e-3)."""
    x = torch.randn(2, m, n, generator=torch.Generator(device=dev).manual_seed(n), device=dev)
    x = x / torch.linalg.matrix_norm(x, keepdim=True) * scale
    p, mom = torch.zeros_like(x), torch.zeros_like(x)
    muon_update_([p], [x], [mom], lr=1.0 / (0.2 * math.sqrt(max(m, n))), momentum=0.0, nesterov=False, weight_decay=0.0)
    assert _off(-p, _exact(x)) <= WIDE


def test_the_largest_iterates_that_do_not_overflow():
    """Singular values of 7.9 before the last step: A stays below 64.  Each of the three steps rounds
    its factor and its iterate by at most 2^-11 together with the Gram matrix not entering."""
    q = torch.linalg.qr(torch.randn(128, 128, generator=torch.Generator(device=dev).manual_seed(1), device=dev))[0]
    a = (7.9 * 128**0.5) ** 0.5
    y = orthogonalize(q, steps=3, coefficients=(a, 0.0, 0.0))
    _native.check_status()
    assert _off(y, a**3 * q.double() / 128**0.5) <= 3 * 2 * 2.0**-11 + 2.0**-8
