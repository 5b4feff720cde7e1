"""Native Newton-Schulz orthogonalisation and Muon update against 64 bits.

Bounds.  The fp16 iteration (operands rounded to 2^-11, early rounding errors carried along)
was simulated against 64 bits over Gaussian, low-rank and power-law spectra before the kernel
ran: at most 2.9e-3 of the result's Frobenius norm.  The bf16 result adds at most half a step,
2^-8, per element.  ITER = 3e-3 and NORM = ITER + 2^-8 are those.
"""

import math

import pytest
import torch

from packbalance_b200.ops import _native
from packbalance_b200.ops.muon import COEFFICIENTS, muon_update_, orthogonalize

pytestmark = pytest.mark.gpu
dev = "cuda"
ITER = 3e-3
NORM = ITER + 2.0**-8


def _exact(u, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = u.double()
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + eps)
    if x.shape[-2] > x.shape[-1]:
        return _exact(u.transpose(-2, -1), steps, coefficients, eps).transpose(-2, -1)
    for _ in range(steps):
        gram = x @ x.transpose(-2, -1)
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return x


def _rand(*shape, seed=0):
    return torch.randn(*shape, generator=torch.Generator(device=dev).manual_seed(seed), device=dev)


def _off(got, want):
    """Largest relative Frobenius distance over the matrices of a batch."""
    d = torch.linalg.matrix_norm(got.double() - want)
    return float((d / torch.linalg.matrix_norm(want).clamp_min(1e-300)).max())


SHAPES = [(1, 1, 1), (1, 1, 17), (2, 17, 1), (3, 2, 3), (1, 31, 33), (1, 64, 64), (2, 63, 130), (1, 128, 128),
          (1, 129, 257), (1, 257, 129), (2, 100, 1001), (2, 1001, 100), (1, 256, 768), (1, 768, 256), (3, 333, 1407),
          (80, 256, 264), (40, 300, 500), (40, 500, 300), (24, 768, 768), (6, 2048, 768), (300, 16, 24)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,m,n", SHAPES)
def test_orthogonalize_matches_definition(batch, m, n, dtype):
    x = _rand(batch, m, n, seed=m + n).to(dtype)
    y = orthogonalize(x)
    _native.check_status()
    assert y.dtype == torch.bfloat16 and y.shape == x.shape and y.is_contiguous()
    assert _off(y, _exact(x)) <= NORM


@pytest.mark.parametrize("m,n", [(200, 320), (320, 200), (300, 300)])
@pytest.mark.parametrize("spectrum", ["rank1", "rank8", "rank8_noise", "power", "rows", "huge", "tiny"])
def test_spectra(m, n, spectrum):
    r = min(m, n)
    x = _rand(2, m, n, seed=3)
    if spectrum.startswith("rank"):
        k = 1 if spectrum == "rank1" else 8
        x = torch.bmm(_rand(2, m, k, seed=4), _rand(2, k, n, seed=5)) + (1e-3 * x if "noise" in spectrum else 0)
    elif spectrum == "power":
        u, _, v = torch.linalg.svd(x, full_matrices=False)
        x = (u / torch.arange(1, r + 1, device=dev)) @ v
    elif spectrum == "rows":
        x = x * torch.exp(1.5 * _rand(2, m, 1, seed=6))
    else:
        x = x * (1e25 if spectrum == "huge" else 1e-3)
    assert _off(orthogonalize(x), _exact(x)) <= NORM


@pytest.mark.parametrize("steps", [1, 2, 3, 4, 7])
def test_steps_and_coefficients(steps):
    x = _rand(2, 96, 200)
    assert _off(orthogonalize(x, steps=steps), _exact(x, steps)) <= NORM
    cubic = (1.5, -0.5, 0.0)  # the classical iteration
    assert _off(orthogonalize(x, steps=steps, coefficients=cubic), _exact(x, steps, cubic)) <= NORM


def test_zero_and_nonfinite_matrices_stay_apart():
    x = _rand(5, 150, 210)
    want = orthogonalize(x)
    x[1] = 0
    x[3, 7, 9] = float("nan")
    y = orthogonalize(x)
    assert not y[1].any()
    assert bool(y[3].isnan().all())
    for k in (0, 2, 4):
        assert torch.equal(y[k], want[k])


def test_views_strides_and_leading_dimensions():
    x = _rand(3, 2, 130, 90)
    want = orthogonalize(x)
    assert torch.equal(orthogonalize(x.reshape(6, 130, 90)), want.reshape(6, 130, 90))
    assert torch.equal(orthogonalize(x[1, 0]), want[1, 0])
    assert _off(orthogonalize(x.transpose(-2, -1)), _exact(x.transpose(-2, -1))) <= NORM
    wide = _rand(4, 64, 100)
    assert torch.equal(orthogonalize(wide[::2, :, 3:67]), orthogonalize(wide[::2, :, 3:67].contiguous()))
    odd = torch.cat((torch.zeros(1, device=dev), wide.flatten()))[1:].view(4, 64, 100)  # 4-byte aligned
    assert torch.equal(orthogonalize(odd), orthogonalize(wide))
    assert orthogonalize(torch.ones(0, 4, 5, device=dev)).shape == (0, 4, 5)
    assert orthogonalize(torch.ones(2, 0, 5, device=dev)).shape == (2, 0, 5)


def test_repeatable_on_two_streams_at_once():
    x = [_rand(24, 256, 512, seed=k) for k in range(2)]
    want = [orthogonalize(t) for t in x]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(3):
        for k, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[k].append(orthogonalize(x[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for y in got[k]:
            assert torch.equal(y, want[k])


def _problem(shapes, seed=0, scale=1e-3):
    p = [0.02 * _rand(*s, seed=seed + 3 * k) for k, s in enumerate(shapes)]
    g = [scale * _rand(*s, seed=seed + 3 * k + 1) for k, s in enumerate(shapes)]
    m = [0.3 * scale * _rand(*s, seed=seed + 3 * k + 2) for k, s in enumerate(shapes)]
    return p, g, m


def _check_update(before, g, after, lr, mu, wd, nesterov=True, clip=1.0):
    p0, m0 = before
    p1, m1 = after
    for k in range(len(g)):
        gk = g[k].double() * clip
        m = m0[k].double() + (1 - mu) * (gk - m0[k].double())
        u = gk + mu * (m - gk) if nesterov else m
        # a difference, two products and two sums in fp32
        assert bool(((m1[k].double() - m).abs() <= 2.0**-22 * (m0[k].double().abs() + gk.abs())).all())
        o = _exact(u)
        step = lr * 0.2 * math.sqrt(max(p0[k].shape[-2:]))
        want = p0[k].double() * (1 - lr * wd) - step * o
        tol = step * ITER * torch.linalg.matrix_norm(o) + 2.0**-22 * torch.linalg.matrix_norm(p0[k].double() + step * o)
        assert bool((torch.linalg.matrix_norm(p1[k].double() - want) <= tol).all()), k


# q/o, k/v, gate/up and down of a small decoder, odd ones, stacks, a single row and column
LISTS = {
    "decoder": [(192, 192), (64, 192), (64, 192), (192, 192), (512, 192), (512, 192), (192, 512)],
    "odd": [(3, 77, 131), (131, 77), (1, 50), (50, 1), (7, 7)],
    "many_shapes": [(8 * k + 8, 40 + k) for k in range(19)],
    "many_matrices": [(250, 12, 20), (16, 16), (3, 20, 12)],
    "large": [(6, 768, 768), (4, 2048, 768), (2, 768, 2048), (6, 256, 768)],
}


@pytest.mark.parametrize("which", LISTS)
@pytest.mark.parametrize("nesterov", [True, False])
def test_update_matches_definition(which, nesterov):
    p, g, m = _problem(LISTS[which])
    before = [t.clone() for t in p], [t.clone() for t in m]
    sh = [torch.zeros_like(t, dtype=torch.bfloat16) for t in p]
    muon_update_(p, g, m, lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, shadows=sh)
    _native.check_status()
    _check_update(before, g, (p, m), 0.02, 0.9, 0.1, nesterov)
    for a, b in zip(sh, p):
        assert torch.equal(a, b.bfloat16())


def test_update_clips_skips_and_reads_the_rate_on_the_device():
    p, g, m = _problem(LISTS["decoder"], seed=50)
    before = [t.clone() for t in p], [t.clone() for t in m]
    norm = torch.tensor(4.0, device=dev)
    hp = torch.tensor([0.01, 0.5, 0.5], device=dev)
    muon_update_(p, g, m, lr=123.0, weight_decay=0.1, grad_norm=norm, max_norm=1.0, hparams=hp)
    _check_update(before, g, (p, m), 0.01, 0.95, 0.1, clip=1.0 / (4.0 + 1e-6))
    kept = [t.clone() for t in p + m]
    for bad in (math.inf, math.nan):
        muon_update_(p, g, m, lr=0.01, grad_norm=torch.tensor(bad, device=dev), max_norm=1.0)
    torch.cuda.synchronize()
    for a, b in zip(kept, p + m):
        assert torch.equal(a, b)


def test_update_of_unaligned_views_leaves_the_rest_alone():
    """Matrices back to back in one buffer at odd offsets, as flat parameter buffers hold them."""
    shapes = [(33, 65), (65, 33), (10, 10), (128, 256)]
    total = sum(a * b for a, b in shapes) + 3
    flat = [_rand(total, seed=k) for k in range(3)]
    keep = [t.clone() for t in flat]
    views = [[], [], []]
    at = 1
    for a, b in shapes:
        for k in range(3):
            views[k].append(flat[k][at : at + a * b].view(a, b))
        at += a * b
    before = [t.clone() for t in views[0]], [t.clone() for t in views[2]]
    muon_update_(views[0], views[1], views[2], lr=0.02, momentum=0.9, weight_decay=0.1)
    _check_update(before, views[1], (views[0], views[2]), 0.02, 0.9, 0.1)
    for k in range(3):
        assert torch.equal(flat[k][:1], keep[k][:1]) and torch.equal(flat[k][-2:], keep[k][-2:])
    assert torch.equal(flat[1], keep[1])


def test_graph_replay_equals_eager():
    p, g, m = _problem(LISTS["decoder"], seed=7)
    q, _, n = _problem(LISTS["decoder"], seed=7)
    hp = torch.tensor([0.01], device=dev)
    muon_update_(*_problem(LISTS["decoder"], seed=8), lr=0.0, hparams=hp)  # warm up
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_update_(p, g, m, lr=0.0, hparams=hp)
    for k in range(3):
        hp.fill_(0.01 * (k + 1))
        for t in g:
            t.mul_(-0.5)
        graph.replay()
        muon_update_(q, g, n, lr=0.01 * (k + 1), hparams=hp)
    for a, b in zip(p + m, q + n):
        assert torch.equal(a, b)


def test_native_refusals():
    p, g, m = _problem([(8, 16)])
    both = torch.zeros(200, device=dev)
    for call, message in [
        (lambda: muon_update_(p * 2, g * 2, [m[0], m[0].clone()], lr=0.1), "listed twice"),
        (lambda: muon_update_([p[0], both[:128].view(8, 16)], g * 2, [m[0], both[64:192].view(8, 16)], lr=0.1),
         "overlap"),
        (lambda: muon_update_(p, m, m, lr=0.1), "gradients must not overlap"),
        (lambda: muon_update_(p, p, m, lr=0.1), "gradients must not overlap"),
        (lambda: muon_update_(p, g, m, lr=0.1, shadows=[p[0].clone()]), "bf16"),
        (lambda: muon_update_(p, g, m, lr=0.1, shadows=[p[0].bfloat16()[:4]]), "size"),
        (lambda: muon_update_(p, g, m, lr=0.1, grad_norm=torch.tensor(1.0), max_norm=1.0), "norm"),
        (lambda: muon_update_(p, g, m, lr=0.1, hparams=torch.tensor([1.0])), "hp"),
        (lambda: muon_update_(p, g, m, lr=0.1, coefficients=(1.0, math.nan, 0.0)), "finite"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            call()
    with pytest.raises(ValueError, match="one device"):
        muon_update_(p, [g[0].cpu()], m, lr=0.1)


# rows (or columns) of 32 and fewer go to one cluster per matrix: slices of odd length, more
# matrices than fit at once, and a long side beyond shared memory
@pytest.mark.parametrize("batch,m,n", [(1, 32, 3001), (2, 7, 5000), (2, 5000, 31), (40, 16, 2500), (200, 9, 700),
                                       (1, 5, 60001), (1, 60001, 30), (3, 300, 1)])
def test_few_rows_and_a_long_side(batch, m, n):
    x = _rand(batch, m, n, seed=m)
    x = x * torch.exp(_rand(batch, m, 1, seed=n))  # rows of unequal size
    assert _off(orthogonalize(x), _exact(x)) <= 2.0**-8 + 1e-4
    p, g, mom = [0.02 * x], [1e-3 * _rand(batch, m, n, seed=2)], [torch.zeros_like(x)]
    before = [t.clone() for t in p], [t.clone() for t in mom]
    muon_update_(p, g, mom, lr=0.02, momentum=0.9, weight_decay=0.1)
    _check_update(before, g, (p, mom), 0.02, 0.9, 0.1)
