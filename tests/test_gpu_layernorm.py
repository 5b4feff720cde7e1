"""Native layer normalisation against its definition in 64 bits.

Bounds.  With u = 2^-24, a sum of n terms in any order is off by at most (n + 16) u times the
sum of the terms' magnitudes (the kernels add in trees, so this is generous); ``k`` covers the
handful of roundings around it.  A bf16 result adds half a step, 2^-8 of its value.
"""

import pytest
import torch

from packbalance_b200.ops import _native
from packbalance_b200.ops.layernorm import add_layernorm, layernorm

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0**-24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0**-8}


def _inputs(rows, n, dtype, seed=0):
    gen = torch.Generator(device=dev).manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    x = rand(rows, n) + 0.5
    x[:, :: max(1, n // 3)] *= 6.0
    return x.to(dtype), 1.0 + 0.2 * rand(n), 0.3 * rand(n), rand(rows, n).to(dtype)


class _Exact:
    """Definition in 64 bits with a bound on what 32-bit evaluation may add."""

    def __init__(self, x, w, b, eps, dy=None, dres=None):
        x, w = x.double(), w.double()
        rows, n = x.shape
        mean = x.mean(1, keepdim=True)
        self.std = torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
        xh = (x - mean) / self.std
        gamma = (n + 16) * U
        # xh: the mean's error over the deviation, the deviation's own relative error
        e = 2 * gamma * (x.abs().mean(1, keepdim=True) / self.std) + (2 * gamma + 8 * U) * xh.abs()
        e = e + 4 * U * x.abs() / self.std
        self.y = xh * w + (0 if b is None else b.double())
        self.y_tol = e * w.abs() + 4 * U * (self.y.abs() + (xh * w).abs())
        if dy is None:
            return
        dy = dy.double()
        g = dy * w
        gm, gx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        self.dx = (g - gm - xh * gx) / self.std
        mag = g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True)
        drift = e * gx.abs() + xh.abs() * (g.abs() * e).mean(1, keepdim=True)
        self.dx_tol = (2 * (gamma + 8 * U) * mag + 2 * drift) / self.std
        if dres is not None:
            self.dx = self.dx + dres.double()
            self.dx_tol = self.dx_tol + 2 * U * (self.dx.abs() + dres.double().abs())
        gr = (rows + 16) * U
        self.dw, self.db = (dy * xh).sum(0), dy.sum(0)
        self.dw_tol = gr * (dy * xh).abs().sum(0) + (dy.abs() * e).sum(0)
        self.db_tol = gr * dy.abs().sum(0)


def _near(got, want, tol):
    tol = tol + HALF_STEP[got.dtype] * want.abs() * (1 + 2**-6) + 1e-30
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.3g} bounds"


SHAPES = [(1, 1), (1, 4096), (7, 2), (3, 31), (5, 33), (257, 64), (40, 127), (333, 768), (129, 1000), (65, 1409),
          (600, 2048), (31, 4096), (17, 5001), (9, 8192), (3, 16384), (2, 40001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", SHAPES)
def test_forward_and_gradients(rows, n, dtype):
    x, w, b, dy = _inputs(rows, n, dtype, seed=n)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = layernorm(*leaves, 1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    ex = _Exact(x, w, b, 1e-5, dy)
    assert y.dtype == dx.dtype == dtype and dw.dtype == db.dtype == torch.float32
    _near(y.detach(), ex.y, ex.y_tol)
    _near(dx, ex.dx, ex.dx_tol)
    _near(dw, ex.dw, ex.dw_tol)
    _near(db, ex.db, ex.db_tol)


@pytest.mark.parametrize("rows,n", [(1, 8), (64, 768), (300, 770), (33, 1409), (5, 4096), (1200, 512)])
def test_add_forward_and_gradients(rows, n):
    x, w, b, _ = _inputs(rows, n, torch.float32, seed=n)
    gen = torch.Generator(device=dev).manual_seed(5)
    delta, dy = (torch.randn(rows, n, generator=gen, device=dev).bfloat16() for _ in range(2))
    dsum = torch.randn(rows, n, generator=gen, device=dev)
    leaves = [t.clone().requires_grad_() for t in (x, delta, w, b)]
    total, y = add_layernorm(*leaves, 1e-5)
    dx, dd, dw, db = torch.autograd.grad((total, y), leaves, (dsum, dy))
    assert torch.equal(total.detach(), x + delta.float())
    ex = _Exact(total.detach(), w, b, 1e-5, dy, dsum)
    assert y.dtype == dd.dtype == torch.bfloat16 and dx.dtype == torch.float32
    _near(y.detach(), ex.y, ex.y_tol)
    _near(dx, ex.dx, ex.dx_tol)
    assert torch.equal(dd, dx.bfloat16())
    _near(dw, ex.dw, ex.dw_tol)
    _near(db, ex.db, ex.db_tol)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", [(9001, 128), (8192, 256), (8192, 512), (8192, 768), (4097, 1408), (3000, 2048),
                                    (2500, 4096), (1500, 8192), (400, 16384), (6000, 257), (3000, 1409)])
def test_many_rows_per_block(rows, n, dtype):
    """Every slot of the row ring is filled several times; every type of dy, with and without a
    residual gradient; the memory the calls get holds NaN beforehand."""
    C = _native.module()
    x, w, b, dy = _inputs(rows, n, dtype, seed=n)
    _, y, mean, rstd = C.add_layernorm_fwd(x, None, w, b, 1e-5, False)
    dres = torch.randn(rows, n, device=dev) if dtype == torch.float32 else None
    for g, res in ((dy, None), (dy, dres), (dy.bfloat16(), dres), (dy.bfloat16(), None)):
        if res is None and dtype == torch.float32 and g.dtype == torch.bfloat16:
            continue
        ex = _Exact(x, w, b, 1e-5, g, res)
        _near(y, ex.y, ex.y_tol)
        copy = torch.empty(rows, n, device=dev, dtype=torch.bfloat16) if dtype == torch.float32 else None
        for _ in range(4):
            torch.full((2 * 512 * n,), float("nan"), device=dev)
            dw, db = torch.empty(n, device=dev), torch.empty(n, device=dev)
            dx = C.layernorm_bwd(g, x, w, mean, rstd, res, copy, dw, db, False)
            _near(dw, ex.dw, ex.dw_tol)
            _near(db, ex.db, ex.db_tol)
        _near(dx, ex.dx, ex.dx_tol)
        if copy is not None:
            assert torch.equal(copy, dx.bfloat16())


def test_unused_sum_output_has_zero_gradient():
    x, w, b, _ = _inputs(12, 96, torch.float32)
    delta = torch.zeros(12, 96, device=dev, dtype=torch.bfloat16)
    x1 = x.clone().requires_grad_()
    _, y = add_layernorm(x1, delta, w, b, 1e-5)
    dy = torch.ones_like(y)
    (dx,) = torch.autograd.grad(y, x1, dy)
    ex = _Exact(x, w, b, 1e-5, dy)
    _near(dx, ex.dx, ex.dx_tol)


def test_without_bias_strided_rows_and_offsets():
    """No bias; rows with a pitch, a transposed view, and storage that starts at odd addresses."""
    x, w, _, dy = _inputs(64, 320, torch.float32)
    for view in (x[:, 3:260], x[::2, 1:], x.t(), x.reshape(4, 16, 320)[1:, :, 2:]):
        wv = w.repeat(2)[1 : 1 + view.shape[-1]]
        leaf = view.detach().clone(memory_format=torch.preserve_format).requires_grad_()
        y = layernorm(view, wv, None, 1e-5)
        ex = _Exact(view.reshape(-1, view.shape[-1]), wv, None, 1e-5)
        _near(y.reshape(-1, view.shape[-1]), ex.y, ex.y_tol)
        g = dy.flatten()[: leaf.numel()].reshape(leaf.shape)
        (dx,) = torch.autograd.grad(layernorm(leaf, wv, None, 1e-5), leaf, g)
        ex = _Exact(leaf.detach().reshape(-1, leaf.shape[-1]), wv, None, 1e-5, g.reshape(-1, leaf.shape[-1]))
        _near(dx.reshape(-1, leaf.shape[-1]), ex.dx, ex.dx_tol)
    # 4-byte and 2-byte aligned storage
    for dtype in (torch.float32, torch.bfloat16):
        buf = torch.randn(1 + 8 * 512, device=dev).to(dtype)
        v = buf[1:].view(8, 512)
        ex = _Exact(v, w.repeat(2)[:512], None, 1e-5)
        _near(layernorm(v, w.repeat(2)[:512], None, 1e-5), ex.y, ex.y_tol)


def test_empty_batch_and_constant_rows():
    w, b = torch.randn(48, device=dev), torch.randn(48, device=dev)
    x = torch.empty(0, 48, device=dev, requires_grad=True)
    w1, b1 = w.clone().requires_grad_(), b.clone().requires_grad_()
    y = layernorm(x, w1, b1, 1e-5)
    dx, dw, db = torch.autograd.grad(y, (x, w1, b1), torch.empty(0, 48, device=dev))
    assert y.shape == dx.shape == (0, 48) and not dw.any() and not db.any()
    # a row without spread normalises to the bias alone (xh = 0), whatever its offset
    const = torch.full((3, 48), 7.0, device=dev)
    assert torch.equal(layernorm(const, w, b, 1e-5), b.expand(3, 48))


def test_nonfinite_rows_stay_apart():
    x, w, b, dy = _inputs(9, 640, torch.float32)
    bad = x.clone()
    bad[4, 100] = float("nan")
    bad[7, 3] = float("inf")
    y, good = layernorm(bad, w, b, 1e-5), layernorm(x, w, b, 1e-5)
    for r in range(9):
        if r in (4, 7):
            assert bool(y[r].isnan().all())
        else:
            assert torch.equal(y[r], good[r])


def test_accumulating_into_given_gradients_and_repeatability():
    C = _native.module()
    x, w, b, dy = _inputs(700, 768, torch.float32)
    _, _, mean, rstd = C.add_layernorm_fwd(x, None, w, b, 1e-5, False)
    runs = []
    for _ in range(2):
        dw, db = torch.full((768,), 3.0, device=dev), torch.full((768,), -2.0, device=dev)
        C.layernorm_bwd(dy, x, w, mean, rstd, None, None, dw, db, True)
        runs.append((dw, db))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])
    ex = _Exact(x, w, b, 1e-5, dy)
    _near(runs[0][0], ex.dw + 3, ex.dw_tol + 4 * U * (ex.dw.abs() + 3))
    _near(runs[0][1], ex.db - 2, ex.db_tol + 4 * U * (ex.db.abs() + 2))


def test_other_stream_and_graph_replay():
    x, w, b, dy = _inputs(256, 768, torch.float32)
    want = layernorm(x, w, b, 1e-5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layernorm(x, w, b, 1e-5)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    C = _native.module()
    static = x.clone()
    dw, db = torch.empty(768, device=dev), torch.empty(768, device=dev)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _, y, mean, rstd = C.add_layernorm_fwd(static, None, w, b, 1e-5, False)
        dx = C.layernorm_bwd(dy, static, w, mean, rstd, None, None, dw, db, False)
    for k in (1, 2):
        static.copy_(x * k + k)
        graph.replay()
        ex = _Exact(static, w, b, 1e-5, dy)
        _near(y, ex.y, ex.y_tol)
        _near(dx, ex.dx, ex.dx_tol)
        _near(dw, ex.dw, ex.dw_tol)


def test_second_derivatives_are_refused():
    x, w, b, dy = _inputs(4, 32, torch.float32)
    x.requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(layernorm(x, w, b), x, dy, create_graph=True)


def test_native_refusals():
    C = _native.module()
    x, w, b, dy = _inputs(4, 32, torch.float32)
    cases = [
        lambda: C.add_layernorm_fwd(x[:, ::2], None, w[:16], b[:16], 1e-5, False),  # rows with gaps
        lambda: C.add_layernorm_fwd(x, None, w[:16], b, 1e-5, False),
        lambda: C.add_layernorm_fwd(x, None, w.bfloat16(), b, 1e-5, False),
        lambda: C.add_layernorm_fwd(x, x, w, b, 1e-5, False),  # fp32 delta
        lambda: C.add_layernorm_fwd(x.cpu(), None, w, b, 1e-5, False),
        lambda: C.add_layernorm_fwd(x, None, w.cpu(), b, 1e-5, False),
        lambda: C.layernorm_bwd(dy[:2], x, w, w[:4].clone(), w[:4].clone(), None, None, w.clone(), None, False),
        lambda: C.layernorm_bwd(dy, x, w, w[:3].clone(), w[:4].clone(), None, None, w.clone(), None, False),
    ]
    for call in cases:
        with pytest.raises(RuntimeError, match="layernorm"):
            call()
    with pytest.raises(ValueError, match="is on"):
        layernorm(x, w.cpu(), b)
