"""Native layer normalisation of rows whose mean is far larger than their spread, and of gradients
whose sums are known.

Bounds, with u = 2^-24.  Up to 16384 columns a thread adds at most 16 elements, then 10 levels of
shuffles and warps' sums follow, so a row's sum passes fewer than D = 40 roundings whatever its width;
beyond, 256 threads take the row in turn and D = n / 256 + 16.  The row's mean is therefore off by at
most D u max|x|; the differences d from it are rounded once; their mean takes the first error out
again and leaves D u mean|d|.  The normalised row is off by at most
  r (2 (D + 2) u (|x - m| + mean|x - m| + D u max|x|)) + |xh| c,
with c = (D + 8) u (1 + (D u max|x|)^2 / (var + eps)) for the deviation's own relative error.  A
column's sum passes at most rows / 148 roundings in a thread and 100 more where blocks are joined."""

import pytest
import torch

from packbalance_b200.ops import _native
from packbalance_b200.ops.layernorm import add_layernorm, layernorm

pytestmark = pytest.mark.gpu
dev = "cuda"
U = 2.0**-24
HALF_STEP = {torch.float32: U, torch.bfloat16: 2.0**-8}


def _near(got, want, tol):
    tol = tol + HALF_STEP[got.dtype] * want.abs() * (1 + 2**-6) + 1e-30
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), f"off by {float((off / tol).max()):.3g} bounds"


class _Exact:
    def __init__(self, x, w, b, eps, dy=None, dres=None):
        x, w = x.double(), w.double()
        rows, n = x.shape
        D = 40 if n <= 16384 else n / 256 + 16
        c = x - x.mean(1, keepdim=True)
        var = (c**2).mean(1, keepdim=True)
        r = 1 / torch.sqrt(var + eps)
        xh = c * r
        off = D * U * x.abs().amax(1, keepdim=True)
        e = 2 * (D + 2) * U * r * (c.abs() + c.abs().mean(1, keepdim=True) + off)
        rel = (D + 8) * U * (1 + off**2 * r**2)
        e = e + rel * xh.abs()
        self.y = xh * w + b.double()
        self.y_tol = e * w.abs() + 4 * U * (self.y.abs() + (xh * w).abs())
        if dy is None:
            return
        dy = dy.double()
        g = dy * w
        gm, gx = g.mean(1, keepdim=True), (g * xh).mean(1, keepdim=True)
        self.dx = (g - gm - xh * gx) * r
        mag = g.abs() + g.abs().mean(1, keepdim=True) + xh.abs() * (g * xh).abs().mean(1, keepdim=True)
        drift = e * gx.abs() + (xh.abs() + e) * (g.abs() * e).mean(1, keepdim=True)
        self.dx_tol = (((D + 8) * U + rel) * mag + drift) * r
        if dres is not None:
            self.dx = self.dx + dres.double()
            self.dx_tol = self.dx_tol + 2 * U * (self.dx.abs() + dres.double().abs())
        gr = (rows / 148 + 100) * U
        self.dw, self.db = (dy * xh).sum(0), dy.sum(0)
        self.dw_tol = gr * (dy * xh).abs().sum(0) + (dy.abs() * e).sum(0)
        self.db_tol = gr * dy.abs().sum(0)


def _offset_rows(n, spread, dtype, seed):
    """Rows around offsets of 1e2 to 2e4 that are no whole numbers, the last few without spread."""
    gen = torch.Generator(device=dev).manual_seed(seed)
    off = torch.logspace(2, 4.3, 24, device=dev).unsqueeze(1) * (1 + 0.1 * torch.rand(24, 1, generator=gen, device=dev))
    x = off + spread * torch.randn(24, n, generator=gen, device=dev)
    x[16:] = off[16:]
    x[::2] *= -1
    w, b = 1 + 0.2 * torch.randn(n, generator=gen, device=dev), 0.3 * torch.randn(n, generator=gen, device=dev)
    return x.to(dtype), w, b, torch.randn(24, n, generator=gen, device=dev)


# widths of every thread count, odd ones, and one for the kernels of any width
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("spread", [0.01, 1.0])
@pytest.mark.parametrize("n", [3, 48, 257, 768, 1409, 4096, 8192, 16376, 20001])
def test_rows_far_from_zero(n, spread, dtype):
    x, w, b, dy = _offset_rows(n, spread, dtype, seed=n)
    dy = dy.to(dtype)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    y = layernorm(*leaves, 1e-5)
    dx, dw, db = torch.autograd.grad(y, leaves, dy)
    ex = _Exact(x, w, b, 1e-5, dy)
    for got, want, tol in ((y.detach(), ex.y, ex.y_tol), (dx, ex.dx, ex.dx_tol), (dw, ex.dw, ex.dw_tol),
                           (db, ex.db, ex.db_tol)):
        _near(got, want, tol)


@pytest.mark.parametrize("n", [48, 770, 1409, 4096, 8192, 20001])
def test_sums_far_from_zero(n):
    x, w, b, dsum = _offset_rows(n, 0.05, torch.float32, seed=n + 1)
    delta, dy = (0.01 * torch.randn(24, n, device=dev)).bfloat16(), torch.randn(24, n, device=dev).bfloat16()
    leaves = [t.clone().requires_grad_() for t in (x, delta, w, b)]
    total, y = add_layernorm(*leaves, 1e-5)
    dx, dd, dw, db = torch.autograd.grad((total, y), leaves, (dsum, dy))
    ex = _Exact(total.detach(), w, b, 1e-5, dy, dsum)
    for got, want, tol in ((y.detach(), ex.y, ex.y_tol), (dx, ex.dx, ex.dx_tol), (dw, ex.dw, ex.dw_tol),
                           (db, ex.db, ex.db_tol)):
        _near(got, want, tol)
    assert torch.equal(dd, dx.bfloat16())
TALL = [(9001, 128), (8192, 256), (8192, 768), (4097, 1408), (2500, 4096), (1500, 8192), (400, 16384), (6000, 257),
          (3000, 1409), (700, 20001)]


def _plain_rows(rows, n, dtype):
    gen = torch.Generator(device=dev).manual_seed(n)
    x = torch.randn(rows, n, generator=gen, device=dev) + 0.5
    return x.to(dtype), 1 + 0.2 * torch.randn(n, generator=gen, device=dev), torch.zeros(n, device=dev), gen


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,n", TALL)
def test_column_sums(rows, n, dtype):
    C = _native.module()
    x, w, b, gen = _plain_rows(rows, n, dtype)
    _, y, mean, rstd = C.add_layernorm_fwd(x, None, w, b, 1e-5, False)

    def grads(dy):
        dw, db = torch.full((n,), float("nan"), device=dev), torch.full((n,), float("nan"), device=dev)
        dx = C.layernorm_bwd(dy, x, w, mean, rstd, None, None, dw, db, False)
        return dx, dw, db

    # whole numbers of 4 bits: every partial sum is exact
    dy = torch.randint(-8, 9, (rows, n), generator=gen, device=dev).to(dtype)
    dx, dw, db = grads(dy)
    ex = _Exact(x, w, b, 1e-5, dy)
    assert torch.equal(db.double(), ex.db)
    _near(dw, ex.dw, ex.dw_tol)
    _near(dx, ex.dx, ex.dx_tol)
    # a gradient in one row alone: the sums are that row's terms
    for at in {0, 1, rows // 2 + 3, rows - 148, rows - 7, rows - 2, rows - 1}:
        dy = torch.zeros(rows, n, device=dev, dtype=dtype)
        dy[at] = torch.randn(n, generator=gen, device=dev).to(dtype)
        dx, dw, db = grads(dy)
        one = _Exact(x[at : at + 1], w, b, 1e-5, dy[at : at + 1])
        assert torch.equal(db, dy[at].float())
        _near(dw, one.dw, one.dw_tol)
        _near(dx[at : at + 1], one.dx, one.dx_tol)
        dx[at] = 0
        assert not dx.any()


def test_native_backward_types():
    """A bf16 dy of an fp32 x without a residual gradient takes the kernels of any width; what no
    forward pass makes is refused."""
    C = _native.module()
    x, w, b, gen = _plain_rows(300, 768, torch.float32)
    _, _, mean, rstd = C.add_layernorm_fwd(x, None, w, b, 1e-5, False)
    dy = torch.randn(300, 768, generator=gen, device=dev).bfloat16()
    dw, db, copy = torch.empty(768, device=dev), torch.empty(768, device=dev), torch.empty_like(dy)
    dx = C.layernorm_bwd(dy, x, w, mean, rstd, None, copy, dw, db, False)
    ex = _Exact(x, w, b, 1e-5, dy)
    for got, want, tol in ((dx, ex.dx, ex.dx_tol), (dw, ex.dw, ex.dw_tol), (db, ex.db, ex.db_tol)):
        _near(got, want, tol)
    assert torch.equal(copy, dx.bfloat16())
    half = x.bfloat16()
    for args in ((dy.float(), None, None), (dy, x, None), (dy, None, copy)):
        with pytest.raises(RuntimeError, match="bf16 x"):
            C.layernorm_bwd(args[0], half, w, mean, rstd, args[1], args[2], dw, db, False)
