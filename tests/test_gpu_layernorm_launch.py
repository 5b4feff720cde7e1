"""Launches of the layer-norm kernels at widths whose row slots just fill 48 KB of shared memory."""

import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

CODE = """
import torch
from packbalance_b200.ops import _native
C = _native.module()
n, dy_type, res = {n}, torch.{dy}, {res}
x, w, b = torch.randn(2000, n, device="cuda"), torch.randn(n, device="cuda"), torch.randn(n, device="cuda")
dy = torch.randn(2000, n, device="cuda").to(dy_type)
dres = torch.randn(2000, n, device="cuda") if res else None
_, y, mean, rstd = C.add_layernorm_fwd(x, None, w, b, 1e-5, False)
dw, db = torch.empty(n, device="cuda"), torch.empty(n, device="cuda")
dx = C.layernorm_bwd(dy, x, w, mean, rstd, dres, None, dw, db, False)
xd = x.double().requires_grad_()
yd = torch.nn.functional.layer_norm(xd, (n,), w.double(), b.double(), 1e-5)
(want,) = torch.autograd.grad(yd, xd, dy.double())
want = want + (0 if dres is None else dres.double())
assert float((dx.double() - want).abs().max()) < 1e-4, float((dx.double() - want).abs().max())
assert float((db.double() - dy.double().sum(0)).abs().max()) < 1e-2
"""


# 48 KB of dynamic shared memory need no opt-in by themselves, with the kernel's static arrays they do;
# each in a process of its own, since the opt-in of one width serves the next
@pytest.mark.parametrize("n,dy,res", [(1532, "float32", False), (3064, "float32", False), (3068, "float32", False),
                                      (2044, "float32", True), (4088, "float32", True), (4092, "float32", True),
                                      (2456, "bfloat16", True)])
def test_width_at_the_shared_memory_border(n, dy, res):
    run = subprocess.run([sys.executable, "-c", CODE.format(n=n, dy=dy, res=res)], capture_output=True, text=True,
                         timeout=300)
    assert run.returncode == 0, run.stderr[-2000:]
