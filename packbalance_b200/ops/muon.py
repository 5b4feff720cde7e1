"""Newton-Schulz orthogonalisation and the Muon update: native sm_100a kernels on CUDA (the
products of all matrices of a step in three grouped tcgen05 launches), torch math on CPU.

``orthogonalize(x)`` pulls every singular value of a matrix towards 1 with a fixed number of
odd polynomial steps.  ``muon_update_`` applies one Muon step to lists of matrices in place.
The CUDA iteration keeps its operands in fp16 at fixed scales and accumulates in fp32; before
the result is rounded to the output type it is within 4e-3 of the 64-bit iteration in the
Frobenius norm (within 5.5e-3 for 33 to 63 rows or columns; up to 32 run in fp32 throughout).
It takes up to 2 GB of workspace, or what the largest matrix needs (6 bytes per element and 4 per
element of its smaller square); longer lists go through in parts.
"""

from __future__ import annotations

import bisect
from collections.abc import Sequence

import torch

from packbalance_b200.ops import _native
from packbalance_b200.ops.reference import newton_schulz_reference

# Slope 3.4 at zero.  Five steps bring singular values from 1.5e-3 of the Frobenius norm up to between
# 0.68 and 1.21, and multiply far smaller ones by 485.
COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS = 5
EPS = 1e-7


def _check_iteration(steps: int, coefficients: Sequence[float], name: str) -> tuple[float, float, float]:
    if not 1 <= int(steps) <= 100:
        raise ValueError(f"{name}: steps must be 1 to 100, got {steps}")
    if len(coefficients) != 3:
        raise ValueError(f"{name}: three coefficients, got {len(coefficients)}")
    return tuple(float(c) for c in coefficients)


def _check_memory(params, grads, momenta, shadows) -> None:
    """What the native update checks of its arguments' memory: shadows of the right kind, nothing
    that is written listed twice, and no gradient in it."""
    for k, (w, p) in enumerate(zip(shadows, params)):
        if w.dtype != torch.bfloat16 or w.device != p.device or w.numel() != p.numel() or not w.is_contiguous():
            raise ValueError(f"muon_update_: shadow {k} must be contiguous bf16 of its parameter's size")

    def spans(tensors):
        return [(t.data_ptr(), t.data_ptr() + t.numel() * t.element_size()) for t in tensors if t.numel()]

    written = sorted(spans([*params, *momenta, *shadows]))
    for (_, end), (start, _) in zip(written, written[1:]):
        if end > start:
            raise ValueError("muon_update_: parameters, momenta and shadows must not overlap or be listed twice")
    for start, end in spans(grads):
        # the written spans are disjoint: the one that starts last before ``end`` also ends last
        k = bisect.bisect_left(written, (end,)) - 1
        if k >= 0 and written[k][1] > start:
            raise ValueError("muon_update_: gradients must not overlap parameters, momenta or shadows")


@torch.no_grad()
def orthogonalize(x: torch.Tensor, steps: int = STEPS, coefficients: Sequence[float] = COEFFICIENTS,
                  eps: float = EPS) -> torch.Tensor:
    """Newton-Schulz iterate of every matrix ``x[..., m, n]`` (fp32 or bf16), in bf16.

    ``X = x / (|x|_F + eps)``, then ``steps`` times ``X <- a X + (b A + c A A) X`` with
    ``A = X X^T`` and ``coefficients = (a, b, c)``.  On CUDA no element of ``A`` or of ``a I +
    b A + c A A`` may reach 64, so rows (or columns, on the shorter side) of an iterate stay below
    a norm of 8: beyond, the fp16 operands overflow to infinity.  (The default coefficients keep
    singular values below 1.21 and the polynomial below 3.5.)  Zero matrices stay zero.  The
    stated accuracy holds for ``|x|_F`` from 1e-6 ``eps`` up.  Not differentiable."""
    if x.dim() < 2:
        raise ValueError(f"orthogonalize: x needs at least two dimensions, got shape {tuple(x.shape)}")
    if x.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"orthogonalize: x must be fp32 or bf16, got {x.dtype}")
    coefficients = _check_iteration(steps, coefficients, "orthogonalize")
    if not x.is_cuda:
        return newton_schulz_reference(x.float(), int(steps), coefficients, eps).to(torch.bfloat16).contiguous()
    x3 = x.reshape(-1, *x.shape[-2:]) if x.numel() else x.new_empty(0, 1, 1)
    return _native.module().ns_orthogonalize(x3.contiguous(), int(steps), list(coefficients), float(eps)).view(x.shape)


@torch.no_grad()
def muon_update_(
    params: Sequence[torch.Tensor],
    grads: Sequence[torch.Tensor],
    momenta: Sequence[torch.Tensor],
    *,
    lr: float,
    momentum: float = 0.95,
    nesterov: bool = True,
    weight_decay: float = 0.1,
    steps: int = STEPS,
    coefficients: Sequence[float] = COEFFICIENTS,
    eps: float = EPS,
    shadows: Sequence[torch.Tensor] | None = None,
    grad_norm: torch.Tensor | None = None,
    max_norm: float = 0.0,
    hparams: torch.Tensor | None = None,
) -> None:
    """One Muon step, in place, on contiguous fp32 tensors ``[..., rows, cols]`` (leading
    dimensions count matrices)::

        m += (1 - momentum) (s g - m)
        u  = s g + momentum (m - s g)  if nesterov else  m
        p  = p (1 - lr weight_decay) - lr 0.2 sqrt(max(rows, cols)) orthogonalize(u)

    The factor 0.2 sqrt(max(rows, cols)) gives the update the root mean square of an AdamW
    step, so one learning rate and weight decay serve both optimizers.  ``shadows``: bf16
    copies of the parameters, refreshed in the same pass.  ``grad_norm`` (fp32 device
    scalar) clips, ``s = min(1, max_norm / (grad_norm + 1e-6))`` when ``max_norm > 0``, and
    leaves everything as it was when it is not finite.  ``hparams`` (CUDA, fp32): the
    learning rate is read from its first element on the device, for captured CUDA graphs."""
    n = len(params)
    if len(grads) != n or len(momenta) != n or (shadows is not None and len(shadows) != n):
        raise ValueError(f"muon_update_: {n} params, {len(grads)} grads, {len(momenta)} momenta"
                         + ("" if shadows is None else f", {len(shadows)} shadows"))
    coefficients = _check_iteration(steps, coefficients, "muon_update_")
    for k, (p, g, m) in enumerate(zip(params, grads, momenta)):
        for t in (p, g, m):
            if t.dim() < 2 or t.shape != p.shape or t.dtype != torch.float32 or t.device != params[0].device:
                raise ValueError(f"muon_update_: entry {k} must be fp32 [..., rows, cols] tensors of one shape on "
                                 f"one device, got {t.dtype} {tuple(t.shape)} on {t.device}")
        if not (p.is_contiguous() and m.is_contiguous()):
            raise ValueError(f"muon_update_: parameter and momentum {k} must be contiguous (updated in place)")
    if n == 0:
        return
    if params[0].is_cuda:
        _native.module().muon_update(
            list(params), [g.contiguous() for g in grads], list(momenta), list(shadows or ()), float(lr),
            float(momentum), bool(nesterov), float(weight_decay), int(steps), list(coefficients), float(eps),
            grad_norm, float(max_norm), hparams)
        torch.autograd.graph.increment_version([*params, *momenta, *(shadows or ())])
        return
    grads = [g.contiguous() for g in grads]
    _check_memory(params, grads, momenta, shadows or ())
    if hparams is not None:
        lr = float(hparams[0])
    scale = 1.0
    if grad_norm is not None:
        if not torch.isfinite(grad_norm):
            return
        if max_norm > 0:
            scale = min(1.0, max_norm / (float(grad_norm) + 1e-6))
    for k, (p, g, m) in enumerate(zip(params, grads, momenta)):
        g = g * scale
        m.lerp_(g, 1.0 - momentum)
        u = g.lerp(m, momentum) if nesterov else m
        o = newton_schulz_reference(u, int(steps), coefficients, eps)
        p.mul_(1.0 - lr * weight_decay).sub_(o, alpha=lr * 0.2 * max(p.shape[-2:]) ** 0.5)
        if shadows is not None:
            shadows[k].copy_(p)
