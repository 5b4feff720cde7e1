"""Layer normalisation: native sm_100a kernels on CUDA (row statistics, the residual add and
both parameter gradients fused), torch math on CPU.

``layernorm(x, weight, bias, eps)`` normalises the last dimension of ``x``;
``add_layernorm(x, delta, weight, bias, eps)`` first adds the bf16 output of a projection to
the fp32 residual stream and returns the sum as well.  Statistics and sums are fp32; the
parameter gradients are summed in a fixed order.
"""

from __future__ import annotations

import torch

from packbalance_b200.ops import _native
from packbalance_b200.ops.reference import layernorm_reference

_TYPES = (torch.float32, torch.bfloat16)


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x`` as contiguous rows of its last dimension."""
    if x.dim() == 2 and x.is_contiguous():
        return x
    return x.reshape(-1, x.shape[-1]).contiguous()


def _param(w: torch.Tensor | None) -> torch.Tensor | None:
    return w if w is None or (w.dtype == torch.float32 and w.is_contiguous()) else w.float().contiguous()


def _wants_grad(*tensors: torch.Tensor | None) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _check(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, name: str) -> None:
    if x.dim() == 0 or x.shape[-1] == 0:
        raise ValueError(f"{name}: x needs a non-empty last dimension, got shape {tuple(x.shape)}")
    if x.dtype not in _TYPES:
        raise ValueError(f"{name}: x must be fp32 or bf16, got {x.dtype}")
    for what, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != (x.shape[-1],):
            raise ValueError(f"{name}: {what} must have shape ({x.shape[-1]},), got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"{name}: {what} is on {p.device}, x on {x.device}")


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        x2 = _rows(x)
        _, y, mean, rstd = _native.module().add_layernorm_fwd(x2, None, _param(weight), _param(bias), eps, False)
        ctx.save_for_backward(x2, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y.view(x.shape)

    @staticmethod
    def backward(ctx, dy):
        x2, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = _backward(dy.reshape(x2.shape).contiguous(), x2, weight, ctx.bias_dtype, mean, rstd)
        return dx.view(dy.shape), dw, db, None


def _backward(dy2, x2, weight, bias_dtype, mean, rstd, dres=None, dx_bf16=None):
    dw = torch.empty(x2.shape[-1], device=x2.device, dtype=torch.float32)
    db = None if bias_dtype is None else torch.empty_like(dw)
    dx = _native.module().layernorm_bwd(dy2, x2, _param(weight), mean, rstd, dres, dx_bf16, dw, db, False)
    return dx, dw.to(weight.dtype), None if db is None else db.to(bias_dtype)


class _AddLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, delta, weight, bias, eps):
        total, y, mean, rstd = _native.module().add_layernorm_fwd(
            _rows(x), _rows(delta), _param(weight), _param(bias), eps, True)
        ctx.save_for_backward(total, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return total.view(x.shape), y.view(x.shape)

    @staticmethod
    def backward(ctx, dtotal, dy):
        total, weight, mean, rstd = ctx.saved_tensors
        ddelta = torch.empty(total.shape, device=total.device, dtype=torch.bfloat16)
        dx, dw, db = _backward(_rows(dy), total, weight, ctx.bias_dtype, mean, rstd, _rows(dtotal), ddelta)
        return dx.view(dy.shape), ddelta.view(dy.shape), dw, db, None


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
              eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in ``x``'s
    type (fp32 or bf16; any width, any leading shape).  ``weight`` and ``bias`` (optional)
    are vectors of that width; their gradients are sums over all rows in fp32."""
    _check(x, weight, bias, "layernorm")
    if not x.is_cuda:
        return layernorm_reference(x, weight, bias, eps)
    if not _wants_grad(x, weight, bias):  # no autograd node, no saved statistics
        y = _native.module().add_layernorm_fwd(_rows(x), None, _param(weight), _param(bias), eps, False, False)[1]
        return y.view(x.shape)
    return _LayerNorm.apply(x, weight, bias, float(eps))


def add_layernorm(x: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                  eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """``(x + delta, layernorm(x + delta))`` for an fp32 residual stream ``x`` and a bf16
    ``delta`` of the same shape; the sum is fp32, the normalised rows are bf16."""
    _check(x, weight, bias, "add_layernorm")
    if x.dtype != torch.float32 or delta.dtype != torch.bfloat16 or delta.shape != x.shape:
        raise ValueError("add_layernorm: fp32 x and bf16 delta of the same shape, got "
                         f"{x.dtype} {tuple(x.shape)} and {delta.dtype} {tuple(delta.shape)}")
    if delta.device != x.device:
        raise ValueError(f"add_layernorm: delta is on {delta.device}, x on {x.device}")
    if not x.is_cuda:
        total = x + delta.float()
        return total, layernorm_reference(total, weight, bias, eps).to(torch.bfloat16)
    if not _wants_grad(x, delta, weight, bias):
        total, y, _, _ = _native.module().add_layernorm_fwd(_rows(x), _rows(delta), _param(weight), _param(bias), eps,
                                                            True, False)
        return total.view(x.shape), y.view(x.shape)
    return _AddLayerNorm.apply(x, delta, weight, bias, float(eps))
