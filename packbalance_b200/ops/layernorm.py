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


def _check(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None, name: str) -> None:
    if x.dtype not in _TYPES:
        raise ValueError(f"{name}: x must be fp32 or bf16, got {x.dtype}")
    shape = x.shape[-1:]
    if len(shape) == 0 or shape[0] == 0:
        raise ValueError(f"{name}: x needs a non-empty last dimension, got shape {tuple(x.shape)}")
    for what, p in (("weight", weight), ("bias", bias)):
        if p is None:
            continue
        if p.shape != shape:
            raise ValueError(f"{name}: {what} must have shape ({shape[0]},), got {tuple(p.shape)}")
        if p.device != x.device:
            raise ValueError(f"{name}: {what} is on {p.device}, x on {x.device}")


def layernorm(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
              eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, in ``x``'s
    type (fp32 or bf16; any width, any leading shape).  ``weight`` and ``bias`` (optional)
    are vectors of that width; their gradients are sums over all rows in fp32.  On CUDA there
    are first derivatives by a backward pass only: forward mode and ``create_graph`` are errors."""
    _check(x, weight, bias, "layernorm")
    if not x.is_cuda:
        return layernorm_reference(x, weight, bias, eps)
    return _native.module().layernorm(x, weight, bias, eps)


def add_layernorm(x: torch.Tensor, delta: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                  eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """``(x + delta, layernorm(x + delta))`` for an fp32 residual stream ``x`` and a bf16
    ``delta`` of the same shape; the sum is fp32, the normalised rows are bf16.  The
    backward pass reads the sum, so change that in place only where none follows."""
    _check(x, weight, bias, "add_layernorm")
    if x.dtype != torch.float32 or delta.dtype != torch.bfloat16 or delta.shape != x.shape:
        raise ValueError("add_layernorm: fp32 x and bf16 delta of the same shape, got "
                         f"{x.dtype} {tuple(x.shape)} and {delta.dtype} {tuple(delta.shape)}")
    if delta.device != x.device:
        raise ValueError(f"add_layernorm: delta is on {delta.device}, x on {x.device}")
    if not x.is_cuda:
        total = x + delta.float()
        return total, layernorm_reference(total, weight, bias, eps).to(torch.bfloat16)
    total, y = _native.module().add_layernorm(x, delta, weight, bias, eps)
    return total, y
