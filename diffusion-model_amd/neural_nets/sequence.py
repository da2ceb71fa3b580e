"""Layers of a conditioning sequence's encoder (the tokens that ConditionalModule attends to): layer norm over the channels of each
token, as autograd functions and modules on the HIP kernels.  They take tokens as rows, [..., C], in bf16, fp16 or fp32; parameters
are fp32, as everywhere in this package.  The reference has no such encoder; its ConditionalModule takes the sequence from
outside (constituent_blocks.py:402-437 there)."""
from __future__ import annotations

from typing import Optional

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from ..runtime import ops


def _need_gpu(what: str, *tensors) -> None:
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"{what} runs on the HIP kernels only: tensors must live on an MI355X (cuda) device")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")


def _rows(t: Tensor, c: int) -> Tensor:
    """t as [rows, c] with contiguous rows that do not overlap (an expanded or transposed tensor is copied)"""
    r = t.reshape(-1, c)
    if r.stride(1) != 1 or (r.shape[0] > 1 and r.stride(0) < c):
        r = r.contiguous()
    return r if r.stride(1) == 1 else r.as_strided(r.shape, (1, 1))         # (c = 1: torch leaves such a stride as it was)


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float):
        rows = _rows(x, x.shape[-1])
        y, stats = ops.layer_norm_forward(rows, weight, bias, eps, want_stats=any(ctx.needs_input_grad))
        ctx.save_for_backward(rows, weight, stats)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Tensor):
        rows, weight, stats = ctx.saved_tensors
        nx, nw, nb, _ = ctx.needs_input_grad
        dx, dw, db = ops.layer_norm_backward(rows, _rows(dy, rows.shape[1]), weight, stats, want_dx=nx, want_dw=nw, want_db=nb)
        return dx.view(dy.shape) if nx else None, dw, db, None


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis (1 to 8192 elements, var over n), statistics in fp32, the
    result in x's type.  weight, bias: fp32 [C] or None.  Differentiable once in x, weight and bias."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x of shape {tuple(x.shape)} has no last axis to normalise")
    _need_gpu("layer_norm", x, weight, bias)
    return _LayerNormFn.apply(x, weight, bias, float(eps))


class LayerNorm(nn.Module):
    """nn.LayerNorm over the last axis (same constructor arguments and state_dict keys) on the HIP kernels"""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None):
        super().__init__()
        self.normalized_shape, self.eps = (int(normalized_shape),), float(eps)
        c = self.normalized_shape[0]
        self.weight = nn.Parameter(torch.ones(c, device=device)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(c, device=device)) if elementwise_affine and bias else None

    def forward(self, x: Tensor) -> Tensor:
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"LayerNorm({self.normalized_shape[0]}): last axis of {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
