"""Global gradient norm and clipping over all parameters of a model in a few launches, with the arguments of
torch.nn.utils.clip_grad_norm_ but `foreach`, which a trainer puts between backward and optimizer.step() (base_trainer.py:226-229 of the
reference steps without it).  FusedAdam(max_grad_norm=...) folds the same clipping into the optimizer's own pass."""
from __future__ import annotations

from typing import Iterable, List, Union

import torch
from torch import Tensor

from ..runtime import ops


def _grads(parameters: Union[Tensor, Iterable[Tensor]]) -> List[Tensor]:
    if isinstance(parameters, Tensor):
        parameters = [parameters]
    return [g for p in parameters if (g := p.grad) is not None]


@torch.no_grad()
def grad_norm(parameters: Union[Tensor, Iterable[Tensor]], norm_type: float = 2.0) -> Tensor:
    """Norm of all gradients together (norm_type 2 or inf) as a 0-dim fp32 tensor; nothing is synchronised.  A parameter that is
    given twice counts once."""
    grads = _grads(parameters)
    return ops.grad_norm(grads, norm_type) if grads else torch.zeros(())


@torch.no_grad()
def clip_grad_norm_(parameters: Union[Tensor, Iterable[Tensor]], max_norm: float, norm_type: float = 2.0,
                    error_if_nonfinite: bool = False) -> Tensor:
    """Multiplies all gradients by min(1, max_norm / (norm + 1e-6)) in place and returns the norm they had before.  bf16 gradients are multiplied
    by that factor rounded to bf16, as torch does it: their norm may end up to 2^-8 above max_norm.  As in torch, a norm
    that is not finite makes them NaN or zero unless error_if_nonfinite asks for an error: then the norm is read back first (the
    host waits for the GPU) and the gradients stay as they are."""
    grads = _grads(parameters)
    if not grads:
        return torch.zeros(())
    if error_if_nonfinite:
        norm = ops.grad_norm(grads, norm_type)
        if not torch.isfinite(norm):
            raise RuntimeError(f"The total norm of order {norm_type} for gradients from `parameters` is non-finite, so it cannot be clipped.")
    return ops.grad_norm(grads, norm_type, float(max_norm))
