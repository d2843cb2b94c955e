"""Softmax cross entropy of a linear head on the HIP kernels, without keeping
the logits, with an exact second derivative.

The reference's meta step takes the masked next-token loss of the model's
logits (cloud_ttt_e2e/ttt_e2e/meta.py:140-222) and differentiates through its
gradient at every inner step.  ``linear_cross_entropy`` is the head's product
and that loss in one: [N, V] logits exist only as tiles on the chip (and, in
the backward passes, as bounded pieces of their gradient), so memory does not
grow with N times V.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib

_TYPES = (torch.float16, torch.bfloat16, torch.float32)
_REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}


def linear_cross_entropy(hidden: torch.Tensor, weight: torch.Tensor, targets: torch.Tensor,
                         mask: Optional[torch.Tensor] = None, *, reduction: str = "mean",
                         ignore_index: int = -100) -> torch.Tensor:
    """Cross entropy of ``hidden @ weight.T`` ([..., D] and [V, D], one dtype of
    float16, bfloat16 or float32) against int64 ``targets`` of hidden's leading
    shape, as float32.

    mask: a weight for each row (any real or bool dtype; a constant: it gets no
    gradient).  reduction "none": weighted losses of targets' shape; "sum":
    their sum; "mean": the sum over ``max(sum of weights, 1)``, so a batch
    whose every row is masked has loss 0.  Rows whose target is ignore_index
    have weight 0.  Rows of weight 0 have loss and gradient 0 and add nothing
    to weight's gradient, whatever they hold.  Any other target outside
    [0, V) makes the loss and its gradients NaN; an infinity in a float32
    operand may too.

    Differentiable twice in hidden and weight (``create_graph=True``) and in
    the incoming gradient; a third derivative raises."""
    if hidden.device.type != "cuda":
        raise RuntimeError("linear_cross_entropy runs on a ROCm GPU; got a tensor on device "
                           f"'{hidden.device}' (there is no CPU path)")
    if hidden.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {hidden.dtype}; expected float16, bfloat16 or float32")
    if hidden.dim() < 1 or weight.dim() != 2 or weight.shape[1] != hidden.shape[-1] or 0 in weight.shape:
        raise ValueError(f"weight of shape {tuple(weight.shape)} does not match hidden {tuple(hidden.shape)}: "
                         "expected [V, D] and [..., D]")
    if weight.dtype != hidden.dtype or weight.device != hidden.device:
        raise ValueError("hidden and weight must share dtype and device")
    if targets.dtype != torch.int64:
        raise TypeError(f"targets are {targets.dtype}: expected int64")
    if targets.shape != hidden.shape[:-1] or targets.device != hidden.device:
        raise ValueError(f"targets of shape {tuple(targets.shape)} on {targets.device} do not match hidden "
                         f"{tuple(hidden.shape)} on {hidden.device}")
    if reduction not in _REDUCTIONS:
        raise ValueError(f"reduction {reduction!r}: expected 'none', 'sum' or 'mean'")
    if mask is not None:
        if mask.shape != targets.shape or mask.device != targets.device:
            raise ValueError(f"mask of shape {tuple(mask.shape)} on {mask.device} does not match targets "
                             f"{tuple(targets.shape)} on {targets.device}")
        if mask.dtype.is_complex:
            raise TypeError(f"mask is {mask.dtype}: expected a real or bool dtype")
        mask = mask.detach().to(torch.float32).contiguous()
    return _lib.ext().linear_cross_entropy(hidden, weight, targets.contiguous(), mask, _REDUCTIONS[reduction],
                                           int(ignore_index))
