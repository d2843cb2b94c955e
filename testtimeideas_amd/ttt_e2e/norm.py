"""Layer norm on the HIP kernels, with an exact second derivative.

The blocks of the reference's TTT model normalise with ``nn.LayerNorm``
(cloud_ttt_e2e/ttt_e2e/model.py:9-143), and its meta step differentiates
through the gradient of every block it adapts.  ``layer_norm`` computes the
same values (the row's mean and variance in fp32, two passes over registers);
its backward runs on the kernels and, under ``create_graph=True``, so does the
gradient of that.  A third derivative raises.
"""
from __future__ import annotations

from typing import Optional

import torch
from torch import nn

from .. import _lib

_TYPES = (torch.float16, torch.bfloat16, torch.float32)


def _check_param(name: str, p: Optional[torch.Tensor], x: torch.Tensor) -> None:
    if p is None:
        return
    if p.shape != x.shape[-1:]:
        raise ValueError(f"{name} of shape {tuple(p.shape)} does not match rows of {x.shape[-1]} values")
    if p.dtype != x.dtype and p.dtype != torch.float32:
        raise TypeError(f"{name} is {p.dtype}: expected {x.dtype} or float32")
    if p.device != x.device:
        raise ValueError(f"{name} is on {p.device}, x on {x.device}")


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension
    of x (float16, bfloat16 or float32, any leading shape and strides; up to
    32768 values a row, 16384 in float32).  weight and bias: [D], of x's dtype
    or float32 (the same for both), or None.  Means, variances and the sums of
    the parameters' gradients are fp32; every output is rounded once."""
    if x.device.type != "cuda":
        raise RuntimeError(f"layer_norm runs on a ROCm GPU; got a tensor on device '{x.device}' (there is no CPU path)")
    if x.dtype not in _TYPES:
        raise TypeError(f"unsupported dtype {x.dtype}; expected float16, bfloat16 or float32")
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm needs rows of at least one value, got shape {tuple(x.shape)}")
    _check_param("weight", weight, x)
    _check_param("bias", bias, x)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype} and bias {bias.dtype}: expected one dtype")
    if not eps >= 0:
        raise ValueError(f"eps must be >= 0, got {eps}")
    return _lib.ext().layer_norm(x, weight, bias, float(eps))


class LayerNorm(nn.LayerNorm):
    """``nn.LayerNorm`` over the last dimension (same constructor, parameters
    and state dict) on ``layer_norm``."""

    def __init__(self, normalized_shape, *args, **kwargs):
        super().__init__(normalized_shape, *args, **kwargs)
        if len(self.normalized_shape) != 1:
            raise ValueError(f"normalized_shape {self.normalized_shape}: only the last dimension is normalised")

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"x of shape {tuple(x.shape)} does not end in {tuple(self.normalized_shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)
