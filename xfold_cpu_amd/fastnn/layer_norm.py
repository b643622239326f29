"""LayerNorm module with the reference's constructor and parameters
(``xfold/fastnn/layer_norm.py:14-53``), dispatching on ``config.layer_norm_implementation``
(``layer_norm.py:55-81``); this package implements the ``"hip"`` value. In training mode the module
is :func:`trainable_layer_norm`, which has a backward pass."""

from __future__ import annotations

import numbers
from typing import Optional

import torch
import torch.nn as nn

from . import config as fastnn_config
from . import native_hip as nh
from . import ops


def trainable_layer_norm(x: torch.Tensor, normalized_shape, weight: Optional[torch.Tensor] = None,
                         bias: Optional[torch.Tensor] = None, eps: float = 1e-5) -> torch.Tensor:
    """F.layer_norm over the trailing ``normalized_shape``, with gradients of ``x``, ``weight`` and
    ``bias`` (once; the backward pass itself is not differentiable). FP32/BF16 input, weight and bias,
    each in a type of its own; statistics and sums in FP32. As with :class:`LayerNorm` in eval mode the
    output is in the input's type, under autocast in FP32 (``xfold/fastnn/layer_norm.py:56-59``)."""
    if fastnn_config.layer_norm_implementation != fastnn_config.HIP:
        raise ValueError("xfold_cpu_amd implements layer_norm_implementation='hip' only, "
                         f"got {fastnn_config.layer_norm_implementation!r}")
    nh.check_gpu(x, weight, bias)
    if any(t is not None and t.dtype not in (torch.float32, torch.bfloat16) for t in (x, weight, bias)):
        raise ValueError("The 'hip' LayerNorm supports FP32/BF16 tensors.")
    shape = (normalized_shape,) if isinstance(normalized_shape, numbers.Integral) else tuple(normalized_shape)
    if not shape or tuple(x.shape[x.dim() - len(shape):]) != shape:
        raise ValueError(f"LayerNorm: input shape {tuple(x.shape)} does not end with {shape}.")
    if any(t is not None and tuple(t.shape) != shape for t in (weight, bias)):
        raise ValueError(f"LayerNorm: weight and bias must have the shape {shape}.")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError("LayerNorm: eps must be nonnegative.")
    cols = 1
    for s in shape:
        cols *= s
    return nh.autograd().trainable_layer_norm(x, weight, bias, cols, eps, torch.is_autocast_enabled("cuda"))


class LayerNorm(nn.Module):
    def __init__(self, normalized_shape, eps: float = 1e-5, elementwise_affine: bool = True,
                 bias: bool = True, device=None, dtype=None) -> None:
        factory = {"device": device, "dtype": dtype}
        super().__init__()
        if isinstance(normalized_shape, numbers.Integral):
            normalized_shape = (normalized_shape,)
        self.normalized_shape = tuple(normalized_shape)
        self.eps = eps
        self.elementwise_affine = elementwise_affine
        if elementwise_affine:
            self.weight = nn.Parameter(torch.ones(self.normalized_shape, **factory))
            if bias:
                self.bias = nn.Parameter(torch.zeros(self.normalized_shape, **factory))
            else:
                self.register_parameter("bias", None)
        else:
            self.register_parameter("weight", None)
            self.register_parameter("bias", None)

    def forward(self, input: torch.Tensor) -> torch.Tensor:
        if fastnn_config.layer_norm_implementation != fastnn_config.HIP:
            raise ValueError("xfold_cpu_amd implements layer_norm_implementation='hip' only, "
                             f"got {fastnn_config.layer_norm_implementation!r}")
        if self.training:
            return trainable_layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps)
        return ops.layer_norm(input, self.normalized_shape, self.weight, self.bias, self.eps, owner=self)

    def extra_repr(self) -> str:
        return f"{self.normalized_shape}, eps={self.eps}, elementwise_affine={self.elementwise_affine}"
