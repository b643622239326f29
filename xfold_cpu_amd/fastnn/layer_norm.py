"""LayerNorm module with the reference's constructor and parameters
(``xfold/fastnn/layer_norm.py:14-53``), dispatching on ``config.layer_norm_implementation``
(``layer_norm.py:55-81``); this package implements the ``"hip"`` value. In training mode the module
is :func:`trainable_layer_norm`, which has a backward pass."""

from __future__ import annotations

import numbers
from typing import Optional

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import config as fastnn_config
from . import native_hip as nh
from . import ops


def _rows(t: torch.Tensor, cols: int):
    """(``t``, or a contiguous copy of it, and its stride between rows of ``cols`` elements)."""
    if not t.is_contiguous():
        if t.dim() == 2 and t.shape[1] == cols and t.stride(1) == 1 and t.stride(0) >= cols:
            return t, t.stride(0)
        t = t.contiguous()
    return t, cols


_CODES = {torch.float32: nh.F32, torch.bfloat16: nh.BF16}


def _arg(t: Optional[torch.Tensor]):
    """Address and type of a parameter vector for the library."""
    return (None, nh.F32) if t is None else (t.data_ptr(), _CODES[t.dtype])


def _forward(x, cols, weight, bias, eps, out_dtype, keep):
    x, stride = _rows(x, cols)
    device = x.device
    rows = x.numel() // cols if cols else 0
    y = torch.empty(x.shape, dtype=out_dtype, device=device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=device) if keep else None
    nh.launch(device, "xfh_layer_norm_train", x.data_ptr(), _CODES[x.dtype], stride, rows, cols, *_arg(weight),
              *_arg(bias), eps, y.data_ptr(), _CODES[out_dtype], None if stats is None else stats.data_ptr())
    return x, y, stats, stride


def _backward(ctx, dy):
    # (Runs in a thread of autograd's, where Python is slow: what is known before is in ctx.call.)
    x, weight, stats = ctx.saved_tensors
    need_x, need_w, need_b, *_ = ctx.needs_input_grad
    cols, rows, x_code, x_stride, out_dtype, out_code, bias, size = ctx.call
    if dy.dtype is not out_dtype:
        dy = dy.to(out_dtype)
    dy_stride = cols
    if not dy.is_contiguous():
        dy, dy_stride = _rows(dy, cols)
    dx = dw = db = None
    dx_at = dw_at = db_at = ws_at = None
    dw_code = db_code = nh.F32
    if need_x:
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dx_at = dx.data_ptr()
    if need_w:
        dw = torch.empty_like(weight)
        dw_at, dw_code = dw.data_ptr(), _CODES[dw.dtype]
    if need_b:
        db = torch.empty(bias[0], dtype=bias[1], device=x.device)
        db_at, db_code = db.data_ptr(), _CODES[bias[1]]
    if size and (need_w or need_b):
        ws = torch.empty(size, dtype=torch.uint8, device=x.device)
        ws_at = ws.data_ptr()
    w_at, w_code = _arg(weight)
    nh.launch(x.device, "xfh_layer_norm_backward", dy.data_ptr(), out_code, dy_stride, x.data_ptr(), x_code, x_stride, rows,
              cols, w_at, w_code, stats.data_ptr(), dx_at, dw_at, dw_code, db_at, db_code, ws_at, size)
    return dx, dw, db, None, None, None


_backward_once = once_differentiable(_backward)


class _TrainableLayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, cols, eps, out_dtype):
        w = None if weight is None else weight.contiguous()
        x, y, stats, stride = _forward(x, cols, w, None if bias is None else bias.contiguous(), eps, out_dtype, True)
        rows = stats.shape[0]
        ctx.save_for_backward(x, w, stats)
        ctx.call = (cols, rows, _CODES[x.dtype], stride, out_dtype, _CODES[out_dtype],
                    None if bias is None else (bias.shape, bias.dtype),
                    nh.function("xfh_layer_norm_backward_workspace_size")(rows, cols))
        return y

    @staticmethod
    def backward(ctx, dy):
        # Gradients that are to be differentiated again get the node that refuses it.
        return _backward_once(ctx, dy) if torch.is_grad_enabled() else _backward(ctx, dy)


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
    out_dtype = torch.float32 if torch.is_autocast_enabled("cuda") else x.dtype
    if nh.needs_gradient(x, weight, bias):
        return _TrainableLayerNorm.apply(x, weight, bias, cols, eps, out_dtype)
    weight, bias = (None if t is None else t.contiguous() for t in (weight, bias))
    return _forward(x, cols, weight, bias, eps, out_dtype, False)[1]


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
