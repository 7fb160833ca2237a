"""Autograd functions of the LayerNorm training passes (`ops.layer_norm_train_forward` and its neighbours).

The reference composes these from torch.nn.LayerNorm, the layer-scale product, timm's DropPath and residual additions
(classification/models/flash_intern_image.py:34-56, 414-432).  Each function below is one kernel forward and one
(plus a small reduction) backward; gradients come out in the dtype of their inputs.
"""
from __future__ import annotations

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import ops


class LayerNormFunction(Function):
    """y = act(LN(x)): apply(x, weight, bias, eps, activation="none", out_dtype=None)."""

    @staticmethod
    def forward(ctx, x, weight, bias, eps, activation="none", out_dtype=None):
        x = x.contiguous()
        y, mean, rstd = ops.layer_norm_train_forward(x, weight, bias, eps, activation, out_dtype)
        ctx.activation = activation
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_y):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        gx, gw, gb = ops.layer_norm_backward(grad_y.contiguous(), x, mean, rstd, weight, bias, ctx.activation)
        return gx, gw, gb, None, None, None


class LayerNormResidualFunction(Function):
    """out = residual + sample_scale * layer_scale * LN(x): apply(x, residual, weight, bias, eps, layer_scale=None,
    sample_scale=None).  `sample_scale` is a constant (a stochastic-depth mask) and gets no gradient."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, layer_scale=None, sample_scale=None):
        x = x.contiguous()
        out, mean, rstd = ops.layer_norm_residual_forward(x, residual.contiguous(), weight, bias, eps, layer_scale,
                                                          sample_scale)
        ctx.save_for_backward(x, weight, bias, mean, rstd, layer_scale, sample_scale)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_out):
        x, weight, bias, mean, rstd, layer_scale, sample_scale = ctx.saved_tensors
        gx, gw, gb, gs = ops.layer_norm_residual_backward(grad_out.contiguous(), x, mean, rstd, weight, bias,
                                                          layer_scale, sample_scale)
        return gx, grad_out, gw, gb, None, gs, None


class AddLayerNormFunction(Function):
    """(h, y) with h = residual + sample_scale * x and y = LN(h): apply(x, residual, weight, bias, eps,
    sample_scale=None).  `sample_scale` gets no gradient."""

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, sample_scale=None):
        ctx.set_materialize_grads(False)
        h, y, mean, rstd = ops.add_layer_norm_forward(x.contiguous(), residual.contiguous(), weight, bias, eps,
                                                      sample_scale)
        ctx.x_dtype = x.dtype
        ctx.save_for_backward(h, weight, mean, rstd, sample_scale)
        return h, y

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_h, grad_y):
        h, weight, mean, rstd, sample_scale = ctx.saved_tensors
        if grad_h is None and grad_y is None:
            return (None,) * 6
        grad_y = torch.zeros_like(h) if grad_y is None else grad_y.contiguous()
        grad_h = None if grad_h is None else grad_h.contiguous()
        gr, gx, gw, gb = ops.add_layer_norm_backward(grad_y, grad_h, h, mean, rstd, weight, sample_scale, ctx.x_dtype)
        return gx, gr, gw, gb, None, None
