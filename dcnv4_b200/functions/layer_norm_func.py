"""Autograd functions of the LayerNorm training passes (`ops.layer_norm_train_forward` and its neighbours).

The reference composes these from torch.nn.LayerNorm, the layer-scale product, timm's DropPath and residual additions
(classification/models/flash_intern_image.py:34-56, 414-432).  Each function below is one kernel forward and one
(plus a small reduction) backward; gradients come out in the dtype of their inputs.  Under `create_graph=True`, and for
gradients that are no plain tensors (batched ones), the backward pass is composed of PyTorch operations instead, so second
derivatives and vectorised Jacobians work as with the stock modules.
"""
from __future__ import annotations

import torch
from torch.autograd import Function

from .. import ops


def kernels_apply(*tensors) -> bool:
    """Whether an autograd function over a foreign kernel may take these tensors: plain tensors with memory behind them, not
    subclasses (fake, distributed, masked ones), and nobody who watches or rewrites operations -- a compiler, a tracer, a
    dispatch mode, a torch.func transform, forward-mode AD, batched gradients -- all of whom only the stock ones support."""
    if torch.compiler.is_compiling() or torch.jit.is_tracing() or torch._C._len_torch_dispatch_stack() > 0:
        return False
    if any(t is not None and not (type(t) in (torch.Tensor, torch.nn.Parameter) and torch._C._has_storage(t)) for t in tensors):
        return False
    return getattr(torch.autograd.forward_ad, "_current_level", -1) < 0


def _layer_norm(x, weight, bias, eps, dtype):
    return torch.nn.functional.layer_norm(x.to(dtype), (x.shape[-1],), weight.to(dtype), bias.to(dtype), eps)


def _per_sample(sample_scale, x):
    return sample_scale.view((-1,) + (1,) * (x.dim() - 1)).repeat_interleave(x.shape[0] // sample_scale.numel(), 0)


def _differentiable(fn, inputs, grads):
    """Gradients of fn(*inputs) that can be differentiated again; None where an input needs none."""
    with torch.enable_grad():
        out = fn(*inputs)
        out = out if isinstance(out, tuple) else (out,)
        pairs = [(o, g) for o, g in zip(out, grads) if g is not None and o.requires_grad]
        wanted = [t for t in inputs if t is not None and t.requires_grad]
        if not pairs or not wanted:          # what was asked for does not go through fn
            return [None] * len(inputs)
        got = iter(torch.autograd.grad([o for o, _ in pairs], wanted, [g for _, g in pairs], create_graph=True,
                                       allow_unused=True))
        return [next(got) if t is not None and t.requires_grad else None for t in inputs]


# The `apply` of each function makes its inputs contiguous in front of it, in the graph: one copy where one is needed, which
# both passes read.


class LayerNormFunction(Function):
    """y = act(LN(x)): apply(x, weight, bias, eps, activation="none", out_dtype=None)."""

    @classmethod
    def apply(cls, x, *args):
        return super().apply(x.contiguous(), *args)

    @staticmethod
    def forward(ctx, x, weight, bias, eps, activation="none", out_dtype=None):
        y, mean, rstd = ops.layer_norm_train_forward(x, weight, bias, eps, activation, out_dtype)
        ctx.eps, ctx.activation = eps, activation
        ctx.save_for_backward(x, weight, bias, mean, rstd)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        x, weight, bias, mean, rstd = ctx.saved_tensors
        if torch.is_grad_enabled() or not kernels_apply(grad_y):
            def plain(x_, w_, b_):
                y = _layer_norm(x_, w_, b_, ctx.eps, grad_y.dtype)
                return torch.nn.functional.gelu(y) if ctx.activation == "gelu" else y
            return (*_differentiable(plain, (x, weight, bias), (grad_y,)), None, None, None)
        gx, gw, gb = ops.layer_norm_backward(grad_y.contiguous(), x, mean, rstd, weight, bias, ctx.activation)
        return gx, gw, gb, None, None, None


class LayerNormResidualFunction(Function):
    """out = residual + sample_scale * layer_scale * LN(x): apply(x, residual, weight, bias, eps, layer_scale=None,
    sample_scale=None).  `sample_scale` is a constant (a stochastic-depth mask) and gets no gradient."""

    @classmethod
    def apply(cls, x, residual, *args):
        return super().apply(x.contiguous(), residual.contiguous(), *args)

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, layer_scale=None, sample_scale=None):
        out, mean, rstd = ops.layer_norm_residual_forward(x, residual, weight, bias, eps, layer_scale, sample_scale)
        ctx.eps = eps
        ctx.save_for_backward(x, weight, bias, mean, rstd, layer_scale, sample_scale)
        return out

    @staticmethod
    def backward(ctx, grad_out):
        x, weight, bias, mean, rstd, layer_scale, sample_scale = ctx.saved_tensors
        if torch.is_grad_enabled() or not kernels_apply(grad_out):
            def plain(x_, w_, b_, s_):
                z = _layer_norm(x_, w_, b_, ctx.eps, grad_out.dtype)
                z = z if s_ is None else z * s_.to(z.dtype)
                return z if sample_scale is None else z * _per_sample(sample_scale, z).to(z.dtype)
            gx, gw, gb, gs = _differentiable(plain, (x, weight, bias, layer_scale), (grad_out,))
            return gx, grad_out, gw, gb, None, gs, None
        gx, gw, gb, gs = ops.layer_norm_residual_backward(grad_out.contiguous(), x, mean, rstd, weight, bias, layer_scale,
                                                          sample_scale)
        return gx, grad_out, gw, gb, None, gs, None


class AddLayerNormFunction(Function):
    """(h, y) with h = residual + sample_scale * x and y = LN(h): apply(x, residual, weight, bias, eps,
    sample_scale=None).  `sample_scale` gets no gradient.  Kept for the backward pass: h where it is float32, and x and
    residual where h has 16 bits, since statistics and y are taken of the sum before it is rounded."""

    @classmethod
    def apply(cls, x, residual, *args):
        return super().apply(x.contiguous(), residual.contiguous(), *args)

    @staticmethod
    def forward(ctx, x, residual, weight, bias, eps, sample_scale=None):
        ctx.set_materialize_grads(False)
        h, y, mean, rstd = ops.add_layer_norm_forward(x, residual, weight, bias, eps, sample_scale)
        ctx.eps, ctx.x_dtype, ctx.from_sum = eps, x.dtype, h.dtype == torch.float32
        kept = (h, None) if ctx.from_sum else (x, residual)
        ctx.save_for_backward(*kept, weight, bias, mean, rstd, sample_scale)
        return h, y

    @staticmethod
    def backward(ctx, grad_h, grad_y):
        first, residual, weight, bias, mean, rstd, sample_scale = ctx.saved_tensors
        if grad_h is None and grad_y is None:
            return (None,) * 6
        if torch.is_grad_enabled() or not kernels_apply(grad_h, grad_y):
            if not ctx.from_sum:
                def both(x_, r_, w_, b_):
                    s_ = x_.float() if sample_scale is None else x_.float() * _per_sample(sample_scale, x_)
                    h_ = r_.float() + s_
                    return h_.to(r_.dtype), _layer_norm(h_, w_, b_, ctx.eps, torch.float32).to(r_.dtype)
                return (*_differentiable(both, (first, residual, weight, bias), (grad_h, grad_y)), None, None)
            h = first                   # an output of this node and so part of the graph
            gr = grad_h
            gw = gb = None
            if grad_y is not None:
                def plain(h_, w_, b_):
                    return _layer_norm(h_, w_, b_, ctx.eps, h_.dtype)
                through, gw, gb = _differentiable(plain, (h, weight, bias), (grad_y,))
                gr = through if gr is None else gr + through
            gx = (gr if sample_scale is None else gr * _per_sample(sample_scale, gr).to(gr.dtype)).to(ctx.x_dtype)
            return gx, gr, gw, gb, None, None
        grad_y = torch.zeros(first.shape, dtype=grad_h.dtype, device=first.device) if grad_y is None else grad_y.contiguous()
        grad_h = None if grad_h is None else grad_h.contiguous()
        if ctx.from_sum:
            gr, gx, gw, gb = ops.add_layer_norm_backward(grad_y, grad_h, first, mean, rstd, weight, sample_scale,
                                                         ctx.x_dtype)
        else:
            gr, gx, gw, gb = ops.add_layer_norm_backward(grad_y, grad_h, None, mean, rstd, weight, sample_scale, None,
                                                         first, residual)
        return gx, gr, gw, gb, None, None
