"""Muon: momentum whose update of each weight matrix is orthogonalised before it is applied.

For a weight W (out, in) with gradient G, momentum mu, learning rate lr and decay wd:
    M <- mu M + (1 - mu) G;   U = mu M + (1 - mu) G  (Nesterov)  or  M
    W <- (1 - lr wd) W - lr s NS(U)
where NS is the Newton-Schulz iteration of `ops.newton_schulz` (singular values towards 1) and s the size adjustment:
"match_rms_adamw" s = 0.2 sqrt(max(out, in)), so that learning rates tuned for AdamW carry over, or "original"
s = sqrt(max(1, out / in)).  Convolution weights are matrices (out, in * kh * kw).  Matrices of one shape are
orthogonalised as one stack: FlashInternImage-L's third stage has 22 of each.

M is kept in float32 whatever the parameter's type: a step adds (1 - mu) of a gradient, which 16 bits would round away once M
is near its limit (bf16 at mu 0.95: 4 % short of it).

Vectors (norms, biases, layer scales) have no singular values to speak of: give them to another optimiser.
`split_parameters` makes the two lists.  The reference's trainers use AdamW for everything (classification/optimizer.py).
"""
from __future__ import annotations

import math
from typing import Iterable, List, Tuple

import torch

from . import ops

_STACK_ELEMENTS = 2 ** 28     # of one orthogonalisation call: 3 GB of workspace


def split_parameters(model: torch.nn.Module) -> Tuple[List[torch.nn.Parameter], List[torch.nn.Parameter]]:
    """(matrices, others): the weights of Linear and of ordinary (not depth-wise) convolution layers, except a classifier
    `head` and what Muon has no room for, and everything else, each parameter once."""
    matrices, seen = [], set()
    for name, m in model.named_modules():
        linear = isinstance(m, torch.nn.Linear) and name.split(".")[-1] != "head"
        conv = isinstance(m, torch.nn.Conv2d) and m.groups == 1
        if ((linear or conv) and m.weight.requires_grad and id(m.weight) not in seen
                and max(_matrix(m.weight)) <= ops.NEWTON_SCHULZ_MAX_SIDE):
            seen.add(id(m.weight))
            matrices.append(m.weight)
    return matrices, [p for p in model.parameters() if p.requires_grad and id(p) not in seen]


def _matrix(p: torch.Tensor) -> Tuple[int, int]:
    """Rows and columns of a weight as a matrix: the outputs, and all inputs of one."""
    return p.shape[0], p.numel() // max(p.shape[0], 1)


class Muon(torch.optim.Optimizer):
    """Muon over weight matrices (parameters of two or more dimensions, CUDA, float32 / float16 / bfloat16); see the
    module's text."""

    def __init__(self, params: Iterable, lr: float = 1e-3, weight_decay: float = 0.1, momentum: float = 0.95,
                 nesterov: bool = True, ns_coefficients=ops.NEWTON_SCHULZ_COEFFICIENTS, eps: float = 1e-7,
                 ns_steps: int = 5, adjust_lr: str = "match_rms_adamw"):
        defaults = dict(lr=lr, weight_decay=weight_decay, momentum=momentum, nesterov=nesterov,
                        ns_coefficients=tuple(ns_coefficients), eps=eps, ns_steps=ns_steps, adjust_lr=adjust_lr)
        self._check(dict(defaults, params=[]))
        super().__init__(params, defaults)

    @staticmethod
    def _check(group):
        """What the constructor and `add_param_group` refuse: a group's options and its parameters."""
        if group["lr"] < 0 or group["weight_decay"] < 0 or not 0 <= group["momentum"] < 1:
            raise ValueError("lr and weight_decay must not be negative, momentum must lie in [0, 1)")
        if not 1 <= group["ns_steps"] <= ops.NEWTON_SCHULZ_MAX_STEPS:
            raise ValueError(f"ns_steps must lie between 1 and {ops.NEWTON_SCHULZ_MAX_STEPS}")
        if group["adjust_lr"] not in ("match_rms_adamw", "original"):
            raise ValueError("adjust_lr must be 'match_rms_adamw' or 'original'")
        if len(tuple(group["ns_coefficients"])) != 3:
            raise ValueError("ns_coefficients are three numbers (a, b, c)")
        for p in group["params"]:
            if p.dim() < 2:
                raise ValueError("Muon is for weight matrices: give vectors to another optimiser (split_parameters)")
            if p.dtype not in (torch.float32, torch.float16, torch.bfloat16):
                raise ValueError(f"Muon takes float32, float16 and bfloat16 parameters, got {p.dtype}")
            if max(_matrix(p)) > ops.NEWTON_SCHULZ_MAX_SIDE:
                raise ValueError(f"a weight of {tuple(p.shape)} has a side above {ops.NEWTON_SCHULZ_MAX_SIDE}: give it to another "
                                 "optimiser")

    @torch._disable_dynamo
    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        try:
            self._check(self.param_groups[-1])
        except ValueError:
            self.param_groups.pop()
            raise

    def load_state_dict(self, state_dict):
        """As every optimiser's, but the momentum stays in float32: the base class casts state to the parameter's type."""
        super().load_state_dict(state_dict)
        params = [p for g in self.param_groups for p in g["params"]]
        saved = [i for g in state_dict["param_groups"] for i in g["params"]]
        hooked = bool(self._optimizer_load_state_dict_pre_hooks)         # these may have put another dict in its place
        for i, p in zip(saved, params):
            buffer = self.state.get(p, {}).get("momentum_buffer")
            if buffer is not None and buffer.dtype != torch.float32:
                source = buffer if hooked else state_dict["state"][i]["momentum_buffer"]
                self.state[p]["momentum_buffer"] = source.to(device=p.device, dtype=torch.float32)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:                # refusals come before anything has been updated
            for p in group["params"]:
                if p.grad is not None and p.grad.is_sparse:
                    raise RuntimeError("Muon does not take sparse gradients")
                if p.grad is not None and not p.is_cuda:
                    raise RuntimeError("Muon: parameter must be a CUDA tensor")
        for group in self.param_groups:
            stacks = {}
            for p in group["params"]:
                if p.grad is not None:
                    stacks.setdefault((*_matrix(p), p.dtype, p.device), []).append(p)
            for (rows, cols, _, _), params in stacks.items():
                if rows * cols == 0:
                    continue
                most = max(1, _STACK_ELEMENTS // (rows * cols))
                for i in range(0, len(params), most):
                    self._update(group, params[i:i + most], rows, cols)
        return loss

    def _update(self, group, params, rows, cols):
        mu, lr = group["momentum"], group["lr"]
        buffers = []
        for p in params:
            state = self.state[p]
            if "momentum_buffer" not in state:
                state["momentum_buffer"] = torch.zeros_like(p.grad, dtype=torch.float32, memory_format=torch.preserve_format)
            buffers.append(state["momentum_buffer"])
        grads = [p.grad.float() for p in params]
        torch._foreach_lerp_(buffers, grads, 1 - mu)
        update = torch._foreach_lerp(grads, buffers, mu) if group["nesterov"] else buffers
        # one stack of matrices; reshape follows the parameter's dimensions whatever its memory order (channels_last)
        stack = torch.stack([u.reshape(rows, cols) for u in update])
        ortho = ops.newton_schulz(stack, group["ns_steps"], group["ns_coefficients"], group["eps"])
        scale = 0.2 * math.sqrt(max(rows, cols)) if group["adjust_lr"] == "match_rms_adamw" else math.sqrt(max(1.0, rows / cols))
        if group["weight_decay"]:
            torch._foreach_mul_(params, 1 - lr * group["weight_decay"])
        torch._foreach_add_(params, [o.view(p.shape).to(p.dtype) for o, p in zip(ortho.unbind(0), params)],
                            alpha=-lr * scale)
