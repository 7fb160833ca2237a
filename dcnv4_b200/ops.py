"""Tensor-level entry points over the C ABI (the role of the reference's `DCNv4.ext` module,
DCNv4_op/src/vision.cpp:14-21): validate torch tensors the way the reference host wrappers
do (DCNv4_op/src/cuda/dcnv4_cuda.cu:26-60, DCNv4_op/src/cuda/flash_deform_attn_cuda.cu:26-58),
allocate outputs with torch (device memory and streams are torch's job here, nothing else),
and call the library on the current CUDA stream.
"""
from __future__ import annotations

import os
from typing import List, Optional, Tuple

import torch

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _code(t: torch.Tensor) -> int:
    try:
        return _DTYPES[t.dtype]
    except KeyError:
        raise RuntimeError(f"dcnv4_b200 supports float32/float16/bfloat16 tensors, got {t.dtype}") from None


def _check_tensor(t: torch.Tensor, name: str) -> None:
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor")
    if not t.is_contiguous():
        raise RuntimeError(f"{name} tensor has to be contiguous")


# Handle of a device's current stream without building a Stream object (2 us of a call's 15); the public route otherwise.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def _stream(t: torch.Tensor) -> int:
    if _raw_stream is not None:
        return _raw_stream(t.get_device())
    return torch.cuda.current_stream(t.device).cuda_stream


def _on_device(t: torch.Tensor, fn, *args) -> int:
    """fn(*args) with the tensor's device current (entered only where it is another one)."""
    if t.get_device() == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(t.device):
        return fn(*args)


def needs_grad(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd would record an operation on these inputs; the kernels without a backward pass stay away then.
    Every input counts, a bias or a residual that learns beside frozen weights too."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _check_step(batch: int, im2col_step: int) -> None:
    step = min(batch, int(im2col_step))
    if step <= 0 or batch % step != 0:
        raise RuntimeError(f"batch({batch}) must divide im2col_step({step})")


def dcnv4_forward(value, p_offset, kernel_h, kernel_w, stride_h, stride_w, pad_h, pad_w,
                  dilation_h, dilation_w, group, group_channels, offset_scale, im2col_step,
                  remove_center, d_stride=None, block_thread=None, softmax=False) -> torch.Tensor:
    """Positional signature of the reference's `ext.dcnv4_forward` (DCNv4_op/src/dcnv4.h:64-83).
    `im2col_step` is validated like the reference does and otherwise unused (the whole batch
    is one launch); `d_stride` / `block_thread` are accepted and ignored."""
    _check_tensor(value, "input")
    _check_tensor(p_offset, "offset")
    if value.dim() != 4 or p_offset.dim() != 4:
        raise RuntimeError("input and offset_mask must be (N,H,W,C) and (N,Ho,Wo,P) tensors")
    if p_offset.dtype != value.dtype:
        raise RuntimeError("input and offset_mask must have the same dtype")
    N, H, W, C = value.shape
    if C != group * group_channels:
        raise RuntimeError(
            f"Input channels and group times group channels wont match: ({C} vs {group * group_channels}).")
    _check_step(N, im2col_step)
    L = _lib.lib()
    Ho = L.dcnv4b200_out_size(H, pad_h, dilation_h, kernel_h, stride_h)
    Wo = L.dcnv4b200_out_size(W, pad_w, dilation_w, kernel_w, stride_w)
    if tuple(p_offset.shape[:3]) != (N, Ho, Wo):
        raise RuntimeError(f"offset_mask must be (N,{Ho},{Wo},P), got {tuple(p_offset.shape)}")
    out = torch.empty((N, Ho, Wo, C), dtype=value.dtype, device=value.device)
    with torch.cuda.device(value.device):
        rc = L.dcnv4b200_fwd(value.data_ptr(), p_offset.data_ptr(), out.data_ptr(), _code(value),
                             N, H, W, group, group_channels, kernel_h, kernel_w, stride_h, stride_w,
                             pad_h, pad_w, dilation_h, dilation_w, float(offset_scale),
                             int(remove_center), p_offset.shape[3], int(bool(softmax)), _stream(value))
    _lib.check(rc, "dcnv4_forward")
    return out


def dcnv4_backward(value, p_offset, kernel_h, kernel_w, stride_h, stride_w, pad_h, pad_w,
                   dilation_h, dilation_w, group, group_channels, offset_scale, im2col_step,
                   grad_output, remove_center, d_stride=None, block_thread=None,
                   softmax=False) -> List[torch.Tensor]:
    """Positional signature of `ext.dcnv4_backward` (DCNv4_op/src/dcnv4.h:85-107).  Returns
    [grad_input, grad_offset_mask] in the dtype of `value` (bf16 included; the reference
    raises a type error for bf16, DCNv4_op/src/cuda/dcnv4_cuda.cu:133-139,161)."""
    _check_tensor(value, "input")
    _check_tensor(p_offset, "offset")
    _check_tensor(grad_output, "grad_output")
    if p_offset.dtype != value.dtype or grad_output.dtype != value.dtype:
        raise RuntimeError("input, offset_mask and grad_output must have the same dtype")
    N, H, W, C = value.shape
    if C != group * group_channels:
        raise RuntimeError(
            f"Input channels and group times group channels wont match: ({C} vs {group * group_channels}).")
    _check_step(N, im2col_step)
    L = _lib.lib()
    Ho = L.dcnv4b200_out_size(H, pad_h, dilation_h, kernel_h, stride_h)
    Wo = L.dcnv4b200_out_size(W, pad_w, dilation_w, kernel_w, stride_w)
    if grad_output.numel() != N * Ho * Wo * C or tuple(p_offset.shape[:3]) != (N, Ho, Wo):
        raise RuntimeError("grad_output / offset_mask shape does not match the output size")
    code = _code(value)
    grad_input = torch.empty_like(value)
    grad_offset = torch.empty_like(p_offset)
    ws_bytes = L.dcnv4b200_bwd_workspace_bytes(code, N, H, W, group, group_channels)
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=value.device) if ws_bytes else None
    with torch.cuda.device(value.device):
        rc = L.dcnv4b200_bwd(value.data_ptr(), p_offset.data_ptr(), grad_output.data_ptr(),
                             grad_input.data_ptr(), grad_offset.data_ptr(),
                             ws.data_ptr() if ws is not None else None, ws_bytes, code,
                             N, H, W, group, group_channels, kernel_h, kernel_w, stride_h, stride_w,
                             pad_h, pad_w, dilation_h, dilation_w, float(offset_scale),
                             int(remove_center), p_offset.shape[3], int(bool(softmax)), _stream(value))
    _lib.check(rc, "dcnv4_backward")
    return [grad_input, grad_offset]


def _check_fda(value, spatial_shapes, level_start_index, sampling_loc_attn, K) -> Tuple[int, ...]:
    _check_tensor(value, "value")
    _check_tensor(spatial_shapes, "spatial_shapes")
    _check_tensor(level_start_index, "level_start_index")
    _check_tensor(sampling_loc_attn, "sampling_loc_attn")
    if spatial_shapes.dtype != torch.int64 or level_start_index.dtype != torch.int64:
        raise RuntimeError("spatial_shapes and level_start_index must be int64 tensors")
    if value.dim() != 4 or sampling_loc_attn.dim() != 4:
        raise RuntimeError("value must be (B,Len_in,G,D) and sampling_loc_attn (B,Len_q,G,3*L*K)")
    if sampling_loc_attn.dtype != value.dtype:
        raise RuntimeError("value and sampling_loc_attn must have the same dtype")
    B, Len_in, G, D = value.shape
    L = spatial_shapes.shape[0]
    Len_q = sampling_loc_attn.shape[1]
    if tuple(sampling_loc_attn.shape) != (B, Len_q, G, 3 * L * K):
        raise RuntimeError(
            f"sampling_loc_attn must be ({B},Len_q,{G},{3 * L * K}), got {tuple(sampling_loc_attn.shape)}")
    return B, Len_in, G, D, L, Len_q


def flash_deform_attn_forward(value, spatial_shapes, level_start_index, sampling_loc_attn,
                              im2col_step=64, K=8, d_stride=None, block_thread=None) -> torch.Tensor:
    """Positional signature of `ext.flash_deform_attn_forward` (DCNv4_op/src/dcnv4.h:19-38).
    Returns (B, Len_q, G*D)."""
    B, Len_in, G, D, L, Len_q = _check_fda(value, spatial_shapes, level_start_index, sampling_loc_attn, K)
    _check_step(B, im2col_step)
    out = torch.empty((B, Len_q, G * D), dtype=value.dtype, device=value.device)
    with torch.cuda.device(value.device):
        rc = _lib.lib().fdab200_fwd(value.data_ptr(), spatial_shapes.data_ptr(), level_start_index.data_ptr(),
                                    sampling_loc_attn.data_ptr(), out.data_ptr(), _code(value),
                                    B, Len_in, G, D, L, Len_q, K, _stream(value))
    _lib.check(rc, "flash_deform_attn_forward")
    return out


def flash_deform_attn_backward(value, spatial_shapes, level_start_index, sampling_loc_attn, grad_output,
                               im2col_step=64, K=8, d_stride=None, block_thread=None) -> List[torch.Tensor]:
    """Positional signature of `ext.flash_deform_attn_backward` (DCNv4_op/src/dcnv4.h:40-62).
    Returns [grad_value, grad_sampling_loc_attn] in the dtype of `value`."""
    B, Len_in, G, D, L, Len_q = _check_fda(value, spatial_shapes, level_start_index, sampling_loc_attn, K)
    _check_tensor(grad_output, "grad_output")
    if grad_output.dtype != value.dtype or grad_output.numel() != B * Len_q * G * D:
        raise RuntimeError("grad_output must be (B,Len_q,G*D) in the dtype of value")
    _check_step(B, im2col_step)
    lib = _lib.lib()
    code = _code(value)
    grad_value = torch.empty_like(value)
    grad_sla = torch.empty_like(sampling_loc_attn)
    ws_bytes = lib.fdab200_bwd_workspace_bytes(code, B, Len_in, G, D)
    ws = torch.empty(ws_bytes // 4, dtype=torch.float32, device=value.device) if ws_bytes else None
    with torch.cuda.device(value.device):
        rc = lib.fdab200_bwd(value.data_ptr(), spatial_shapes.data_ptr(), level_start_index.data_ptr(),
                             sampling_loc_attn.data_ptr(), grad_output.data_ptr(), grad_value.data_ptr(),
                             grad_sla.data_ptr(), ws.data_ptr() if ws is not None else None, ws_bytes,
                             code, B, Len_in, G, D, L, Len_q, K, _stream(value))
    _lib.check(rc, "flash_deform_attn_backward")
    return [grad_value, grad_sla]


def layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float,
                       activation: str = "none") -> torch.Tensor:
    """LayerNorm over the last dimension of a contiguous CUDA tensor with the library's
    channels-last kernel (forward only; no autograd), optionally followed by GELU (erf form) in
    the same pass.  Raises ValueError for sizes the kernel does not cover -- callers that want a
    fallback check `layer_norm_supported` first."""
    if activation not in ("none", "gelu"):
        raise ValueError("activation must be 'none' or 'gelu'")
    _check_tensor(x, "input")
    _check_tensor(weight, "weight")
    _check_tensor(bias, "bias")
    C = x.shape[-1]
    if weight.numel() != C or bias.numel() != C or weight.dtype != bias.dtype:
        raise RuntimeError("weight and bias must have the size of the last dimension and one dtype")
    y = torch.empty_like(x)
    with torch.cuda.device(x.device):
        rc = _lib.lib().dcnv4b200_layernorm_act_fwd(x.data_ptr(), weight.data_ptr(), bias.data_ptr(), y.data_ptr(),
                                                    _code(x), _code(weight), x.numel() // max(C, 1), C, float(eps),
                                                    1 if activation == "gelu" else 0, _stream(x))
    _lib.check(rc, "layer_norm_forward")
    return y


def center_scale_blend_supported(x: torch.Tensor, weight: torch.Tensor, D: int) -> bool:
    """True when `center_scale_blend_forward` covers this input (dtype, size, layout)."""
    if not (x.is_cuda and x.is_contiguous() and x.dtype in _DTYPES and x.numel() > 0):
        return False
    C, es = x.shape[-1], x.element_size()
    G = weight.shape[0]
    return (C == G * D and (D * es) % 16 == 0 and C <= (1024 if es == 4 else 2048) and G <= 128
            and weight.is_cuda and weight.is_contiguous() and weight.dtype in (torch.float32, x.dtype)
            and x.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0)


def center_scale_blend_forward(x: torch.Tensor, x_proj: torch.Tensor, weight: torch.Tensor,
                               bias: torch.Tensor) -> torch.Tensor:
    """`x * (1 - s) + x_proj * s` with `s = sigmoid(x @ weight.T + bias)` repeated over each group's
    channels: the centre-feature-scale blend of the DCNv4 module in one pass (forward only; no autograd).
    x, x_proj (..., G*D) contiguous; weight (G, G*D); bias (G)."""
    for t, n in ((x, "x"), (x_proj, "x_proj"), (weight, "weight"), (bias, "bias")):
        _check_tensor(t, n)
    G, C = weight.shape
    if x.shape != x_proj.shape or x.shape[-1] != C or x.dtype != x_proj.dtype or C % G != 0 \
            or bias.numel() != G or bias.dtype != weight.dtype:
        raise RuntimeError("x and x_proj must be (..., G*D) in one dtype, weight (G, G*D), bias (G)")
    out = torch.empty_like(x)
    with torch.cuda.device(x.device):
        rc = _lib.lib().dcnv4b200_center_scale_blend_fwd(x.data_ptr(), x_proj.data_ptr(), weight.data_ptr(),
                                                         bias.data_ptr(), out.data_ptr(), _code(x), _code(weight),
                                                         x.numel() // C, G, C // G, _stream(x))
    _lib.check(rc, "center_scale_blend_forward")
    return out


def layer_norm_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """True when `layer_norm_forward` covers this input (dtype, size, layout)."""
    if not (x.is_cuda and x.is_contiguous() and x.dtype in _DTYPES and x.numel() > 0):
        return False
    C, es = x.shape[-1], x.element_size()
    if (C * es) % 16 != 0 or C > (1024 if es == 4 else 2048):
        return False
    return weight is not None and weight.is_cuda and weight.dtype in (torch.float32, x.dtype) \
        and x.data_ptr() % 16 == 0


# LayerNorm training passes ---------------------------------------------------------------------------------

LAYER_NORM_MAX_CHANNELS = 8192
LAYER_NORM_MAX_ROWS = 2 ** 30
_LN_PLAIN, _LN_POST, _LN_PRE = 0, 1, 2


def layer_norm_train_supported(x: torch.Tensor, weight: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> bool:
    """True when the LayerNorm training passes cover this input (dtypes, size, layout)."""
    return x.is_contiguous() and layer_norm_train_covers(x, weight, out_dtype)


def layer_norm_train_covers(x: torch.Tensor, weight: torch.Tensor, out_dtype: Optional[torch.dtype] = None) -> bool:
    """`layer_norm_train_supported` of `x.contiguous()`, asked without making the copy."""
    return (x.is_cuda and x.dtype in _DTYPES and x.dim() > 0
            and 0 < x.shape[-1] <= LAYER_NORM_MAX_CHANNELS and x.numel() // x.shape[-1] <= LAYER_NORM_MAX_ROWS
            and weight is not None and weight.is_cuda and weight.is_contiguous()
            and weight.dtype in (torch.float32, x.dtype) and out_dtype in (None, torch.float32, x.dtype))


def _check_ln(x, x_dtype, weight, bias, others, layer_scale, sample_scale, out_dtype):
    """Argument checks of the training passes; returns (rows, C, rows_per_sample).  `x_dtype` is the dtype of the
    branch input (x itself, except in the backward pass over a stored sum)."""
    C = x.shape[-1] if x.dim() else 0
    for t, n in ((x, "input"), (weight, "weight"), (bias, "bias"), (layer_scale, "layer_scale"),
                 (sample_scale, "sample_scale")):
        if t is not None:
            _check_tensor(t, n)
            if t.device != x.device:
                raise RuntimeError(f"{n} must be on the device of the input")
    _code(x)
    if x_dtype not in _DTYPES:
        raise RuntimeError(f"dcnv4_b200 supports float32/float16/bfloat16 tensors, got {x_dtype}")
    if out_dtype not in (torch.float32, x_dtype):
        raise RuntimeError("the result must have the dtype of the input or be float32")
    if C == 0:
        raise RuntimeError("the last dimension must not be empty")
    if C > LAYER_NORM_MAX_CHANNELS:          # before it becomes a C int
        raise ValueError(f"at most {LAYER_NORM_MAX_CHANNELS} channels, got {C}")
    for t, n in ((weight, "weight"), (bias, "bias"), (layer_scale, "layer_scale")):
        if t is not None and (t.numel() != C or t.dtype != weight.dtype):
            raise RuntimeError(f"{n} must have the size of the last dimension and the dtype of weight")
    if weight.dtype not in (torch.float32, x_dtype):
        raise RuntimeError("parameters must have the dtype of the input or be float32")
    for t, n in others:
        if t is not None:
            _check_tensor(t, n)
            if t.shape != x.shape or t.dtype != out_dtype or t.device != x.device:
                raise RuntimeError(f"{n} must have the shape of the input, dtype {out_dtype}, and its device")
    rows = x.numel() // C
    per = rows
    if sample_scale is not None:
        n = sample_scale.numel()
        if sample_scale.dtype != torch.float32 or x.dim() < 2 or (x.shape[0] % n if n else x.shape[0]) != 0:
            raise RuntimeError("sample_scale must be float32 with one factor per sample (its size divides the first "
                               "dimension of the input)")
        per = max(rows // n, 1) if n else 1
    return rows, C, per


def _ptr(t):
    return None if t is None else t.data_ptr()


_binding = None


def _load_binding():
    global _binding
    _binding = _lib.bindings()
    return _binding


def _ln_forward(mode, x, residual, weight, bias, eps, layer_scale, sample_scale, activation, out_dtype, what):
    """(y, mean, rstd), with h in front for the pre-norm seam.  The binding takes ordinary calls; what it declines -- wrong
    arguments, empty tensors, a device that is not the current one -- comes through here."""
    act = 1 if activation == "gelu" else 0
    got = (_binding or _load_binding()).ln_forward(mode, x, residual, weight, bias, eps, layer_scale, sample_scale, act,
                                                   _DTYPES.get(out_dtype, -1))
    if got.__class__ is tuple:
        return got
    if got is not None:
        _lib.check(got, what)
    rows, C, per = _check_ln(x, x.dtype, weight, bias, ((residual, "residual"),), layer_scale, sample_scale, out_dtype)
    y = torch.empty_like(x) if out_dtype == x.dtype else x.new_empty(x.shape, dtype=out_dtype)
    h = torch.empty_like(y) if mode == _LN_PRE else None
    mean = x.new_empty(rows, dtype=torch.float32)
    rstd = torch.empty_like(mean)
    rc = _on_device(
        x, _lib.lib().dcnv4b200_layernorm_train_fwd, x.data_ptr(), _ptr(residual), weight.data_ptr(), bias.data_ptr(),
        _ptr(layer_scale), _ptr(sample_scale), y.data_ptr(), _ptr(h), mean.data_ptr(), rstd.data_ptr(), mode,
        _DTYPES[x.dtype], _DTYPES[out_dtype], _DTYPES[weight.dtype], rows, C, per, eps, act, _stream(x))
    _lib.check(rc, what)
    return (y, mean, rstd) if h is None else (h, y, mean, rstd)


def _ln_backward(mode, grad_y, grad_h, x, mean, rstd, weight, bias, layer_scale, sample_scale, activation, x_dtype,
                 what, residual=None):
    """(grad_x, grad_branch, grad_weight, grad_bias, grad_layer_scale); see `_ln_forward`.  With `residual` (the seam
    in 16 bits) x is the branch, else it is the normalised tensor."""
    act = 1 if activation == "gelu" else 0
    got = (_binding or _load_binding()).ln_backward(mode, grad_y, grad_h, x, residual, mean, rstd, weight, bias,
                                                    layer_scale, sample_scale, act, _DTYPES.get(x_dtype, -1))
    if got.__class__ is tuple:
        return got
    if got is not None:
        _lib.check(got, what)
    out_dtype = grad_y.dtype
    pre = mode == _LN_PRE
    grads = ((grad_y, "grad_y"), (grad_h, "grad_h"), (residual, "residual"),
             (x, "h" if residual is None else "x")) if pre else ((grad_y, "grad_y"),)
    rows, C, per = _check_ln(x, x_dtype, weight, bias, grads, layer_scale, sample_scale, out_dtype)
    for t in (mean, rstd):
        if not (t.device == x.device and t.dtype == torch.float32 and t.is_contiguous() and t.numel() == rows):
            raise RuntimeError("mean and rstd must be the float32 row statistics the forward pass returned")
    lib = _lib.lib()
    code = _DTYPES[x_dtype]
    grad_x = torch.empty_like(x)
    branch = x.new_empty(x.shape, dtype=x_dtype) if pre and (sample_scale is not None or x_dtype != out_dtype) else None
    grad_w = torch.empty_like(weight)
    grad_b = torch.empty_like(bias)
    grad_s = None if layer_scale is None else torch.empty_like(layer_scale)
    ws_bytes = lib.dcnv4b200_layernorm_train_bwd_workspace_bytes(code, rows, C)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    if residual is not None:
        rc = _on_device(
            x, lib.dcnv4b200_add_layernorm_bwd, grad_y.data_ptr(), _ptr(grad_h), x.data_ptr(), residual.data_ptr(),
            mean.data_ptr(), rstd.data_ptr(), weight.data_ptr(), _ptr(sample_scale), grad_x.data_ptr(), _ptr(branch),
            grad_w.data_ptr(), grad_b.data_ptr(), ws.data_ptr(), ws_bytes, code, _DTYPES[weight.dtype], rows, C, per,
            _stream(x))
        _lib.check(rc, what)
        return grad_x, grad_x if branch is None else branch, grad_w, grad_b, None
    rc = _on_device(
        x, lib.dcnv4b200_layernorm_train_bwd, grad_y.data_ptr(), _ptr(grad_h), x.data_ptr(), mean.data_ptr(),
        rstd.data_ptr(), weight.data_ptr(), bias.data_ptr(), _ptr(layer_scale), _ptr(sample_scale), grad_x.data_ptr(),
        _ptr(branch), grad_w.data_ptr(), grad_b.data_ptr(), _ptr(grad_s), ws.data_ptr(), ws_bytes, mode, code,
        _DTYPES[out_dtype], _DTYPES[weight.dtype], rows, C, per, act, _stream(x))
    _lib.check(rc, what)
    return grad_x, grad_x if branch is None else branch, grad_w, grad_b, grad_s


def layer_norm_train_forward(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor, eps: float,
                             activation: str = "none", out_dtype: Optional[torch.dtype] = None):
    """LayerNorm over the last dimension of a contiguous CUDA tensor for training: (y, mean, rstd), with y optionally
    through the GELU in its erf form in the same pass (within 2.5e-7 |z| before the result is rounded; PyTorch's fp32 one is
    within 1.0e-7 |z|) and the fp32 row statistics that `layer_norm_backward` reads.  `out_dtype`
    is the dtype of x (default) or float32; weight and bias are float32 or have the dtype of x.  Up to 2^30 rows, 1 to
    8192 channels."""
    if activation not in ("none", "gelu"):
        raise ValueError("activation must be 'none' or 'gelu'")
    return _ln_forward(_LN_PLAIN, x, None, weight, bias, eps, None, None, activation,
                       x.dtype if out_dtype is None else out_dtype, "layer_norm_train_forward")


def layer_norm_backward(grad_y: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor, bias: torch.Tensor, activation: str = "none"):
    """(grad_x, grad_weight, grad_bias) of `layer_norm_train_forward`, each in the dtype of what it is the gradient
    of.  Deterministic."""
    if activation not in ("none", "gelu"):
        raise ValueError("activation must be 'none' or 'gelu'")
    gx, _, gw, gb, _ = _ln_backward(_LN_PLAIN, grad_y, None, x, mean, rstd, weight, bias, None, None, activation,
                                    x.dtype, "layer_norm_backward")
    return gx, gw, gb


def layer_norm_residual_forward(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                                eps: float, layer_scale: Optional[torch.Tensor] = None,
                                sample_scale: Optional[torch.Tensor] = None):
    """The tail of a post-norm block in one pass: out = residual + sample_scale * layer_scale * LN(x), returned with
    the row statistics as (out, mean, rstd).  `layer_scale` (C) like weight; `sample_scale` (N) float32, one factor
    per sample of the first dimension (stochastic depth: 0 or 1 / keep probability).  out and residual have the dtype
    of x or are float32."""
    return _ln_forward(_LN_POST, x, residual, weight, bias, eps, layer_scale, sample_scale, "none", residual.dtype,
                       "layer_norm_residual_forward")


def layer_norm_residual_backward(grad_out: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                                 weight: torch.Tensor, bias: torch.Tensor, layer_scale: Optional[torch.Tensor] = None,
                                 sample_scale: Optional[torch.Tensor] = None):
    """(grad_x, grad_weight, grad_bias, grad_layer_scale or None) of `layer_norm_residual_forward`; the gradient of
    the residual is `grad_out` itself.  Deterministic."""
    g = _ln_backward(_LN_POST, grad_out, None, x, mean, rstd, weight, bias, layer_scale, sample_scale, "none", x.dtype,
                     "layer_norm_residual_backward")
    return g[0], g[2], g[3], g[4]


def add_layer_norm_forward(x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor,
                           eps: float, sample_scale: Optional[torch.Tensor] = None):
    """The seam of two pre-norm branches in one pass: h = residual + sample_scale * x and y = LN(h), returned as
    (h, y, mean, rstd).  Statistics and y are taken of the fp32 sum, before h is rounded.  Types and `sample_scale`
    as `layer_norm_residual_forward`."""
    return _ln_forward(_LN_PRE, x, residual, weight, bias, eps, None, sample_scale, "none", residual.dtype,
                       "add_layer_norm_forward")


def add_layer_norm_backward(grad_y: torch.Tensor, grad_h: Optional[torch.Tensor], h: Optional[torch.Tensor],
                            mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor,
                            sample_scale: Optional[torch.Tensor] = None, x_dtype: Optional[torch.dtype] = None,
                            x: Optional[torch.Tensor] = None, residual: Optional[torch.Tensor] = None):
    """(grad_residual, grad_x, grad_weight, grad_bias) of `add_layer_norm_forward`; `grad_h` may be None, `x_dtype` is
    the dtype of the forward's x (default: that of h).  A float32 h is all the pass needs.  A 16-bit h has lost bits of
    the sum whose statistics mean and rstd are: give the forward's x and residual too (h may then be None), and the pass
    forms that sum again, bit for bit.  From a 16-bit h alone come the gradients at h as stored, normalised by its own
    mean and by rstd or what h's own spread allows, whichever is less.  Without `sample_scale` and with equal dtypes the
    first two results are one tensor.  Deterministic."""
    if (x is None) != (residual is None):
        raise RuntimeError("x and residual go together")
    if residual is not None and residual.dtype != torch.float32:
        if x_dtype not in (None, x.dtype):
            raise RuntimeError("x_dtype must be the dtype of x")
        return _ln_backward(_LN_PRE, grad_y, grad_h, x, mean, rstd, weight, weight, None, sample_scale, "none", x.dtype,
                            "add_layer_norm_backward", residual)[:4]
    if h is None:
        raise RuntimeError("h is needed where it is float32")
    return _ln_backward(_LN_PRE, grad_y, grad_h, h, mean, rstd, weight, weight, None, sample_scale, "none",
                        h.dtype if x_dtype is None else x_dtype, "add_layer_norm_backward")[:4]


NEWTON_SCHULZ_MAX_SIDE = 65536
NEWTON_SCHULZ_MAX_STEPS = 100
NEWTON_SCHULZ_COEFFICIENTS = (3.4445, -4.7750, 2.0315)   # the quintic published with the Muon optimiser


def newton_schulz(x: torch.Tensor, steps: int = 5, coefficients: Tuple[float, float, float] = NEWTON_SCHULZ_COEFFICIENTS,
                  eps: float = 1e-7) -> torch.Tensor:
    """Orthogonalise a matrix or a stack of matrices (..., m, n) by the quintic Newton-Schulz iteration:
    X = x / (|x|_F + eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T.  Contiguous CUDA tensor in
    float32 / float16 / bfloat16; the result is a new bfloat16 tensor.  The products take float16 operands whatever the
    input's type (X carries 22 bits until the last two steps) and add in float32: five steps are within 4.8e-3 of the exact
    iteration in the 2-norm, the result's rounding included, and within 2.0e-2 for a matrix of a few rows, of which a
    rounding moves a whole singular direction.  |x| may be far below eps.  Sides up to 65536, 1 to 100 steps.  No autograd.
    Deterministic."""
    _check_tensor(x, "input")
    if x.dim() < 2:
        raise RuntimeError("input must be a matrix or a stack of matrices (..., m, n)")
    a, b, c = (float(v) for v in coefficients)
    code = _code(x)
    m, n = x.shape[-2:]
    if max(m, n) > NEWTON_SCHULZ_MAX_SIDE or steps > NEWTON_SCHULZ_MAX_STEPS:          # before they become C ints
        raise ValueError(f"matrices of up to {NEWTON_SCHULZ_MAX_SIDE} rows and columns and {NEWTON_SCHULZ_MAX_STEPS} steps, got "
                         f"{m} x {n}, {steps} steps")
    out = x.new_empty(x.shape, dtype=torch.bfloat16)
    if out.numel() == 0:
        return out
    batch = out.numel() // (m * n)
    L = _lib.lib()
    ws_bytes = L.dcnv4b200_newton_schulz_workspace_bytes(batch, m, n)
    ws = x.new_empty(ws_bytes, dtype=torch.uint8)
    rc = _on_device(x, L.dcnv4b200_newton_schulz, x.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes, code, batch, m, n,
                    int(steps), a, b, c, float(eps), _stream(x))
    _lib.check(rc, "newton_schulz")
    return out


def linear_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor] = None,
                   residual: Optional[torch.Tensor] = None, activation: str = "none") -> torch.Tensor:
    """y = act(x @ weight.T + bias) [+ residual] in one tensor-core kernel (forward only; no
    autograd; fp16 / bf16).  `activation` is "none" or "gelu" (erf form, as nn.GELU()).  Raises
    ValueError / RuntimeError for inputs the kernel does not cover -- callers that want a
    fallback check `linear_supported` first."""
    _check_tensor(x, "input")
    _check_tensor(weight, "weight")
    if activation not in ("none", "gelu"):
        raise ValueError("activation must be 'none' or 'gelu'")
    N, K = weight.shape
    if x.shape[-1] != K or weight.dtype != x.dtype:
        raise RuntimeError("weight must be (out_features, in_features) in the dtype of the input")
    for t, name in ((bias, "bias"), (residual, "residual")):
        if t is not None:
            _check_tensor(t, name)
            if t.dtype != x.dtype:
                raise RuntimeError(f"{name} must have the dtype of the input")
    M = x.numel() // max(K, 1)
    if bias is not None and bias.numel() != N:
        raise RuntimeError("bias must have out_features elements")
    if residual is not None and residual.numel() != M * N:
        raise RuntimeError("residual must have the shape of the output")
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        rc = _lib.lib().dcnv4b200_linear_fwd(x.data_ptr(), weight.data_ptr(),
                                             bias.data_ptr() if bias is not None else None,
                                             residual.data_ptr() if residual is not None else None,
                                             y.data_ptr(), _code(x), M, N, K, 1 if activation == "gelu" else 0,
                                             _stream(x))
    _lib.check(rc, "linear_forward")
    return y


def linear_layer_norm_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                              residual: Optional[torch.Tensor], ln_weight: torch.Tensor, ln_bias: torch.Tensor,
                              eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, LayerNorm(y)) with y = x @ weight.T + bias [+ residual], one tensor-core kernel
    (forward only; fp16 / bf16; out_features at most 256 and a multiple of 32, of 64 above 128)."""
    _check_tensor(x, "input")
    _check_tensor(weight, "weight")
    N, K = weight.shape
    if x.shape[-1] != K or weight.dtype != x.dtype:
        raise RuntimeError("weight must be (out_features, in_features) in the dtype of the input")
    for t, name in ((bias, "bias"), (residual, "residual"), (ln_weight, "ln_weight"), (ln_bias, "ln_bias")):
        if t is not None:
            _check_tensor(t, name)
            if t.dtype != x.dtype:
                raise RuntimeError(f"{name} must have the dtype of the input")
    M = x.numel() // max(K, 1)
    if (bias is not None and bias.numel() != N) or ln_weight.numel() != N or ln_bias.numel() != N:
        raise RuntimeError("bias and LayerNorm parameters must have out_features elements")
    if residual is not None and residual.numel() != M * N:
        raise RuntimeError("residual must have the shape of the output")
    y = torch.empty(x.shape[:-1] + (N,), dtype=x.dtype, device=x.device)
    z = torch.empty_like(y)
    with torch.cuda.device(x.device):
        rc = _lib.lib().dcnv4b200_linear_ln_fwd(x.data_ptr(), weight.data_ptr(),
                                                bias.data_ptr() if bias is not None else None,
                                                residual.data_ptr() if residual is not None else None,
                                                y.data_ptr(), ln_weight.data_ptr(), ln_bias.data_ptr(), float(eps),
                                                z.data_ptr(), _code(x), M, N, K, _stream(x))
    _lib.check(rc, "linear_layer_norm_forward")
    return y, z


def linear_pair_forward(x: torch.Tensor, weight: torch.Tensor, bias: Optional[torch.Tensor],
                        n1: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Two Linear layers over the same input in one tensor-core product: `weight` is the two
    weights stacked along the output dimension, `n1` (a multiple of 64) the first layer's
    out_features.  Returns (x @ W1.T + b1, x @ W2.T + b2) as two contiguous tensors (forward
    only; fp16 / bf16)."""
    _check_tensor(x, "input")
    _check_tensor(weight, "weight")
    N, K = weight.shape
    if x.shape[-1] != K or weight.dtype != x.dtype or not 0 < n1 < N:
        raise RuntimeError("weight must be (n1 + n2, in_features) in the dtype of the input")
    if bias is not None:
        _check_tensor(bias, "bias")
        if bias.dtype != x.dtype or bias.numel() != N:
            raise RuntimeError("bias must have n1 + n2 elements in the dtype of the input")
    M = x.numel() // max(K, 1)
    y1 = torch.empty(x.shape[:-1] + (n1,), dtype=x.dtype, device=x.device)
    y2 = torch.empty(x.shape[:-1] + (N - n1,), dtype=x.dtype, device=x.device)
    with torch.cuda.device(x.device):
        rc = _lib.lib().dcnv4b200_linear_pair_fwd(x.data_ptr(), weight.data_ptr(),
                                                  bias.data_ptr() if bias is not None else None,
                                                  y1.data_ptr(), n1, y2.data_ptr(), N - n1, _code(x), M, K,
                                                  _stream(x))
    _lib.check(rc, "linear_pair_forward")
    return y1, y2


def fused_offset_supported(value: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                           bias: Optional[torch.Tensor], group: int, group_channels: int) -> bool:
    """True when `dcnv4_fused_offset_forward` covers these tensors (the kernel is specialised for
    3x3 / stride 1 / pad 1 / dilation 1, which the caller checks)."""
    if not (value.is_cuda and value.dtype in (torch.float16, torch.bfloat16) and value.is_contiguous()
            and value.dim() == 4 and value.numel() > 0 and value.data_ptr() % 32 == 0):
        return False
    if not (x.is_cuda and x.dtype == value.dtype and x.is_contiguous() and x.data_ptr() % 16 == 0):
        return False
    if not (weight.is_cuda and weight.dtype == value.dtype and weight.is_contiguous() and weight.dim() == 2
            and weight.data_ptr() % 16 == 0):
        return False
    if bias is not None and not (bias.is_cuda and bias.dtype == value.dtype and bias.is_contiguous()
                                 and bias.numel() == weight.shape[0]):
        return False
    N, H, W, C = value.shape
    rows, K = weight.shape
    return (group_channels == 16 and C == 16 * group and 0 < group <= 128
            and K % 8 == 0 and x.shape[-1] == K and x.numel() == N * H * W * K and rows >= 27 * group
            and value.numel() < 2 ** 31)


def dcnv4_fused_offset_forward(value: torch.Tensor, x: torch.Tensor, weight: torch.Tensor,
                               bias: Optional[torch.Tensor], group: int, group_channels: int,
                               offset_scale: float) -> torch.Tensor:
    """`dcnv4_forward(value, linear(x, weight, bias), 3, 3, 1, 1, 1, 1, 1, 1, group, group_channels,
    offset_scale, ...)` in one kernel: the offset/mask rows are computed by the CTA that samples
    for them and are never stored (forward only; fp16 / bf16).  value (N,H,W,C), x (N,H*W,K) or
    (N,H,W,K), weight (P,K) with P >= 27*group, bias (P) or None."""
    for t, name in ((value, "input"), (x, "offset_mask input"), (weight, "weight")):
        _check_tensor(t, name)
    if value.dim() != 4:
        raise RuntimeError("input must be an (N,H,W,C) tensor")
    N, H, W, C = value.shape
    if C != group * group_channels:
        raise RuntimeError(
            f"Input channels and group times group channels wont match: ({C} vs {group * group_channels}).")
    rows, K = weight.shape
    if x.dtype != value.dtype or weight.dtype != value.dtype or x.shape[-1] != K or x.numel() != N * H * W * K:
        raise RuntimeError("offset_mask input must be (N,H*W,K) and weight (P,K), in the dtype of the input")
    if bias is not None:
        _check_tensor(bias, "bias")
        if bias.dtype != value.dtype or bias.numel() != rows:
            raise RuntimeError("bias must have one element per weight row, in the dtype of the input")
    out = torch.empty_like(value)
    with torch.cuda.device(value.device):
        rc = _lib.lib().dcnv4b200_fwd_fused_offset(value.data_ptr(), x.data_ptr(), weight.data_ptr(),
                                                   bias.data_ptr() if bias is not None else None, out.data_ptr(),
                                                   _code(value), N, H, W, group, group_channels, K, rows,
                                                   float(offset_scale), _stream(value))
    _lib.check(rc, "dcnv4_fused_offset_forward")
    return out


class PairedLinear:
    """Inference-time cache of two nn.Linear layers that read the same input, stacked for
    `linear_pair_forward`.  The stacked copy is rebuilt whenever a parameter changed (version
    counters), moved or changed dtype.  Writes through `.data` (`param.data.copy_()` in an EMA
    update, `constant_(w.data)`) do not bump a version counter: the owning module therefore
    calls `invalidate()` from `train()`, `_load_from_state_dict()` and `_reset_parameters()`, and
    code that writes `.data` by other routes must call it too."""

    def __init__(self, first: "torch.nn.Linear", second: "torch.nn.Linear"):
        self.first, self.second = first, second
        self._key, self._weight, self._bias = None, None, None

    def invalidate(self) -> None:
        self._key, self._weight, self._bias = None, None, None

    def usable(self, x: torch.Tensor) -> bool:
        a, b = self.first, self.second
        return (FUSED_LINEAR and not needs_grad(x, a.weight, b.weight, a.bias, b.bias)
                and not torch.is_autocast_enabled() and linear_supported(x, a.weight)
                and b.weight.dtype == x.dtype and b.weight.is_cuda and a.in_features == b.in_features
                and a.in_features <= FUSED_LINEAR_MAX_K and a.out_features % 64 == 0 and b.out_features % 8 == 0
                and (a.bias is None) == (b.bias is None) and (a.bias is None or a.bias.dtype == x.dtype))

    def __call__(self, x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        a, b = self.first, self.second
        params = [t for t in (a.weight, b.weight, a.bias, b.bias) if t is not None]
        key = tuple((t.data_ptr(), t._version, t.dtype, t.device) for t in params)
        if key != self._key:
            with torch.no_grad():
                self._weight = torch.cat([a.weight, b.weight], 0).contiguous()
                self._bias = None if a.bias is None else torch.cat([a.bias, b.bias], 0).contiguous()
            self._key = key
        return linear_pair_forward(x, self._weight, self._bias, a.out_features)


def linear_supported(x: torch.Tensor, weight: torch.Tensor) -> bool:
    """True when `linear_forward` covers this input (dtype, size, layout)."""
    if not (x.is_cuda and x.is_contiguous() and x.dtype in (torch.float16, torch.bfloat16) and x.numel() > 0):
        return False
    if weight is None or not weight.is_cuda or weight.dtype != x.dtype or not weight.is_contiguous():
        return False
    N, K = weight.shape
    return N % 8 == 0 and K % 8 == 0 and x.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0


FUSED_LINEAR = True  # benchmarks turn this off to time the stock nn.Linear / GELU / add kernels
# The fused kernel streams both operands through one SM's shared memory (no 2-CTA tiles), which
# bounds long reductions by L2 bandwidth: measured against cuBLAS + separate element-wise kernels
# it wins up to K = 1024 and loses at K = 2048 (FlashInternImage-T stage-4 fc2: 45 vs 36 us).
FUSED_LINEAR_MAX_K = 1024
# DCNv4 module at inference: compute the offset/mask rows inside the sampling kernel
# (`dcnv4_fused_offset_forward`) instead of storing them from the paired projection.  Measured on a
# B200, fp16, value projection + fused kernel against paired projection + sampling kernel, us:
#   batch 256: 56x56x64 330 / 338, 28x28x128 175 / 193, 14x14x256 100 / 114, 7x7x512 68 / 67;
#   batch 32:  60 / 56, 40 / 42, 33 / 37, 30 / 37.
# It pays from 128 channels upward at any batch and at 64 channels only for large batches, hence the
# two thresholds.  Environment variable DCNV4B200_FUSED_OFFSET=0 turns it off, =1 forces it wherever
# the kernel applies (tests).
_FUSED_OFFSET_ENV = os.environ.get("DCNV4B200_FUSED_OFFSET", "")
FUSED_OFFSET_MASK = _FUSED_OFFSET_ENV != "0"
FUSED_OFFSET_MIN_CHANNELS = 128
FUSED_OFFSET_MIN_ROWS_NARROW = 4096  # rows per SM below which 64-channel layers keep the two-step path


def fused_offset_pays(rows: int, channels: int, device) -> bool:
    """Whether the module should take the fused kernel for a layer of this size (see above)."""
    if not FUSED_OFFSET_MASK:
        return False
    if _FUSED_OFFSET_ENV == "1" or channels >= FUSED_OFFSET_MIN_CHANNELS:
        return True
    return rows >= FUSED_OFFSET_MIN_ROWS_NARROW * _sm_count(device)


# The LayerNorm epilogue needs a whole row in one tile, i.e. one CTA per 128 rows: below this many
# rows per SM the separate kernels (narrower tiles, more CTAs) are faster.
LN_FUSION_MIN_ROWS_PER_SM = 64


def linear_module_forward(x: torch.Tensor, lin: "torch.nn.Linear", residual: Optional[torch.Tensor] = None,
                          activation: str = "none", norm: Optional["torch.nn.LayerNorm"] = None):
    """`y = residual + act(lin(x))` for an nn.Linear, and with `norm` (an nn.LayerNorm over the
    output features) the pair `(y, norm(y))`.  One fused tensor-core kernel when autograd is not
    needed and the kernel covers the input, else the stock PyTorch operations (same result up
    to fp rounding: the fused kernel rounds at the same points)."""
    fused = (FUSED_LINEAR and not needs_grad(x, lin.weight, lin.bias, residual)
             and not torch.is_autocast_enabled() and linear_supported(x, lin.weight) and lin.in_features <= FUSED_LINEAR_MAX_K
             and (lin.bias is None or (lin.bias.dtype == x.dtype and lin.bias.data_ptr() % 16 == 0))
             and (residual is None or (residual.dtype == x.dtype and residual.is_contiguous()
                                       and residual.data_ptr() % 16 == 0)))
    # The LayerNorm epilogue needs a whole row in one tile, i.e. one tile per 128 rows: with row
    # tiles for fewer than half of the SMs the separate kernels (narrower tiles, more CTAs) are
    # faster (measured on FlashInternImage-T stage 3: 98 tiles fused wins, 49 tiles it loses).
    if (fused and norm is not None and activation == "none" and not needs_grad(norm.weight, norm.bias)
            and _norm_fusable(norm, lin.out_features, x.dtype)
            and x.numel() // lin.in_features >= LN_FUSION_MIN_ROWS_PER_SM * _sm_count(x.device)):
        return linear_layer_norm_forward(x, lin.weight, lin.bias, residual, norm.weight, norm.bias, norm.eps)
    if fused:
        y = linear_forward(x, lin.weight, lin.bias, residual, activation)
    else:
        y = torch.nn.functional.linear(x, lin.weight, lin.bias)
        if activation == "gelu":
            y = torch.nn.functional.gelu(y)
        if residual is not None:
            y = residual + y
    return y if norm is None else (y, norm(y))


_SM_COUNT = {}


def _sm_count(device) -> int:
    idx = torch.device(device).index
    idx = torch.cuda.current_device() if idx is None else idx
    if idx not in _SM_COUNT:
        _SM_COUNT[idx] = torch.cuda.get_device_properties(idx).multi_processor_count
    return _SM_COUNT[idx]


def _norm_fusable(norm, features: int, dtype: torch.dtype) -> bool:
    return (isinstance(norm, torch.nn.LayerNorm) and norm.elementwise_affine and norm.bias is not None
            and tuple(norm.normalized_shape) == (features,) and features <= 256
            and features % (64 if features > 128 else 32) == 0
            and norm.weight.dtype == dtype and norm.bias.dtype == dtype
            and norm.weight.data_ptr() % 16 == 0 and norm.bias.data_ptr() % 16 == 0)


def bias_act_(x: torch.Tensor, bias: torch.Tensor, activation: str = "none") -> torch.Tensor:
    """In place: x = act(x + bias) over the last dimension of a contiguous fp16 / bf16 CUDA
    tensor (forward only).  `activation` is "none" or "gelu" (erf form)."""
    _check_tensor(x, "input")
    _check_tensor(bias, "bias")
    if activation not in ("none", "gelu"):
        raise ValueError("activation must be 'none' or 'gelu'")
    C = x.shape[-1]
    if bias.numel() != C or bias.dtype != x.dtype:
        raise RuntimeError("bias must have the size of the last dimension and the dtype of the input")
    with torch.cuda.device(x.device):
        rc = _lib.lib().dcnv4b200_bias_act_fwd(x.data_ptr(), bias.data_ptr(), x.data_ptr(), _code(x),
                                               x.numel() // max(C, 1), C, 1 if activation == "gelu" else 0,
                                               _stream(x))
    _lib.check(rc, "bias_act_")
    return x


def conv2d_bias_act(x: torch.Tensor, conv: "torch.nn.Conv2d", activation: str = "none") -> torch.Tensor:
    """act(conv(x)) for a biased nn.Conv2d on a channels-last image batch: at inference in fp16 /
    bf16 the bias and the activation are applied in place by one pass over the convolution's
    output instead of PyTorch's separate broadcast addition and activation kernels."""
    F = torch.nn.functional
    if (FUSED_LINEAR and not needs_grad(x, conv.weight, conv.bias) and not torch.is_autocast_enabled()
            and x.is_cuda and conv.bias is not None
            and x.dtype in (torch.float16, torch.bfloat16) and conv.weight.dtype == x.dtype
            and conv.bias.dtype == x.dtype and conv.out_channels % 8 == 0 and conv.padding_mode == "zeros"
            and conv.bias.data_ptr() % 16 == 0):
        y = F.conv2d(x, conv.weight, None, conv.stride, conv.padding, conv.dilation, conv.groups)
        rows = y.permute(0, 2, 3, 1)            # channels-last storage seen as (N, H, W, C)
        if rows.is_contiguous() and y.data_ptr() % 16 == 0:
            bias_act_(rows, conv.bias, activation)
            return y
        y = y + conv.bias.view(1, -1, 1, 1)
    else:
        y = conv(x)
    return F.gelu(y) if activation == "gelu" else y


def dcnv4_corners(p_offset, H, W, kernel_h, kernel_w, stride_h, stride_w, pad_h, pad_w, dilation_h,
                  dilation_w, group, offset_scale, remove_center) -> torch.Tensor:
    """(N,Ho,Wo,G,K,2) int32 corner indices the kernels select (test aid)."""
    _check_tensor(p_offset, "offset")
    N, Ho, Wo, P = p_offset.shape
    K = kernel_h * kernel_w - int(bool(remove_center))
    corners = torch.empty((N, Ho, Wo, group, K, 2), dtype=torch.int32, device=p_offset.device)
    with torch.cuda.device(p_offset.device):
        rc = _lib.lib().dcnv4b200_fwd_corners(p_offset.data_ptr(), corners.data_ptr(), _code(p_offset),
                                              N, H, W, group, kernel_h, kernel_w, stride_h, stride_w,
                                              pad_h, pad_w, dilation_h, dilation_w, float(offset_scale),
                                              int(remove_center), P, _stream(p_offset))
    _lib.check(rc, "dcnv4_corners")
    return corners


def flash_deform_attn_corners(spatial_shapes, sampling_loc_attn, K) -> torch.Tensor:
    """(B,Len_q,G,L*K,2) int32 corner indices the kernels select (test aid)."""
    _check_tensor(sampling_loc_attn, "sampling_loc_attn")
    B, Len_q, G, _ = sampling_loc_attn.shape
    L = spatial_shapes.shape[0]
    corners = torch.empty((B, Len_q, G, L * K, 2), dtype=torch.int32, device=sampling_loc_attn.device)
    with torch.cuda.device(sampling_loc_attn.device):
        rc = _lib.lib().fdab200_fwd_corners(spatial_shapes.data_ptr(), sampling_loc_attn.data_ptr(),
                                            corners.data_ptr(), _code(sampling_loc_attn), B, G, L, Len_q, K,
                                            _stream(sampling_loc_attn))
    _lib.check(rc, "flash_deform_attn_corners")
    return corners


def device_status() -> int:
    """Read-and-clear the current device's kernel status word (synchronises; test aid)."""
    import ctypes as C
    v = C.c_int(0)
    _lib.check(_lib.lib().dcnv4b200_device_status(C.byref(v)), "device_status")
    return v.value
