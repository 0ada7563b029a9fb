"""Layer norm and RMS norm over the last dimension, on gfx950: what stands before a decoder block's products
(torchure/models/qwen3/qwen3.py:86-217,243-274: the block's and the final RMS norm, and those of the query and key heads).

One kernel each way, and one that adds the workgroups' sums of the weight's gradient in order (``tm_norm_forward``,
``tm_norm_backward``). Statistics, products and sums are fp32 whatever the types; results are rounded once.
Autocast does not change what is computed: ``dtype`` says what comes out, so that the fp32 residual stream's norm
can be the bf16 operand of the product behind it.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from torchure_amd import _native
from torchure_amd.linear import _current, _NoRows, _on_gpu, _wants_autograd

_BF16, _F32 = torch.bfloat16, torch.float32
MAX_FEATURES = 16384


class _Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, layer, eps, y_f32):
        with _current(x.device):
            y, *kept = _native.layer_host().norm_forward(x, weight, bias, layer, eps, y_f32, any(ctx.needs_input_grad[:3]),
                                                         _native.stream_handle(x.device))
        ctx.meta = (x.shape, layer, weight is not None and weight.dtype == _F32, bias is not None and bias.dtype == _F32)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need = ctx.needs_input_grad[:3]
        grads = (None,) * 3
        if any(need):
            with _current(dy.device):
                grads = _native.layer_host().norm_backward(dy, *ctx.saved_tensors, *ctx.meta, *need,
                                                           _native.stream_handle(dy.device))
        return *grads, None, None, None


def _checked(who, x, weight, bias, dtype):
    for t, what in ((x, "x"), (weight, "weight"), (bias, "bias")):
        if t is None:
            continue
        _on_gpu(t, who, what)
        if t.device != x.device:
            raise RuntimeError(f"{who}: all tensors must be on one device, {what} is on {t.device}, x on {x.device}")
        if t.layout != torch.strided:
            raise NotImplementedError(f"{who}: {what} must be dense, got {t.layout}")
        if t.dtype not in (_BF16, _F32):
            raise NotImplementedError(f"{who}: {what} must be bfloat16 or float32, got {t.dtype}")
    if x.dim() == 0:
        raise ValueError(f"{who}: x must have at least one dimension")
    features = x.shape[-1]
    if not 0 < features <= MAX_FEATURES:
        raise RuntimeError(f"{who}: {features} features, supported are 1 to {MAX_FEATURES}")
    for t, what in ((weight, "weight"), (bias, "bias")):
        if t is not None and tuple(t.shape) != (features,):
            raise RuntimeError(f"{who}: {what} of shape {tuple(t.shape)} for {features} features")


def _norm(who, x, weight, bias, layer, eps, dtype):
    host = _native.layer_host()
    if dtype is None:
        dtype = x.dtype
    elif dtype not in (_BF16, _F32):
        raise NotImplementedError(f"{who}: dtype must be bfloat16 or float32, got {dtype}")
    eps = float(eps)
    if not eps >= 0.0:
        raise ValueError(f"{who}: eps must not be negative, got {eps}")
    if not x.is_cuda or not host.norm_plain(x, weight, bias, torch.cuda.current_device()):
        _checked(who, x, weight, bias, dtype)
        if x.numel() == 0:
            return _NoRows.apply(x.shape, dtype, x, *(t for t in (weight, bias) if t is not None))
    if _wants_autograd(x, weight, bias):
        return _Norm.apply(x, weight, bias, layer, eps, dtype == _F32)
    with _current(x.device):
        return host.norm_forward(x, weight, bias, layer, eps, dtype == _F32, False, _native.stream_handle(x.device))[0]


def rms_norm(
    x: torch.Tensor,  # (..., features), bf16 or fp32
    weight: torch.Tensor | None = None,  # (features,), bf16 or fp32
    eps: float = 1e-6,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in ``dtype`` (bf16 or fp32; x's by default). All
    gradients, in their tensors' types; what no gradient needs is neither kept nor computed. Kept for the backward
    pass are x and one fp32 value a row. Differentiable once, in reverse mode."""
    return _norm("rms_norm", x, weight, None, False, eps, dtype)


def layer_norm(
    x: torch.Tensor,  # (..., features), bf16 or fp32
    weight: torch.Tensor | None = None,  # (features,), bf16 or fp32
    bias: torch.Tensor | None = None,  # (features,)
    eps: float = 1e-5,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``(x - mean(x)) / sqrt(var(x) + eps) * weight + bias`` over the last dimension (var: the mean squared distance from the
    mean), in ``dtype`` (bf16 or fp32; x's by default). Gradients and what is kept as for ``rms_norm``, with two fp32
    values a row."""
    return _norm("layer_norm", x, weight, bias, True, eps, dtype)
