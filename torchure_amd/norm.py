"""Layer norm and RMS norm over the last dimension, on gfx950: what stands before a decoder block's products
(torchure/models/qwen3/qwen3.py:86-217,243-274: the block's and the final RMS norm, and those of the query and key heads).

One kernel each way, and one that adds the workgroups' sums of the weight's gradient in order (``tm_norm_forward``,
``tm_norm_backward``). Statistics, products and sums are fp32 whatever the types; results are rounded once.
Autocast does not change what is computed: ``dtype`` says what comes out, so that the fp32 residual stream's norm
can be the bf16 operand of the product behind it.
"""

from __future__ import annotations

import torch
from torch.autograd import forward_ad

from torchure_amd import _native
from torchure_amd.linear import _NoRows, _on_gpu

_BF16, _F32 = torch.bfloat16, torch.float32
MAX_FEATURES = 16384


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


def _refuse_tangents(who, *tensors):
    """A forward-mode tangent is refused: the kernels would drop it."""
    if forward_ad._current_level >= 0:  # inside dual_level
        if any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
            raise NotImplementedError(f"{who}: forward-mode derivatives are not supported")


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
            _refuse_tangents(who, x, weight, bias)
            return _NoRows.apply(x.shape, dtype, x, *(t for t in (weight, bias) if t is not None))
    _refuse_tangents(who, x, weight, bias)
    return host.norm(x, weight, bias, layer, eps, dtype == _F32, _native.stream_handle(x.device))


def rms_norm(
    x: torch.Tensor,  # (..., features), bf16 or fp32
    weight: torch.Tensor | None = None,  # (features,), bf16 or fp32
    eps: float = 1e-6,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``x / sqrt(mean(x^2) + eps) * weight`` over the last dimension, in ``dtype`` (bf16 or fp32; x's by default). All
    gradients, in their tensors' types. Kept for the backward pass are x and one fp32 value a row, for x's and the
    weight's gradient, and for x's the weight; what no gradient needs is not kept. Differentiable once, in reverse mode."""
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
    values a row; for the bias's gradient nothing is."""
    return _norm("layer_norm", x, weight, bias, True, eps, dtype)
