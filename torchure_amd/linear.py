"""Linear layers of a decoder block with everything that follows them, and 8-bit activations, on gfx950.

- ``fused_linear``: ``act(x W^T + b) + r`` in one product kernel, with all gradients.
- ``swiglu_mlp``: the gated feed-forward ``(silu(x Wg^T) * (x Wu^T)) Wd^T + r`` of
  torchure/models/qwen3/qwen3.py:220-230, with all gradients.
- ``quantize_activation`` / ``dequantize_activation``: the 8-bit form (``QuantizedActivation``) in which
  the two above keep what they need for the backward pass when called with ``checkpoint="e4m3"``.

The products are this package's bf16 MFMA GEMMs (``tm_lin``) with fp32 accumulation; bias, activation,
residual, the gate and its gradient, and the 8-bit form of what is kept are done on the accumulators. What
a product reads is rounded to bf16 first, as autocast and a bf16 module's autograd do: fp32 operands, the
gated result, and in the backward pass the gradients of the pre-activation, gate and up.
As in the trainer (torchure/train/trainer.py:374), hidden states are bf16, or fp32 under bf16 autocast;
weights are bf16, or fp32 masters of which the bf16 working copy is read where it is current.
"""

from __future__ import annotations

import contextlib
import dataclasses

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from torchure_amd import _native
from torchure_amd.optimizer.working import current_copy

_BF16, _F32 = torch.bfloat16, torch.float32
_HELD = {None: _native.TM_HELD_BF16, "e4m3": _native.TM_HELD_E4M3}
_ACTS = {None: 0, **{name: i for i, name in enumerate(_native.TM_ACTS)}}


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


def _on_gpu(t: torch.Tensor, who: str, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{who}: {what} must be on a ROCm GPU device, got {t.device} (torchure_amd has no CPU path)")


def _current(device: torch.device):
    """Makes ``device`` the current one, which a launch's kernels are looked up on."""
    if device.index is None or device.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(device)


# ---------------------------------------------------------------------------- 8-bit activations


@dataclasses.dataclass(frozen=True)
class QuantizedActivation:
    """A tensor's values in 8 bits. ``values`` (uint8, rows x the width's next multiple of 32) are
    e4m3 bits, ``exponents`` (uint8, one for each block of 32 rows x 32 columns) are e + 127: a value is
    e4m3 * 2^e. ``shape`` and ``dtype`` are the tensor's own; its rows are those of ``shape`` with
    all dimensions but the last taken together."""

    values: torch.Tensor
    exponents: torch.Tensor
    shape: torch.Size
    dtype: torch.dtype

    @property
    def nbytes(self) -> int:
        return self.values.numel() + self.exponents.numel()


def quantize_activation(x: torch.Tensor) -> QuantizedActivation:
    """``x`` (bf16 or fp32, any shape, at least one dimension) in 8 bits: e4m3 values with one power of
    two for each block of 32 rows x 32 columns, the least with which the block's largest finite
    magnitude is at most 448 times it. A value is off by at most 2^-4 of itself, or 2^-10 of
    its block's power of two. Infinities and NaN come back as NaN, values past 448 * 2^119 as that.
    Not differentiable: the result is data."""
    who = "quantize_activation"
    _on_gpu(x, who, "x")
    if x.dtype not in (_BF16, _F32):
        raise NotImplementedError(f"{who}: x must be bfloat16 or float32, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError(f"{who}: x must have at least one dimension")
    if x.numel() == 0:
        rows, cols = x.shape[:-1].numel(), x.shape[-1]
        values = torch.zeros((rows, _up(cols, 32)), dtype=torch.uint8, device=x.device)
        exponents = torch.zeros((-(-rows // 32), -(-cols // 32)), dtype=torch.uint8, device=x.device)
    else:
        with _current(x.device):
            values, exponents = _native.lin_host().act_quantize(x, _native.stream_handle(x.device))
    return QuantizedActivation(values, exponents, x.shape, x.dtype)


def dequantize_activation(q: QuantizedActivation, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values that ``q`` holds, in ``dtype`` (bf16 or fp32; the quantised tensor's by default).
    Both hold them exactly."""
    who = "dequantize_activation"
    dtype = q.dtype if dtype is None else dtype
    if dtype not in (_BF16, _F32):
        raise NotImplementedError(f"{who}: dtype must be bfloat16 or float32, got {dtype}")
    v, e = q.values, q.exponents
    _on_gpu(v, who, "values")
    rows, cols = (q.shape[:-1].numel(), q.shape[-1]) if len(q.shape) else (0, 0)
    if (not len(q.shape) or v.dtype != torch.uint8 or e.dtype != torch.uint8 or e.device != v.device
            or v.shape != (rows, _up(cols, 32)) or e.shape != (-(-rows // 32), -(-cols // 32))
            or not v.is_contiguous() or not e.is_contiguous() or v.data_ptr() % 16):
        raise RuntimeError(f"{who}: values {tuple(v.shape)} and exponents {tuple(e.shape)} are not those of a tensor of "
                           f"shape {tuple(q.shape)}")
    with _current(v.device):
        return _native.lin_host().act_dequantize(v, e, q.shape, dtype == _F32, _native.stream_handle(v.device))


# ---------------------------------------------------------------------------- checks


def _checked(who, x, weights, bias, residual, out_features, checkpoint):
    tensors = [(x, "x"), *weights] + [(t, n) for t, n in ((bias, "bias"), (residual, "residual")) if t is not None]
    for t, what in tensors:
        _on_gpu(t, who, what)
        if t.device != x.device:
            raise RuntimeError(f"{who}: all tensors must be on one device, {what} is on {t.device}, x on {x.device}")
    autocast = torch.is_autocast_enabled("cuda")
    if autocast and torch.get_autocast_dtype("cuda") != _BF16:
        raise NotImplementedError(f"{who}: CUDA autocast with {torch.get_autocast_dtype('cuda')} is not supported; the "
                                  "products run in bf16 (bf16 autocast, or none)")
    if x.dtype != _BF16 and not (x.dtype == _F32 and autocast):
        raise NotImplementedError(f"{who}: x must be bfloat16, or float32 inside bf16 CUDA autocast, got {x.dtype} with "
                                  "autocast " + ("on" if autocast else "off"))
    for t, what in tensors[1:]:
        if t.dtype not in (_BF16, _F32):
            raise NotImplementedError(f"{who}: {what} must be bfloat16 or float32, got {t.dtype}")
    if bias is not None and tuple(bias.shape) != (out_features,):
        raise RuntimeError(f"{who}: bias of shape {tuple(bias.shape)} for {out_features} out features")
    if residual is not None and tuple(residual.shape) != (*x.shape[:-1], out_features):
        raise RuntimeError(f"{who}: residual of shape {tuple(residual.shape)}, the result's is "
                           f"{(*x.shape[:-1], out_features)}")
    if checkpoint not in _HELD:
        raise ValueError(f"{who}: checkpoint must be None or 'e4m3', got {checkpoint!r}")


def _bf16_source(w: torch.Tensor) -> torch.Tensor:
    """What a weight's operand is made of: of an fp32 master its bf16 working copy where that is current (the
    bits of the cast), else the weight."""
    if w.dtype == _F32:
        copy = current_copy(w)
        if copy is not None:
            return copy
    return w


def _wants_autograd(*tensors) -> bool:
    """Whether a call goes through its autograd function: a tensor requires a gradient, or carries a
    forward-mode tangent, which the function refuses and a direct call would drop."""
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    if forward_ad._current_level >= 0:  # inside dual_level
        return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)
    return False


class _NoRows(torch.autograd.Function):
    """A call without rows: an empty result, zero gradients."""

    @staticmethod
    def forward(ctx, shape, dtype, *tensors):
        ctx.like = [(t.shape, t.dtype, t.device) for t in tensors]
        return torch.empty(shape, dtype=dtype, device=tensors[0].device)

    @staticmethod
    def backward(ctx, dy):
        return None, None, *(torch.zeros(s, dtype=t, device=d) if need else None
                             for (s, t, d), need in zip(ctx.like, ctx.needs_input_grad[2:]))


def _no_rows(x, tensors, residual, out_features):
    dtype = _F32 if residual is not None and residual.dtype == _F32 else _BF16
    return _NoRows.apply((*x.shape[:-1], out_features), dtype, x, *(t for t in (*tensors, residual) if t is not None))


# ---------------------------------------------------------------------------- linear


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, kind):
        need_x, need_w, need_b, _ = ctx.needs_input_grad[:4]
        with _current(x.device):
            y, *kept = _native.lin_host().lin_forward(x, _bf16_source(weight), bias, residual, act, kind, need_w,
                                                      bool(act) and (need_x or need_w or need_b), need_x,
                                                      _native.stream_handle(x.device))
        ctx.meta = (x.shape, x.dtype == _F32, weight.dtype == _F32, bias is not None and bias.dtype == _F32, act, kind)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        dx = dw = db = None
        if need_x or need_w or need_b:
            with _current(dy.device):
                dx, dw, db = _native.lin_host().lin_backward(dy, *ctx.saved_tensors, *ctx.meta, need_x, need_w, need_b,
                                                             _native.stream_handle(dy.device))
        return dx, dw, db, dy if need_r else None, None, None


def fused_linear(
    x: torch.Tensor,  # (..., in), bf16, or fp32 inside bf16 autocast
    weight: torch.Tensor,  # (out, in), bf16 or an fp32 master
    bias: torch.Tensor | None = None,  # (out,)
    residual: torch.Tensor | None = None,  # (..., out)
    activation: str | None = None,
    checkpoint: str | None = None,
) -> torch.Tensor:
    """``activation(x @ weight.T + bias) + residual``: one product with the rest done on its fp32
    sums, rounded once. The result is bf16, or fp32 with an fp32 residual (the trainer's residual stream).

    ``activation``: None or "none", "relu", "silu", "gelu" or "gelu_tanh". ``checkpoint``: how the input (for
    the weight's gradient) and the pre-activation (for all of them) are kept until the backward
    pass: None for bf16, "e4m3" for 8 bits (``quantize_activation``'s form): half the bytes, and
    gradients made from what is kept (of an fp32 x its fp32 values in 8 bits). The forward result is the same.

    The gradient of the pre-activation (without an activation an fp32 result's gradient itself) is rounded to
    bf16 for the products that make x's and the weight's gradients from it, whatever their types, and not for
    the bias's. Gradients have their tensors' types; what no gradient needs is neither kept nor computed.
    Differentiable once, in reverse mode."""
    host = _native.lin_host()
    act, kind = _ACTS.get(activation), _HELD.get(checkpoint)
    if act is None or kind is None or torch.is_autocast_enabled("cuda") or not x.is_cuda or not host.lin_plain(
            x, (weight,), bias, residual, weight.shape[0] if weight.dim() else 0,
            torch.cuda.current_device()) or weight.shape[1] != x.shape[-1]:
        who = "fused_linear"
        if act is None:
            raise ValueError(f"{who}: activation must be None or one of {', '.join(_native.TM_ACTS)}, got {activation!r}")
        if weight.dim() != 2 or x.dim() == 0 or weight.shape[1] != x.shape[-1]:
            raise RuntimeError(f"{who}: shapes x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
        _checked(who, x, [(weight, "weight")], bias, residual, weight.shape[0], checkpoint)
        if weight.numel() == 0:
            raise RuntimeError(f"{who}: weight of shape {tuple(weight.shape)} has no elements")
        if x.numel() == 0:
            return _no_rows(x, (weight, bias), residual, weight.shape[0])
    if _wants_autograd(x, weight, bias, residual):
        return _FusedLinear.apply(x, weight, bias, residual, act, kind)
    with _current(x.device):
        return host.lin_forward(x, _bf16_source(weight), bias, residual, act, kind, False, False, False,
                                _native.stream_handle(x.device))[0]


# ---------------------------------------------------------------------------- gated feed-forward


class _SwigluMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, residual, kind):
        need_x, need_g, need_u, need_d, _ = ctx.needs_input_grad[:5]
        behind_gate = need_x or need_g or need_u
        with _current(x.device):
            y, *kept = _native.lin_host().mlp_forward(
                x, _bf16_source(w_gate), _bf16_source(w_up), _bf16_source(w_down), residual, kind, need_g or need_u,
                behind_gate or need_d, need_x, behind_gate, _native.stream_handle(x.device))
        ctx.meta = (x.shape, w_gate.shape[0], *(t.dtype == _F32 for t in (x, w_gate, w_up, w_down)), kind)
        ctx.save_for_backward(*kept)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need, need_r = ctx.needs_input_grad[:4], ctx.needs_input_grad[4]
        grads = (None,) * 4
        if any(need):
            with _current(dy.device):
                grads = _native.lin_host().mlp_backward(dy, *ctx.saved_tensors, *ctx.meta, *need,
                                                        _native.stream_handle(dy.device))
        return *grads, dy if need_r else None, None


def swiglu_mlp(
    x: torch.Tensor,  # (..., dim), bf16, or fp32 inside bf16 autocast
    w_gate: torch.Tensor,  # (ffn, dim), bf16 or an fp32 master
    w_up: torch.Tensor,  # (ffn, dim)
    w_down: torch.Tensor,  # (out, ffn)
    residual: torch.Tensor | None = None,  # (..., out)
    checkpoint: str | None = None,
) -> torch.Tensor:
    """``(silu(x @ w_gate.T) * (x @ w_up.T)) @ w_down.T + residual``, the feed-forward of
    torchure/models/qwen3/qwen3.py:220-230 (no biases) with the block's residual. The result is bf16, or
    fp32 with an fp32 residual.

    The forward pass is two products: gate and up together, with the gate applied to their fp32 sums
    and its result rounded to bf16, then the down projection with the residual. Kept for the backward
    pass are the input and the two products, in bf16 or, with ``checkpoint="e4m3"``, in 8 bits
    (``quantize_activation``'s form); the gated result is made from them again, where an
    ordinary module keeps it too. The backward pass applies the gate's gradient on the sums of its first
    product, whose two results, of gate and up, are made together where either's weight or x wants a
    gradient; both are rounded to bf16 for the products behind them, as is an fp32 result's gradient for
    the first. Gradients have their tensors' types; what else no gradient needs is neither kept nor computed.
    Differentiable once, in reverse mode."""
    host = _native.lin_host()
    kind = _HELD.get(checkpoint)
    shapes_fit = (w_gate.dim() == 2 and w_up.shape == w_gate.shape and w_down.dim() == 2 and x.dim() > 0
                  and w_down.shape[1] == w_gate.shape[0] and w_gate.shape[1] == x.shape[-1])
    if kind is None or not shapes_fit or torch.is_autocast_enabled("cuda") or not x.is_cuda or not host.lin_plain(
            x, (w_gate, w_up, w_down), None, residual, w_down.shape[0], torch.cuda.current_device()):
        who = "swiglu_mlp"
        if not shapes_fit:
            raise RuntimeError(f"{who}: shapes x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}, "
                               f"w_down {tuple(w_down.shape)} do not match")
        _checked(who, x, [(w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")], None, residual, w_down.shape[0],
                 checkpoint)
        if w_gate.numel() == 0 or w_down.numel() == 0:
            raise RuntimeError(f"{who}: weights of shapes {tuple(w_gate.shape)} and {tuple(w_down.shape)} have no elements")
        if x.numel() == 0:
            return _no_rows(x, (w_gate, w_up, w_down), residual, w_down.shape[0])
    if _wants_autograd(x, w_gate, w_up, w_down, residual):
        return _SwigluMlp.apply(x, w_gate, w_up, w_down, residual, kind)
    with _current(x.device):
        return host.mlp_forward(x, _bf16_source(w_gate), _bf16_source(w_up), _bf16_source(w_down), residual, kind, False,
                                False, False, False, _native.stream_handle(x.device))[0]
