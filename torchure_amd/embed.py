"""Token embedding with scaling, and the table's gradient, on gfx950: the way into a decoder
(torchure/models/qwen3/qwen3.py:285-286, whose table is the head's weight too).

The lookup is one kernel. The gradient puts the tokens in order by id and sums their rows in fp32, without atomics
on values: the same bits every time (``tm_embed_lookup``, ``tm_embed_grad``).
"""

from __future__ import annotations

import torch

from torchure_amd import _native
from torchure_amd.linear import _current, _NoRows, _on_gpu
from torchure_amd.norm import _refuse_tangents

_BF16, _F32 = torch.bfloat16, torch.float32


def _checked(who, ids, table, name):
    for t, what in ((table, name), (ids, "ids")):
        _on_gpu(t, who, what)
        if t.device != table.device:
            raise RuntimeError(f"{who}: all tensors must be on one device, {what} is on {t.device}, {name} on {table.device}")
        if t.layout != torch.strided:
            raise NotImplementedError(f"{who}: {what} must be dense, got {t.layout}")
    if table.dtype not in (_BF16, _F32):
        raise NotImplementedError(f"{who}: {name} must be bfloat16 or float32, got {table.dtype}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise NotImplementedError(f"{who}: ids must be int64 or int32, got {ids.dtype}")
    if table.dim() != 2 or table.numel() == 0:
        raise RuntimeError(f"{who}: {name} of shape {tuple(table.shape)}, expected (ids, features) with elements")


def _padding(who, padding_idx, vocab) -> int:
    if padding_idx is None:
        return -1
    if not -vocab <= padding_idx < vocab:
        raise ValueError(f"{who}: padding_idx {padding_idx} for {vocab} ids")
    return padding_idx % vocab


def embedding(
    ids: torch.Tensor,  # (...), int64 or int32
    weight: torch.Tensor,  # (ids, features), bf16 or fp32
    scale: float = 1.0,
    padding_idx: int | None = None,
    dtype: torch.dtype | None = None,
) -> torch.Tensor:
    """``scale * weight[ids]``, in ``dtype`` (bf16 or fp32; the weight's by default), rounded once. The weight's gradient is a whole
    table in its type: ``scale`` times the sums of the result's gradients by id, in fp32 and in the tokens' order; tokens whose
    id is ``padding_idx`` take no part in it. Kept for the backward pass are the ids.

    An id outside the table gives a row of NaN and no gradient: ids are on the device, where the host cannot look at them
    without waiting. Autocast changes nothing. Differentiable once, in reverse mode."""
    who = "embedding"
    host = _native.layer_host()
    if dtype is not None and dtype not in (_BF16, _F32):
        raise NotImplementedError(f"{who}: dtype must be bfloat16 or float32, got {dtype}")
    if not weight.is_cuda or not host.embedding_plain(ids, weight, torch.cuda.current_device()):
        _checked(who, ids, weight, "weight")
    padding = -1 if padding_idx is None else _padding(who, padding_idx, weight.shape[0])
    dtype = weight.dtype if dtype is None else dtype
    _refuse_tangents(who, weight)
    if ids.numel() == 0:
        return _NoRows.apply((*ids.shape, weight.shape[1]), dtype, weight)
    return host.embedding(ids, weight, scale, padding, dtype == _F32, _native.stream_handle(weight.device))


def _apart(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether the bytes from a's first to its last element and b's have none in common."""
    spans = []
    for t in (a, b):
        last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
        spans.append((t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size()))
    return spans[0][1] <= spans[1][0] or spans[1][1] <= spans[0][0]


@torch.no_grad()
def embedding_grad_(
    grad: torch.Tensor,  # (ids, features), bf16 or fp32
    ids: torch.Tensor,  # (...), int64 or int32
    dy: torch.Tensor,  # (..., features), bf16 or fp32
    scale: float = 1.0,
    padding_idx: int | None = None,
) -> torch.Tensor:
    """Adds ``embedding``'s weight gradient to ``grad`` in place and returns it: only the rows of ids that occur are read and
    written, where autograd fills a whole table and adds two (a tied head's: 2 x 622 MB beside the 34 of 8192 tokens at 1024 features of
    151,936 ids). Each row is rounded once. For a program that has the embedding's output gradient, as its last step back:

        x = embedding(ids, weight.detach()).requires_grad_()
        ...                                                  # the loss from x; its backward pass fills weight.grad and x.grad
        embedding_grad_(weight.grad, ids, x.grad)
    """
    who = "embedding_grad_"
    _checked(who, ids, grad, "grad")
    _on_gpu(dy, who, "dy")
    if dy.device != grad.device:
        raise RuntimeError(f"{who}: all tensors must be on one device, dy is on {dy.device}, grad on {grad.device}")
    if dy.layout != torch.strided:
        raise NotImplementedError(f"{who}: dy must be dense, got {dy.layout}")
    if dy.dtype not in (_BF16, _F32):
        raise NotImplementedError(f"{who}: dy must be bfloat16 or float32, got {dy.dtype}")
    if tuple(dy.shape) != (*ids.shape, grad.shape[1]):
        raise RuntimeError(f"{who}: dy of shape {tuple(dy.shape)} for ids {tuple(ids.shape)} and {grad.shape[1]} features")
    rows, features = grad.shape
    if (features > 1 and grad.stride(1) != 1) or (rows > 1 and grad.stride(0) < features) or grad.is_neg():
        raise RuntimeError(f"{who}: grad of strides {grad.stride()}, its rows must lie apart, each in one piece")
    if grad.requires_grad:
        raise RuntimeError(f"{who}: grad requires a gradient itself and cannot be changed in place")
    if grad.is_inference() and not torch.is_inference_mode_enabled():
        raise RuntimeError(f"{who}: grad is an inference tensor and cannot be changed in place outside inference mode")
    padding = _padding(who, padding_idx, rows)
    _refuse_tangents(who, grad, dy)
    if ids.numel() == 0:
        return grad
    if not _apart(grad, dy):
        raise RuntimeError(f"{who}: grad and dy share memory")
    with _current(grad.device):
        _native.layer_host().embedding_grad(grad, ids, dy, scale, padding, _native.stream_handle(grad.device))
    _native.host().bump([grad])
    return grad
