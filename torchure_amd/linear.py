"""Linear layers of a decoder block with everything that follows them, and 8-bit activations, on gfx950.

- ``fused_linear``: ``act(x W^T + b) + r`` in one product kernel, with all gradients.
- ``swiglu_mlp``: the gated feed-forward ``(silu(x Wg^T) * (x Wu^T)) Wd^T + r`` of
  torchure/models/qwen3/qwen3.py:220-230, with all gradients.
- ``quantize_activation`` / ``dequantize_activation``: the 8-bit form (``QuantizedActivation``) in which
  the two above keep what they need for the backward pass when called with ``checkpoint="e4m3"``.

The products are this package's bf16 MFMA GEMMs (``tm_lin``) with fp32 accumulation; bias, activation,
residual, the gate and its gradient, and the 8-bit form of what is kept are done on the accumulators.
As in the trainer (torchure/train/trainer.py:374), hidden states are bf16, or fp32 under bf16 autocast;
weights are bf16, or fp32 masters of which the bf16 working copy is read where it is current.
"""

from __future__ import annotations

import ctypes
import dataclasses

import torch
from torch.autograd.function import once_differentiable

from torchure_amd import _native
from torchure_amd.optimizer.working import current_copy

_BF16, _F32 = torch.bfloat16, torch.float32
_HELD = {None: _native.TM_HELD_BF16, "e4m3": _native.TM_HELD_E4M3}


def _up(n: int, to: int) -> int:
    return -(-n // to) * to


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


def _on_gpu(t: torch.Tensor, who: str, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{who}: {what} must be on a ROCm GPU device, got {t.device} (torchure_amd has no CPU path)")


def _flat(t: torch.Tensor) -> torch.Tensor:
    """``t`` as rows of its last dimension, the elements of a row next to each other and rows apart by
    at least their length."""
    t = t.detach()
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.is_neg():
        t = t.resolve_neg()
    n, d = t.shape
    if (t.stride(1) != 1 and d > 1) or (n > 1 and t.stride(0) < d):
        t = t.contiguous()
    return t


def _ld(t: torch.Tensor) -> int:
    """Elements from one row of ``_flat``'s result to the next."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _quantize(x: torch.Tensor, copy: torch.Tensor | None = None):
    n, d = x.shape
    values = torch.empty((n, _up(d, 32)), dtype=torch.uint8, device=x.device)
    exps = torch.empty((-(-n // 32), -(-d // 32)), dtype=torch.uint8, device=x.device)
    _native.check(
        _native.lib().tm_quantize_e4m3(
            values.data_ptr(), exps.data_ptr(), values.shape[1], x.data_ptr(), int(x.dtype == _F32), _ld(x), n, d,
            None if copy is None else copy.data_ptr(), 0 if copy is None else copy.shape[1],
            _native.stream_handle(x.device)),
        "tm_quantize_e4m3")
    return values, exps


def _dequantize(values, exps, out: torch.Tensor, cols: int) -> torch.Tensor:
    _native.check(
        _native.lib().tm_dequantize_e4m3(
            out.data_ptr(), int(out.dtype == _F32), out.stride(0), values.data_ptr(), exps.data_ptr(), values.shape[1],
            values.shape[0], cols, _native.stream_handle(out.device)),
        "tm_dequantize_e4m3")
    return out


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
    with torch.cuda.device(x.device):
        if x.shape[-1] == 0:
            rows = x.numel() if x.dim() == 1 else int(torch.Size(x.shape[:-1]).numel())
            empty = torch.empty((rows, 0), dtype=torch.uint8, device=x.device)
            return QuantizedActivation(empty, torch.empty((-(-rows // 32), 0), dtype=torch.uint8, device=x.device),
                                       x.shape, x.dtype)
        return QuantizedActivation(*_quantize(_flat(x)), x.shape, x.dtype)


def dequantize_activation(q: QuantizedActivation, dtype: torch.dtype | None = None) -> torch.Tensor:
    """The values that ``q`` holds, in ``dtype`` (bf16 or fp32; the quantised tensor's by default).
    Both hold them exactly."""
    who = "dequantize_activation"
    dtype = q.dtype if dtype is None else dtype
    if dtype not in (_BF16, _F32):
        raise NotImplementedError(f"{who}: dtype must be bfloat16 or float32, got {dtype}")
    _on_gpu(q.values, who, "values")
    cols = q.shape[-1]
    rows = q.shape[:-1].numel()
    if (q.values.dtype != torch.uint8 or q.exponents.dtype != torch.uint8 or q.exponents.device != q.values.device
            or tuple(q.values.shape) != (rows, _up(cols, 32))
            or tuple(q.exponents.shape) != (-(-rows // 32), -(-cols // 32))
            or not q.values.is_contiguous() or not q.exponents.is_contiguous() or q.values.data_ptr() % 16):
        raise RuntimeError(f"{who}: values {tuple(q.values.shape)} and exponents {tuple(q.exponents.shape)} are not those "
                           f"of a tensor of shape {tuple(q.shape)}")
    with torch.cuda.device(q.values.device):
        out = torch.empty(q.shape, dtype=dtype, device=q.values.device)
        if out.numel():
            _dequantize(q.values, q.exponents, out.view(rows, cols), cols)
    return out


# ---------------------------------------------------------------------------- products


def _product(op, rows, inp, out, a, b0, o0, *, b1=None, o1=None, two=False, out_f32=False, act=0, bias=None, res=None,
             held=None):
    """One ``tm_lin`` call. ``a``, ``b0`` and ``b1`` are operands (tensor, elements between rows); ``o0``
    and ``o1`` are tensors; ``held``: (kind, z0, exponents, z1, exponents)."""
    lib = _native.lib()
    d = _native.TmLin(rows=rows, inp=inp, out=out, a=a[0].data_ptr(), lda=a[1], b0=b0[0].data_ptr(), ldb=b0[1],
                      o0=o0.data_ptr(), ldo=o0.stride(0), op=op, act=act, out_f32=int(out_f32))
    if b1 is not None:
        d.b1 = b1[0].data_ptr()
    if o1 is not None:
        d.o1, d.ldo1 = o1.data_ptr(), o1.stride(0)
    if bias is not None:
        d.bias, d.bias_f32 = bias.data_ptr(), int(bias.dtype == _F32)
    if res is not None:
        d.res, d.ldr, d.res_f32 = res.data_ptr(), _ld(res), int(res.dtype == _F32)
    if held is not None:
        kind, z0, s0, z1, s1 = held
        d.held, d.z0, d.ldz = kind, z0.data_ptr(), z0.shape[1]
        if s0 is not None:
            d.s0 = s0.data_ptr()
        if z1 is not None:
            d.z1 = z1.data_ptr()
            if s1 is not None:
                d.s1 = s1.data_ptr()
    need = lib.tm_lin_workspace_bytes(op, rows, inp, out, int(two))
    ws = torch.empty(need, dtype=torch.uint8, device=o0.device) if need else None
    _native.check(lib.tm_lin(ctypes.byref(d), None if ws is None else ws.data_ptr(), need,
                             _native.stream_handle(o0.device)), "tm_lin")


def _act_grad(dz, dbias, dy, z, act):
    """``tm_act_grad``: ``dz`` = dy act'(z) (or dy, cast) into padded bf16 rows, ``dbias`` its column sums;
    either may be None. ``z``: (kind, values, exponents) or None."""
    lib = _native.lib()
    n, d = dy.shape
    need = lib.tm_act_grad_workspace_bytes(n, d) if dbias is not None else 0
    ws = torch.empty(need, dtype=torch.uint8, device=dy.device) if need else None
    kind, zv, zs = z if z is not None else (_native.TM_HELD_NOT, None, None)
    _native.check(
        lib.tm_act_grad(None if dz is None else dz.data_ptr(), 0 if dz is None else dz.stride(0),
                        None if dbias is None else dbias.data_ptr(), int(dbias is not None and dbias.dtype == _F32),
                        dy.data_ptr(), int(dy.dtype == _F32), _ld(dy), None if zv is None else zv.data_ptr(),
                        None if zs is None else zs.data_ptr(), 0 if zv is None else zv.shape[1], kind, act, n, d,
                        None if ws is None else ws.data_ptr(), need, _native.stream_handle(dy.device)),
        "tm_act_grad")


def _fits(t: torch.Tensor) -> bool:
    """Whether the kernels read the rows of ``t`` as they lie: whole 16-byte groups."""
    return t.dtype == _BF16 and t.shape[1] % 8 == 0 and _ld(t) % 8 == 0 and t.data_ptr() % 16 == 0


def _operand(t: torch.Tensor):
    """(tensor, elements between rows) of a product's operand: ``t``'s rows where the kernels read them as they
    lie, else their bf16 values in rows padded with zeros."""
    if _fits(t):
        return t, _ld(t)
    p = torch.empty((t.shape[0], _up(t.shape[1], 8)), dtype=_BF16, device=t.device)
    _act_grad(p, None, t, None, 0)
    return p, p.shape[1]


def _weight(w: torch.Tensor):
    """The operand of a weight: bf16 as it is, of an fp32 master its current working copy, or a cast."""
    if w.dtype == _F32:
        copy = current_copy(w)
        if copy is not None:
            w = copy
    return _operand(_flat(w))


def _mode(x, who):
    """Whether fp32 hidden states are cast, as autocast does; raises for what has no kernel."""
    if torch.is_autocast_enabled("cuda") and torch.get_autocast_dtype("cuda") != _BF16:
        raise NotImplementedError(f"{who}: CUDA autocast with {torch.get_autocast_dtype('cuda')} is not supported; the "
                                  "products run in bf16 (bf16 autocast, or none)")
    if x.dtype != _BF16 and not (x.dtype == _F32 and torch.is_autocast_enabled("cuda")):
        raise NotImplementedError(f"{who}: x must be bfloat16, or float32 inside bf16 CUDA autocast, got {x.dtype} with "
                                  "autocast " + ("on" if torch.is_autocast_enabled("cuda") else "off"))


def _checked(who, x, weights, bias, residual, out_features, checkpoint):
    tensors = [(x, "x"), *weights] + [(t, n) for t, n in ((bias, "bias"), (residual, "residual")) if t is not None]
    for t, what in tensors:
        _on_gpu(t, who, what)
        if t.device != x.device:
            raise RuntimeError(f"{who}: all tensors must be on one device, {what} is on {t.device}, x on {x.device}")
    _mode(x, who)
    if x.dim() == 0:
        raise RuntimeError(f"{who}: x must have at least one dimension")
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


def _out_type(residual):
    return _F32 if residual is not None and residual.dtype == _F32 else _BF16


def _held_like(kind, rows, cols, device):
    """Room for a matrix as it is kept: (values, exponents)."""
    if kind == _native.TM_HELD_BF16:
        return torch.empty((rows, _up(cols, 8)), dtype=_BF16, device=device), None
    return (torch.empty((rows, _up(cols, 32)), dtype=torch.uint8, device=device),
            torch.empty((-(-rows // 32), -(-cols // 32)), dtype=torch.uint8, device=device))


def _input(x2, kind, keep):
    """The first product's operand, and what is kept of it for the weight's gradient (None: nothing):
    (values, exponents)."""
    if not keep or kind == _native.TM_HELD_BF16:
        a = _operand(x2)
        return a, ((a[0], None) if keep else None)
    if _fits(x2):
        return (x2, _ld(x2)), _quantize(x2)
    copy = torch.empty((x2.shape[0], _up(x2.shape[1], 8)), dtype=_BF16, device=x2.device)
    return (copy, copy.shape[1]), _quantize(x2, copy)


def _kept_operand(values, exps, cols):
    """The bf16 operand of a kept input."""
    if exps is None:
        return values, _ld(values)
    p = torch.empty((values.shape[0], _up(cols, 8)), dtype=_BF16, device=values.device)
    if p.shape[1] != cols:
        p[:, cols:] = 0
    return _dequantize(values, exps, p, cols), p.shape[1]


def _aligned_vector(b):
    return None if b is None else b.detach().contiguous()


# ---------------------------------------------------------------------------- linear


def _linear_forward(x2, wt, bias, res2, act, out_features, held):
    """(y as rows, the input operand's kept form)."""
    rows, inp = x2.shape
    kind, keep_x, z = held
    a, kept = _input(x2, kind, keep_x)
    y = torch.empty((rows, out_features), dtype=_out_type(res2), device=x2.device)
    _product(_native.TM_LIN_FORWARD, rows, inp, out_features, a, wt, y, out_f32=y.dtype == _F32, act=act, bias=bias,
             res=res2, held=None if z is None else (kind, *z, None, None))
    return y, kept


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, kind):
        need_x, need_w, need_b, _ = ctx.needs_input_grad[:4]
        x2, out_features = _flat(x), weight.shape[0]
        rows = x2.shape[0]
        wt = _weight(weight)
        z = None
        if act and (need_x or need_w or need_b):
            z = _held_like(kind, rows, out_features, x.device)
        y, kept = _linear_forward(x2, wt, _aligned_vector(bias), None if residual is None else _flat(residual), act,
                                  out_features, (kind, need_w, z))
        ctx.meta = (x.shape, x.dtype, weight.shape, weight.dtype, None if bias is None else bias.dtype, act, kind, wt[1])
        ctx.save_for_backward(*(kept or (None, None)), *(z or (None, None)), wt[0] if need_x else None)
        return y.view(*x.shape[:-1], out_features)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_w, need_b, need_r = ctx.needs_input_grad[:4]
        x_shape, x_type, w_shape, w_type, b_type, act, kind, ldw = ctx.meta
        xv, xs, zv, zs, w = ctx.saved_tensors
        dx = dw = db = None
        if need_x or need_w or need_b:
            with torch.cuda.device(dy.device):
                d2 = _flat(dy)
                rows, out = d2.shape
                inp, dev = w_shape[1], dy.device
                if need_b:
                    db = torch.empty((out,), dtype=b_type, device=dev)
                products = need_x or need_w
                if act or (products and not _fits(d2)):
                    dz = torch.empty((rows, _up(out, 8)), dtype=_BF16, device=dev) if products else None
                    _act_grad(dz, db, d2, (kind, zv, zs) if act else None, act)
                else:
                    dz = d2
                    if need_b:
                        _act_grad(None, db, d2, None, 0)
                if need_x:
                    dx = torch.empty((rows, inp), dtype=x_type, device=dev)
                    _product(_native.TM_LIN_GRAD_X, rows, inp, out, (dz, _ld(dz)), (w, ldw), dx, out_f32=x_type == _F32)
                    dx = dx.view(x_shape)
                if need_w:
                    dw = torch.empty(w_shape, dtype=w_type, device=dev)
                    _product(_native.TM_LIN_GRAD_W, rows, inp, out, (dz, _ld(dz)), _kept_operand(xv, xs, inp), dw,
                             out_f32=w_type == _F32)
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
    gradients made from what is kept. The forward result is the same. Gradients have their tensors'
    types; what no gradient needs is neither kept nor computed. Differentiable once."""
    who = "fused_linear"
    if activation is None:
        activation = "none"
    if activation not in _native.TM_ACTS:
        raise ValueError(f"{who}: activation must be None or one of {', '.join(_native.TM_ACTS)}, got {activation!r}")
    if weight.dim() != 2 or x.dim() == 0 or weight.shape[1] != x.shape[-1]:
        raise RuntimeError(f"{who}: shapes x {tuple(x.shape)} and weight {tuple(weight.shape)} do not match")
    out_features = weight.shape[0]
    _checked(who, x, [(weight, "weight")], bias, residual, out_features, checkpoint)
    if weight.numel() == 0:
        raise RuntimeError(f"{who}: weight of shape {tuple(weight.shape)} has no elements")
    act, kind = _native.TM_ACTS.index(activation), _HELD[checkpoint]
    with torch.cuda.device(x.device):
        if x.numel() == 0:
            return _no_rows(x, [weight] + [t for t in (bias, residual) if t is not None], out_features, _out_type(residual))
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, bias, residual)):
            return _FusedLinear.apply(x, weight, bias, residual, act, kind)
        y, _ = _linear_forward(_flat(x), _weight(weight), _aligned_vector(bias),
                               None if residual is None else _flat(residual), act, out_features, (kind, False, None))
        return y.view(*x.shape[:-1], out_features)


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


def _no_rows(x, tensors, out_features, dtype):
    return _NoRows.apply((*x.shape[:-1], out_features), dtype, x, *tensors)


# ---------------------------------------------------------------------------- gated feed-forward


def _mlp_forward(x2, wg, wu, wd, res2, dim, ffn, held):
    """(y as rows, the input operand's kept form). ``held``: kind, whether the input is kept, and room for
    the gate's and up's products or None."""
    rows = x2.shape[0]
    kind, keep_x, z = held
    a, kept = _input(x2, kind, keep_x)
    h = torch.empty((rows, _up(ffn, 8)), dtype=_BF16, device=x2.device)
    _product(_native.TM_LIN_GATE, rows, x2.shape[1], ffn, a, wg, h, b1=wu, held=None if z is None else (kind, *z))
    y = torch.empty((rows, dim), dtype=_out_type(res2), device=x2.device)
    _product(_native.TM_LIN_FORWARD, rows, ffn, dim, (h, h.shape[1]), wd, y, out_f32=y.dtype == _F32, res=res2)
    return y, kept


def _pair(wg, wu):
    """The operands of two weights of one shape, with equal row strides."""
    g, u = _weight(wg), _weight(wu)
    if g[1] != u[1]:
        g, u = ((t[0][:, : wg.shape[1]].contiguous(), wg.shape[1]) if wg.shape[1] % 8 == 0 else t for t in (g, u))
    return g, u


class _SwigluMlp(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w_gate, w_up, w_down, residual, kind):
        need = ctx.needs_input_grad
        x2 = _flat(x)
        rows, dim, ffn = x2.shape[0], w_down.shape[0], w_gate.shape[0]
        wg, wu = _pair(w_gate, w_up)
        wd = _weight(w_down)
        z = None
        if any(need[:4]):
            z = (*_held_like(kind, rows, ffn, x.device), *_held_like(kind, rows, ffn, x.device))
        y, kept = _mlp_forward(x2, wg, wu, wd, None if residual is None else _flat(residual), dim, ffn,
                               (kind, need[1] or need[2], z))
        ctx.meta = (x.shape, x.dtype, (w_gate.shape, w_gate.dtype), (w_up.shape, w_up.dtype), (w_down.shape, w_down.dtype),
                    kind, wg[1], wd[1])
        ctx.save_for_backward(*(kept or (None, None)), *(z or (None,) * 4), *((wg[0], wu[0]) if need[0] else (None, None)),
                              wd[0] if any(need[:4]) else None)
        return y.view(*x.shape[:-1], dim)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        need_x, need_g, need_u, need_d, need_r = ctx.needs_input_grad[:5]
        x_shape, x_type, (g_shape, g_type), (u_shape, u_type), (d_shape, d_type), kind, ldw, ldd = ctx.meta
        xv, xs, g, gs, u, us, wg, wu, wd = ctx.saved_tensors
        dx = dg = du = dd = None
        if need_x or need_g or need_u or need_d:
            with torch.cuda.device(dy.device):
                d2 = _flat(dy)
                rows, out = d2.shape
                ffn, dim = g_shape
                dev, pad = dy.device, _up(ffn, 64)
                a = _operand(d2)
                # [d_gate | d_up] and the product of the down projection's input again
                both = torch.empty((rows, 2 * pad), dtype=_BF16, device=dev)
                h = torch.empty((rows, pad), dtype=_BF16, device=dev) if need_d else None
                _product(_native.TM_LIN_GATE_GRAD, rows, ffn, out, a, (wd, ldd), both, o1=h, held=(kind, g, gs, u, us))
                if need_d:
                    dd = torch.empty(d_shape, dtype=d_type, device=dev)
                    _product(_native.TM_LIN_GRAD_W, rows, ffn, out, a, (h, pad), dd, out_f32=d_type == _F32)
                    del h
                if need_x:
                    dx = torch.empty((rows, dim), dtype=x_type, device=dev)
                    _product(_native.TM_LIN_GRAD_X, rows, dim, ffn, (both, 2 * pad), (wg, ldw), dx, b1=(wu, ldw), two=True,
                             out_f32=x_type == _F32)
                    dx = dx.view(x_shape)
                if need_g or need_u:
                    xb = _kept_operand(xv, xs, dim)
                    if need_g:
                        dg = torch.empty(g_shape, dtype=g_type, device=dev)
                    if need_u:
                        du = torch.empty(u_shape, dtype=u_type, device=dev)
                    if need_g and need_u and g_type == u_type:
                        _product(_native.TM_LIN_GRAD_W, rows, dim, ffn, (both, 2 * pad), xb, dg, o1=du, two=True,
                                 out_f32=g_type == _F32)
                    else:
                        for d, at in ((dg, 0), (du, pad)):
                            if d is not None:
                                _product(_native.TM_LIN_GRAD_W, rows, dim, ffn, (both[:, at:], 2 * pad), xb, d,
                                         out_f32=d.dtype == _F32)
        return dx, dg, du, dd, dy if need_r else None, None


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
    product. Gradients have their tensors' types; what no gradient needs is neither kept nor computed.
    Differentiable once."""
    who = "swiglu_mlp"
    if (w_gate.dim() != 2 or w_up.shape != w_gate.shape or w_down.dim() != 2 or w_down.shape[1] != w_gate.shape[0]
            or x.dim() == 0 or w_gate.shape[1] != x.shape[-1]):
        raise RuntimeError(f"{who}: shapes x {tuple(x.shape)}, w_gate {tuple(w_gate.shape)}, w_up {tuple(w_up.shape)}, "
                           f"w_down {tuple(w_down.shape)} do not match")
    dim, ffn = w_down.shape
    _checked(who, x, [(w_gate, "w_gate"), (w_up, "w_up"), (w_down, "w_down")], None, residual, dim, checkpoint)
    if w_gate.numel() == 0 or w_down.numel() == 0:
        raise RuntimeError(f"{who}: weights of shapes {tuple(w_gate.shape)} and {tuple(w_down.shape)} have no elements")
    kind = _HELD[checkpoint]
    with torch.cuda.device(x.device):
        if x.numel() == 0:
            return _no_rows(x, [w_gate, w_up, w_down] + ([] if residual is None else [residual]), dim, _out_type(residual))
        if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, w_gate, w_up, w_down, residual)):
            return _SwigluMlp.apply(x, w_gate, w_up, w_down, residual, kind)
        wg, wu = _pair(w_gate, w_up)
        y, _ = _mlp_forward(_flat(x), wg, wu, _weight(w_down), None if residual is None else _flat(residual), dim, ffn,
                            (kind, False, None))
        return y.view(*x.shape[:-1], dim)
