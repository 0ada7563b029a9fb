"""Forward-mode derivatives of the linear layers: refused, never dropped. Without a GPU: the native calls
are stubs of the right shapes, the rest is the operators' own path."""

from __future__ import annotations

import types

import pytest
import torch
from torch.autograd import forward_ad

import torchure_amd as ta
from torchure_amd import _native, linear

BF16 = torch.bfloat16


@pytest.fixture
def stubs(monkeypatch):
    def lin_forward(x, weight, bias, residual, act, kind, keep_x, keep_z, keep_w, stream):
        return (x.new_zeros(*x.shape[:-1], weight.shape[0]), *(None,) * 5)

    def mlp_forward(x, w_gate, w_up, w_down, residual, kind, keep_x, keep_z, keep_in, keep_down, stream):
        return (x.new_zeros(*x.shape[:-1], w_down.shape[0]), *(None,) * 9)

    host = types.SimpleNamespace(lin_plain=lambda *a: False, lin_forward=lin_forward, mlp_forward=mlp_forward)
    monkeypatch.setattr(linear, "_on_gpu", lambda t, who, what: None)
    monkeypatch.setattr(_native, "lin_host", lambda: host)
    monkeypatch.setattr(_native, "stream_handle", lambda device: 0)


def ones(*shape):
    return torch.ones(shape, dtype=BF16)


CALLS = {"linear": (ta.fused_linear, lambda: [ones(3, 4), ones(5, 4), ones(5), ones(3, 5)]),
         "mlp": (ta.swiglu_mlp, lambda: [ones(3, 4), ones(6, 4), ones(6, 4), ones(5, 6), ones(3, 5)])}


@pytest.mark.parametrize("rows", [3, 0])
@pytest.mark.parametrize("grad", [True, False])
@pytest.mark.parametrize("name,at", [(n, i) for n, k in (("linear", 4), ("mlp", 5)) for i in range(k)])
def test_a_tangent_is_refused(stubs, name, at, grad, rows):
    call, make = CALLS[name]
    args = make()
    args[0], args[-1] = args[0][:rows], args[-1][:rows]
    with torch.set_grad_enabled(grad), forward_ad.dual_level():
        args[at] = forward_ad.make_dual(args[at], torch.ones_like(args[at]))
        with pytest.raises(NotImplementedError):
            call(*args)


@pytest.mark.parametrize("name", list(CALLS))
def test_without_tangents(stubs, name):
    """Inside a dual level, tensors that carry none take the direct call, or autograd's where one needs a gradient."""
    call, make = CALLS[name]
    with forward_ad.dual_level():
        assert call(*make()).grad_fn is None
        args = make()
        args[1].requires_grad_()
        y = call(*args)
        assert y.grad_fn is not None and forward_ad.unpack_dual(y).tangent is None
