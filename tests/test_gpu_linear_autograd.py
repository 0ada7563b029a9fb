"""The linear layers and the gated feed-forward among a program's other tensors: results that are changed in
place afterwards. Bit for bit against the same calls without that."""

from __future__ import annotations

import pytest
import torch

import test_gpu_linear as T
import torchure_amd as ta
from test_gpu_linear_calls import BF16, DEV, F32, on_device, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (2, 1, 3)])
def test_results_changed_in_place(lead, checkpoint):
    """y.mul_(2).add_(r) gives y's gradients twice, for any number of dimensions."""
    rows = torch.Size(lead).numel()
    t, dy = T.linear_case(rows, 40, 48, "silu", BF16, F32, checkpoint, seed=30)
    m, mdy = T.mlp_case(rows, 40, 56, 48, None, seed=30)
    for call, args, dy in ((lambda x, w, b, r: ta.fused_linear(x, w, b, r, "silu", checkpoint), on_device(t), dy),
                           (lambda x, *w: ta.swiglu_mlp(x, *w[:3], None, checkpoint), on_device(m), mdy)):
        args = {k: v if v is None or k not in ("x", "residual") else v.detach().view(*lead, v.shape[-1]).requires_grad_()
                for k, v in args.items()}
        wanted = [v for v in args.values() if v is not None]
        dy = dy.to(DEV).view(*lead, 48)
        y = call(*args.values())
        want = torch.autograd.grad(y, wanted, 2 * dy)
        z = call(*args.values())
        assert not z._is_view()
        z.mul_(2).add_(dy)
        same(z, (y.detach() * 2).add_(dy))
        for a, b in zip(torch.autograd.grad(z, wanted, dy), want):
            same(a, b)
