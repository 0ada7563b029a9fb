"""AdamW on 8-bit moments: states that checkpoints bring along and that are not what they look like."""

from __future__ import annotations

import copy

import pytest
import torch

import torchure_amd as ta
from torchure_amd.optimizer.adamw import held_bytes

pytestmark = pytest.mark.gpu

DEV = "cuda"


def optimizer(n, bits, steps=0):
    p = torch.nn.Parameter(torch.linspace(-1.0, 1.0, n, device=DEV))
    opt = ta.AdamW([p], lr=1e-3, state_bits=bits, seed=3)
    for k in range(steps):
        p.grad = torch.cos(torch.arange(n, device=DEV) + k)
        opt.step()
    p.grad = torch.ones_like(p)
    return p, opt


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("n", [193, 256, 400, 512])
def test_values_as_many_as_a_params_bytes(n, bits):
    """A 32-bit checkpoint of a tensor whose elements are as many as this param's 8-bit moments have bytes is
    another tensor's, and is refused."""
    _, other = optimizer(held_bytes(n), 32, steps=2)
    p, opt = optimizer(n, bits)
    before = p.detach().clone()
    opt.load_state_dict(copy.deepcopy(other.state_dict()))
    with pytest.raises(RuntimeError, match="elements"):
        opt.step()
    assert torch.equal(p, before)


@pytest.mark.parametrize("bits", [32, 8])
def test_bytes_that_a_hook_puts_in(bits):
    """What counts is what the loader gets, behind the program's own hooks."""
    p, opt = optimizer(300, 8, steps=3)
    saved = copy.deepcopy(opt.state_dict())
    q, other = optimizer(300, bits)
    other.register_load_state_dict_pre_hook(lambda _, __: copy.deepcopy(saved))
    empty = copy.deepcopy(saved)
    empty["state"] = {}
    other.load_state_dict(empty)
    held, wide = opt.state[p], other.state[q]
    if bits == 8:
        assert torch.equal(held["exp_avg"], wide["exp_avg"]) and torch.equal(held["exp_avg_sq"], wide["exp_avg_sq"])
    else:
        assert torch.equal(opt.flat_moments()[0].float(), wide["exp_avg"])
        assert torch.equal(opt.flat_moments()[1].float().square(), wide["exp_avg_sq"])
    other.step()
    assert len(other._optimizer_load_state_dict_pre_hooks) == 1  # the program's


def test_negative_zeros():
    """A second moment of -0.0 is zero, and stays its own element's."""
    n = 520
    v = torch.linspace(0.1, 1.0, n, device=DEV).square_()
    v[::3] = 0.0
    p, opt = optimizer(n, 8)
    state = {"step": torch.tensor(1.0), "exp_avg": torch.zeros(n, device=DEV)}
    saved = opt.state_dict()
    held = []
    for zero in (0.0, -0.0):
        values = torch.where(v == 0.0, torch.full_like(v, zero), v)
        saved["state"] = {0: {**state, "exp_avg_sq": values}}
        opt.load_state_dict(copy.deepcopy(saved))
        held.append(opt.state[p]["exp_avg_sq"].clone())
        _, root = opt.flat_moments()
        assert not root[::3].any() and not torch.signbit(root).any()
    assert torch.equal(*held)
