"""The products' larger tiles and split ones, with what is kept and what follows them: every kind of end on tiles of
each size, whole, at edges, and joined from parts, against the formulas in 64 bits by the bounds of
test_gpu_linear. Sizes are those for which the cost model takes the tile that a case names; short in the
dimensions that it allows to be. The 64 bits are computed on the GPU."""

from __future__ import annotations

import pytest
import torch

import test_gpu_linear as T
import torchure_amd as ta
from test_gpu_linear_calls import BF16, DEV, F32, linear_grads, mlp_grads, same
from torchure_amd import _native

pytestmark = pytest.mark.gpu


def two_to(e):
    """2^e in 64 bits, to the bit (a power function on the GPU may be off in its last place)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def e4m3_blocks(x):
    """T.e4m3_64 of a finite matrix, all blocks at once."""
    n, d = x.shape
    rows, cols = -(-n // 32) * 32, -(-d // 32) * 32
    b = torch.zeros(rows, cols, dtype=x.dtype, device=x.device)
    b[:n, :d] = x
    b = b.view(rows // 32, 32, cols // 32, 32)
    frac, ex = torch.frexp(b.abs().amax(dim=(1, 3), keepdim=True))  # 448 = 0.875 2^9
    e = (ex - 9 + (frac > 0.875).int()).clamp(-117, 119)
    v = (b * two_to(-e)).clamp(-448, 448)
    step = two_to((torch.frexp(v.abs())[1] - 1).clamp_min(-6) - 3)
    return (torch.round(v / step) * step * two_to(e)).view(rows, cols)[:n, :d]


@pytest.mark.parametrize("device", ["cpu", DEV])
def test_the_format_all_blocks_at_once(device):
    g = torch.Generator().manual_seed(40)
    x = torch.randn(70, 100, generator=g).double() * torch.exp2(torch.randint(-140, 120, (70, 100), generator=g).double())
    x[:32, :32] = 0
    x[:, 40:50] *= 2.0 ** -100
    x[33, 33] = 448.0 * 2.0 ** 119
    x[64:] = torch.randint(-2000, 2000, (6, 100), generator=g).double() * 2.0 ** -8  # ties among them
    assert torch.equal(e4m3_blocks(x.to(device)).cpu(), PLAIN(x))


PLAIN = T.e4m3_64


@pytest.fixture(autouse=True)
def all_blocks_at_once(monkeypatch):
    monkeypatch.setattr(T, "e4m3_64", e4m3_blocks)


def close(got, want, bound, what):
    got = got.detach().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max()):.3g}"


def to_gpu(t):
    return {k: None if v is None else v.to(DEV) for k, v in t.items()}


def leaves(t):
    return {k: None if v is None else v.detach().requires_grad_() for k, v in t.items()}


def in_parts(op, rows, inp, out):
    return _native.lib().tm_lin_workspace_bytes(op, rows, inp, out, 0) > 0


# the forward product's tile, and whether some of the tiles, or all, are in parts of K
LINEAR = [
    (300, 300, 64, "128 x 128"), (300, 1000, 300, "128 x 128, all in parts"),
    (512, 4096, 512, "128 x 128, all in parts"),
    (10_000, 64, 777, "192 x 256"), (300, 8192, 6000, "192 x 256, all in parts"),
    (2000, 100, 6000, "256 x 256"), (5000, 4096, 777, "256 x 256, all in parts"),
    (6144, 1000, 2700, "256 x 256, some in parts"), (2048, 128, 8192, "256 x 256, whole ones only"),
]


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("rows,inp,out,tile", LINEAR)
def test_linear(rows, inp, out, tile, checkpoint):
    assert in_parts(_native.TM_LIN_FORWARD, rows, inp, out) == ("parts" in tile)
    act, bias, res = ("silu", BF16, F32) if checkpoint else ("gelu_tanh", F32, BF16)
    t, dy = T.linear_case(rows, inp, out, act, bias, res, checkpoint, seed=rows + inp)
    t, dy = to_gpu(t), dy.to(DEV)
    want = T.linear_want(t, dy, act, checkpoint)
    y, grads = linear_grads(leaves(t), dy, act, checkpoint)
    close(y, *want["y"], "y")
    for k, got in grads.items():
        close(got, *want[k], "gradient of " + k)
    again, twice = linear_grads(leaves(t), dy, act, checkpoint)
    same(y, again)
    for k in grads:
        same(grads[k], twice[k], k)


# first the tile of the gate, then of its gradient
MLP = [
    (520, 320, 300, 64, "128 x 256, all in parts", "128 x 128"),
    (300, 256, 300, 100, "192 x 256, all in parts", "128 x 128, all in parts"),
    (1500, 4096, 2700, 64, "128 x 256, some in parts", "128 x 128"),
    (8192, 256, 2304, 64, "192 x 256, some in parts", "192 x 256"),
    (1000, 64, 6000, 64, "256 x 256", "128 x 128"),
    (6144, 4096, 300, 64, "256 x 256, all in parts", "128 x 128"),
    (3000, 1000, 2700, 100, "256 x 256, some in parts", "192 x 256"),
    (4100, 64, 4000, 100, "192 x 256", "128 x 128, some in parts"),
    (520, 100, 4000, 100, "128 x 256", "192 x 256, all in parts"),
    (10_000, 64, 777, 64, "192 x 256", "192 x 256"),
    (2000, 100, 6000, 100, "128 x 256", "192 x 256, some in parts"),
    (5000, 64, 777, 4096, "192 x 256", "256 x 256, all in parts"),
    (5000, 64, 2700, 1000, "192 x 256", "256 x 256"),
    (6144, 64, 2700, 1500, "192 x 256", "256 x 256, some in parts"),
]


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("rows,dim,ffn,out,gate,grad", MLP)
def test_mlp(rows, dim, ffn, out, gate, grad, checkpoint):
    assert in_parts(_native.TM_LIN_GATE, rows, dim, ffn) == ("parts" in gate)
    assert in_parts(_native.TM_LIN_GATE_GRAD, rows, ffn, out) == ("parts" in grad)
    res = F32 if checkpoint else BF16
    t, dy = T.mlp_case(rows, dim, ffn, out, res, seed=rows + ffn)
    t, dy = to_gpu(t), dy.to(DEV)
    want = T.mlp_want(t, dy, checkpoint)
    y, grads = mlp_grads(leaves(t), dy, checkpoint)
    close(y, *want["y"], "y")
    for k, got in grads.items():
        close(got, *want[k], "gradient of " + k)
    again, twice = mlp_grads(leaves(t), dy, checkpoint)
    same(y, again)
    for k in grads:
        same(grads[k], twice[k], k)
