"""The norms' backward pass where the sums over rows can be checked exactly, and what it keeps, reads and runs on."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import torchure_amd as ta

pytestmark = pytest.mark.gpu

DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32
U = 2.0 ** -24


def call(t, layer, eps=1e-5):
    if layer:
        return ta.layer_norm(t["x"], t["weight"], t["bias"], eps)
    return ta.rms_norm(t["x"], t["weight"], eps)


def whole(d):
    """Whether d times the fp32 reciprocal of d is 1: the mean of d equal numbers is then exact."""
    return np.float32(d) * (np.float32(1.0) / np.float32(d)) == np.float32(1.0)


# ---------------------------------------------------------------------------- sums over rows, exactly


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("x", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 24), (5, 1000), (1027, 64), (70_000, 24), (40_001, 128), (9001, 260), (9000, 334), (5003, 1024), (4099, 1500),
                                       (2600, 2560), (2049, 2800), (1100, 4100), (3001, 6144), (700, 9000), (600, 16384)])
def test_every_row_counts_once(rows, cols, layer, x):
    """Rows of 1 and -1, as many of each, have xhat of 1 and -1, and their products with small whole numbers have exact sums in
    any order: dw and db are those sums to the bit, whichever rows meet where."""
    assert whole(cols) and cols % 2 == 0
    g = torch.Generator(device=DEV).manual_seed(rows + cols)
    sign = torch.ones(cols, device=DEV)
    sign[torch.randperm(cols, generator=g, device=DEV)[: cols // 2]] = -1.0
    flip = torch.randint(0, 2, (rows, 1), generator=g, device=DEV) * 2.0 - 1.0
    t = {"x": (sign * flip).to(x), "weight": torch.ones(cols, device=DEV, requires_grad=True),
         "bias": torch.zeros(cols, device=DEV, requires_grad=True) if layer else None}
    dy = torch.randint(1, 8, (rows, cols), generator=g, device=DEV).to(x)  # (no two rows' cancel)
    y = call(t, layer, 0.0)
    assert torch.equal(y.float(), t["x"].float())
    keys = [k for k in ("weight", "bias") if t[k] is not None]
    got = dict(zip(keys, torch.autograd.grad(y, [t[k] for k in keys], dy)))
    assert torch.equal(got["weight"].double(), (dy.double() * t["x"].double()).sum(0))
    if layer:
        assert torch.equal(got["bias"].double(), dy.double().sum(0))


# ---------------------------------------------------------------------------- rows far from zero


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("cols", [1, 2, 4, 8, 16, 32])
def test_constant_rows_far_from_zero(cols, out):
    """A row of one large number has xhat of 0, and dx = (g - mean(g)) / sqrt(eps), also where mean times rstd is past
    fp32: what lies past a row's end has no part in it. (Of 2^k equal numbers the mean is exact in fp32.)"""
    eps = 1e-5
    g = torch.Generator(device=DEV).manual_seed(cols)
    x = torch.randn(7, cols, generator=g, device=DEV)
    x[2], x[5] = 2.0 ** 121, -(2.0 ** 121)
    t = {"x": x.to(out).requires_grad_(), "weight": torch.ones(cols, device=DEV, requires_grad=True),
         "bias": torch.zeros(cols, device=DEV, requires_grad=True)}
    dy = torch.randn(7, cols, generator=g, device=DEV).to(out)
    y = call(t, True, eps)
    assert not y[2].any() and not y[5].any()
    dx, dw, db = torch.autograd.grad(y, [t["x"], t["weight"], t["bias"]], dy)
    d = dy.double()
    for r in (2, 5):
        want = (d[r] - d[r].mean()) / eps ** 0.5
        # a sum at most 80 additions deep, its scaling, the difference; eps, its root and reciprocal; the product; the result
        bound = (84 * U * d[r].abs().mean() + U * (d[r] - d[r].mean()).abs()) / eps ** 0.5 + 5 * U * want.abs()
        bound = bound + {BF16: 2.0 ** -8, F32: U}[out] * (want.abs() + bound)
        assert bool(((dx[r].double() - want).abs() <= bound).all()), r
    keep = torch.tensor([0, 1, 3, 4, 6], device=DEV)
    rest = {"x": t["x"].detach()[keep].requires_grad_(), "weight": t["weight"], "bias": t["bias"]}
    same, part, _ = torch.autograd.grad(call(rest, True, eps), [rest["x"], t["weight"], t["bias"]], dy[keep])
    assert torch.equal(dx[keep], same) and bool(torch.isfinite(dw).all())


# ---------------------------------------------------------------------------- what is kept


@pytest.mark.parametrize("layer", [True, False])
def test_kept_for_what_is_wanted(layer):
    g = torch.Generator(device=DEV).manual_seed(1)
    rows, cols = 37, 200
    values = {"x": torch.randn(rows, cols, generator=g, device=DEV).to(BF16), "weight": torch.randn(cols, generator=g, device=DEV),
              "bias": torch.randn(cols, generator=g, device=DEV) if layer else None}
    dy = torch.randn(rows, cols, generator=g, device=DEV).to(BF16)
    names = [k for k, v in values.items() if v is not None]
    every = {k: v if v is None else v.clone().requires_grad_() for k, v in values.items()}
    full = dict(zip(names, torch.autograd.grad(call(every, layer), [every[k] for k in names], dy)))
    stats = (2 if layer else 1, rows)
    for bits in range(1, 1 << len(names)):
        keys = [k for i, k in enumerate(names) if bits >> i & 1]
        t = {k: v if v is None else v.clone().requires_grad_(k in keys) for k, v in values.items()}
        kept = []
        with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(tuple(v.shape)) or v, lambda v: v):
            y = call(t, layer)
        want = []
        if "x" in keys or "weight" in keys:
            want += [(rows, cols), stats]
        if "x" in keys:
            want.append((cols,))
        assert sorted(kept) == sorted(want), (keys, kept)
        with torch.no_grad():  # what is not kept may change
            for k, needed in (("x", "x" in keys or "weight" in keys), ("weight", "x" in keys), ("bias", False)):
                if t[k] is not None and not needed:
                    t[k].add_(1.0)
        for k, got in zip(keys, torch.autograd.grad(y, [t[k] for k in keys], dy)):
            assert got.dtype == values[k].dtype and torch.equal(got, full[k]), (keys, k)


# ---------------------------------------------------------------------------- streams


def beside():
    """A stream whose work runs beside the current one's (streams share the few hardware queues)."""
    for _ in range(8):
        s, done = torch.cuda.Stream(), torch.cuda.Event()
        torch.cuda._sleep(20_000_000)  # a bounded spin
        done.record()
        with torch.cuda.stream(s):
            torch.ones(1, device=DEV)
        s.synchronize()
        free = not done.query()
        torch.cuda.synchronize()
        if free:
            return s
    pytest.skip("no stream runs beside the current one")


@pytest.mark.parametrize("layer", [True, False])
def test_node_called_on_another_stream(layer):
    """A node that is called directly runs where it is called, not where its forward pass ran."""
    g = torch.Generator(device=DEV).manual_seed(2)
    t = {"x": torch.randn(400, 1000, generator=g, device=DEV).requires_grad_(), "weight": torch.randn(1000, generator=g, device=DEV).requires_grad_(),
         "bias": torch.randn(1000, generator=g, device=DEV).requires_grad_() if layer else None}
    dy = torch.randn(400, 1000, generator=g, device=DEV)
    keys = [k for k in t if t[k] is not None]
    want = torch.autograd.grad(call(t, layer), [t[k] for k in keys], dy)
    y = call(t, layer)
    torch.cuda.synchronize()
    s = beside()
    with torch.cuda.stream(s):
        spoilt = [torch.full_like(w, float("nan")) for w in want]
    s.synchronize()
    del spoilt  # (its blocks are the results')
    torch.cuda._sleep(100_000_000)  # the forward pass's stream is busy
    with torch.no_grad(), torch.cuda.stream(s):
        got = [v.clone() for v in y.grad_fn(dy)[: len(keys)]]
    s.synchronize()
    for k, a, b in zip(keys, want, got):
        assert torch.equal(a, b), k
    torch.cuda.synchronize()
