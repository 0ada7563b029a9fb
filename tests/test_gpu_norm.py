"""Layer norm and RMS norm against the same formulas in 64 bits, and as programs call them: sizes that take every shape of the
kernels, layouts, types, partial gradients, special values, streams, graphs.

The bounds (``want``) count roundings: a sum over a row is at most ``SUM`` additions deep in any lane (64 elements of a lane, 6 steps
over lanes, 8 waves, the scaling), each of 2^-24 of the sum of magnitudes; a sum over rows as deep as there are rows."""

from __future__ import annotations

import math

import pytest
import torch

import torchure_amd as ta
from torchure_amd import _native

pytestmark = pytest.mark.gpu

DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
U = 2.0 ** -24
SUM = 80


def formula(x, w, b, layer, eps):
    """y of 64-bit tensors, by elementary operations (differentiable)."""
    if layer:
        x = x - x.mean(-1, keepdim=True)
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w
    return y if b is None else y + b


def want(t, dy, layer, eps, out):
    """{name: (value, bound)} of y and the gradients, in 64 bits."""
    x, w, b = (None if t[k] is None else t[k].double() for k in ("x", "weight", "bias"))
    d = x.shape[-1]
    one = torch.ones(d, dtype=torch.float64, device=x.device) if w is None else w
    mean = x.mean(-1, keepdim=True) if layer else torch.zeros_like(x[..., :1])
    c = x - mean
    rstd = 1 / torch.sqrt((c * c).mean(-1, keepdim=True) + eps)
    xhat = c * rstd
    e_mean = SUM * U * x.abs().mean(-1, keepdim=True) if layer else 0 * mean
    e_rel = (SUM + 8) * U / 2 + 3 * U + (e_mean * rstd) ** 2
    e_hat = (e_mean + U * c.abs()) * rstd + xhat.abs() * (e_rel + U)
    y = xhat * one + (0 if b is None else b)
    e = e_hat * one.abs() + U * (xhat * one).abs() + U * y.abs()
    found = {"y": (y, e + HALF[out] * (y.abs() + e))}
    if dy is None:
        return found
    dy = dy.double()
    g = dy * one
    along = (g * xhat).mean(-1, keepdim=True)
    e_along = (g.abs() * e_hat).mean(-1, keepdim=True) + (SUM + 3) * U * (g * xhat).abs().mean(-1, keepdim=True)
    mid = g.mean(-1, keepdim=True) if layer else 0 * along
    e_mid = SUM * U * g.abs().mean(-1, keepdim=True) if layer else 0
    inner = g - mid - along * xhat
    e = (e_along * xhat.abs() + along.abs() * e_hat + e_mid + 3 * U * (g.abs() + along.abs() * xhat.abs() + mid.abs())) * rstd
    e = e + (inner * rstd).abs() * (e_rel + U)
    found["x"] = (inner * rstd, e + HALF[t["x"].dtype] * ((inner * rstd).abs() + e))
    rows = x.numel() // d
    flat = lambda v: v.reshape(rows, d)  # noqa: E731
    s = flat(dy * xhat).sum(0)
    e = flat(dy.abs() * e_hat).sum(0) + (rows + 2) * U * flat((dy * xhat).abs()).sum(0)
    if t["weight"] is not None:
        found["weight"] = (s, e + HALF[t["weight"].dtype] * (s.abs() + e))
    if t["bias"] is not None:
        s, e = flat(dy).sum(0), (rows + 2) * U * flat(dy.abs()).sum(0)
        found["bias"] = (s, e + HALF[t["bias"].dtype] * (s.abs() + e))
    return found


def call(t, layer, eps=1e-5, dtype=None):
    if layer:
        return ta.layer_norm(t["x"], t["weight"], t["bias"], eps, dtype)
    return ta.rms_norm(t["x"], t["weight"], eps, dtype)


def case(shape, layer, x=BF16, w=BF16, b=BF16, out=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + sum(shape))
    r = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    d = shape[-1]
    t = {"x": (r(*shape) * torch.exp(0.5 * r(d)) + 0.3 * r(d)).to(x), "weight": None if w is None else (1 + 0.2 * r(d)).to(w),
         "bias": (0.1 * r(d)).to(b) if b is not None and layer else None}
    return {k: v if v is None else v.requires_grad_() for k, v in t.items()}, r(*shape).to(out or x)


def close(got, value, bound, what):
    got = got.detach().double()
    assert got.shape == value.shape, what
    bad = ~((got - value.detach()).abs() <= bound.detach())
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - value).abs().max()):.3g}"


def check(t, dy, layer, eps=1e-5, out=None):
    y = call(t, layer, eps, out)
    assert y.dtype == dy.dtype and y.shape == t["x"].shape
    w = want(t, dy, layer, eps, y.dtype)
    close(y, *w["y"], "y")
    with torch.no_grad():
        same(call(t, layer, eps, out), y, "without gradients")
    keys = [k for k in t if t[k] is not None]
    grads = dict(zip(keys, torch.autograd.grad(y, [t[k] for k in keys], dy)))
    for k, v in grads.items():
        assert v.dtype == t[k].dtype
        close(v, *w[k], "gradient of " + k)
    return y, grads


def same(a, b, what=""):
    assert a.dtype == b.dtype and a.shape == b.shape, what
    kind = torch.int16 if a.dtype == BF16 else torch.int32
    assert torch.equal(a.detach().contiguous().view(kind), b.detach().contiguous().view(kind)), what


WIDTHS = [1, 2, 7, 8, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 256, 257, 500, 512, 513, 777, 1024, 1237, 1536, 1800, 2048, 2560,
          2816, 4000, 4096, 4097, 5000, 6144, 8000, 8192, 9728, 12000, 16383, 16384]


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("cols", WIDTHS)
def test_widths(cols, layer):
    for rows, x, out in ((1, BF16, BF16), (5, BF16, BF16), (37, F32, BF16), (3, F32, F32), (6, BF16, F32)):
        t, dy = case((rows, cols), layer, x, F32 if rows == 37 else BF16, out=out)
        check(t, dy, layer, out=out)


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("rows,cols", [(70_000, 24), (40_001, 128), (9000, 333), (5003, 1024), (2600, 2560), (1100, 4100), (700, 9000),
                                       (600, 16384)])
def test_more_rows_than_the_grid(rows, cols, layer):
    for x in (BF16, F32):
        t, dy = case((rows, cols), layer, x, F32)
        y, grads = check(t, dy, layer)
        again, twice = check(t, dy, layer)
        same(y, again)
        for k in grads:
            same(grads[k], twice[k], "two runs: " + k)


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("w,b", [(None, None), (F32, None), (None, F32), (BF16, F32), (F32, BF16)])
def test_weights(w, b, layer):
    t, dy = case((33, 500), layer, BF16, w, b)
    check(t, dy, layer)


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("x", [BF16, F32])
def test_layouts(x, layer):
    t, dy = case((60, 200), layer, x)
    y, grads = check(t, dy, layer)
    room = torch.full((64, 333), float("nan"), dtype=x, device=DEV)
    views = [room[2:62, 3:203], torch.empty(120, 200, dtype=x, device=DEV)[::2], torch.empty(200, 60, dtype=x, device=DEV).t(),
             torch.empty(60, 400, dtype=x, device=DEV)[:, ::2], torch.empty(60 * 200 + 1, dtype=x, device=DEV)[1:].view(60, 200)]
    for v in views:
        with torch.no_grad():
            v.copy_(t["x"])
        u = {**t, "x": v.detach().requires_grad_()}
        z = call(u, layer)
        same(y, z)
        back = torch.empty(200, 60, dtype=x, device=DEV).t().copy_(dy)
        keys = list(grads)
        for k, got in zip(keys, torch.autograd.grad(z, [u[k] for k in keys], back)):
            same(grads[k], got, k)
    wide = torch.zeros(400, dtype=BF16, device=DEV)[::2].copy_(t["weight"].detach())
    same(call({**t, "weight": wide}, layer), y)
    odd = torch.zeros(201, dtype=BF16, device=DEV)[1:].copy_(t["weight"].detach())
    same(call({**t, "weight": odd}, layer), y)


@pytest.mark.parametrize("layer", [True, False])
def test_dimensions_and_broadcast_gradients(layer):
    t, dy = case((24, 40), layer)
    y, grads = check(t, dy, layer)
    cube = {**t, "x": t["x"].detach().view(2, 3, 4, 40).requires_grad_()}
    z = call(cube, layer)
    assert z.shape == (2, 3, 4, 40)
    same(z.reshape(24, 40), y)
    got, = torch.autograd.grad(z, cube["x"], dy.view(2, 3, 4, 40))
    assert got.shape == cube["x"].shape
    same(got.reshape(24, 40), grads["x"])
    heads = torch.randn(2, 5, 3, 40, device=DEV).to(BF16).transpose(1, 2)  # (batch, head, token, 40), strided
    same(call({**t, "x": heads}, layer), call({**t, "x": heads.contiguous()}, layer))
    same(call({**t, "x": t["x"][7]}, layer), y[7])
    a = torch.autograd.grad(call(t, layer).sum(), [t["x"], t["weight"]])
    b = torch.autograd.grad(call(t, layer), [t["x"], t["weight"]], torch.ones_like(dy))
    for p, q in zip(a, b):
        same(p, q)
    one = t["x"].detach()[:1].requires_grad_()  # one row for all: its gradient is the rows' sum
    got, = torch.autograd.grad(call({**t, "x": one.expand(24, 40)}, layer), one, dy)
    parts, = torch.autograd.grad(call({**t, "x": (many := one.detach().expand(24, 40).contiguous().requires_grad_())}, layer), many, dy)
    assert bool(((got.double() - parts.double().sum(0, keepdim=True)).abs() <= 30 * 2.0 ** -8 * parts.double().abs().sum(0)).all())


@pytest.mark.parametrize("layer", [True, False])
def test_some_gradients(layer):
    t, dy = case((50, 300), layer)
    _, every = check(t, dy, layer)
    names = list(every)
    for bits in range(1, 1 << len(names)):
        keys = [k for i, k in enumerate(names) if bits >> i & 1]
        some = {k: v if v is None else v.detach().requires_grad_(k in keys) for k, v in t.items()}
        for k, got in zip(keys, torch.autograd.grad(call(some, layer), [some[k] for k in keys], dy)):
            same(got, every[k], f"{keys}: {k}")


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("cols", [40, 1000, 5000])
def test_against_differences(cols, layer):
    """The gradients along random directions against central differences of the formula in 64 bits: off by the bounds along the
    direction, and 1e-6 of the terms for the third derivative at steps of 1e-4."""
    t, dy = case((6, cols), layer, F32, F32, F32)
    _, grads = check(t, dy, layer)
    w = want(t, dy, layer, 1e-5, F32)
    base = {k: None if v is None else v.detach().double() for k, v in t.items()}
    for k, got in grads.items():
        v = torch.randn_like(base[k])
        up, down = ({**base, k: base[k] + s * v} for s in (1e-4, -1e-4))
        f = lambda a: float((formula(a["x"], a["weight"], a["bias"], layer, 1e-5) * dy.double()).sum())  # noqa: E731
        numeric = (f(up) - f(down)) / 2e-4
        along = float((got.double() * v).sum())
        terms = float((w[k][0] * v).abs().sum())
        assert abs(numeric - along) <= float((w[k][1] * v.abs()).sum()) + 1e-6 * terms, k


# ---------------------------------------------------------------------------- special values


@pytest.mark.parametrize("cols", [33, 1024, 5000])
def test_far_from_zero(cols):
    """A mean a thousand times the spread: distances are taken before they are squared."""
    t, dy = case((9, cols), True, F32, F32)
    with torch.no_grad():
        t["x"] += 1000.0
    check(t, dy, True)


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("size", [1e-30, 1e-18, 1e15, 1e17])
def test_small_and_large_values(size, layer):
    """(300 squares of values about 1.2e18 would be 4.3e38, past fp32's 3.4e38.)"""
    t, dy = case((9, 300), layer, F32, F32)
    t["x"] = (t["x"].detach() * size).requires_grad_()
    if size < 1:  # eps decides: the squares vanish beside it
        check(t, dy, layer, 1e-5)
    else:
        check(t, dy, layer, 0.0)


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("cols", [16, 1024, 6000])
def test_constant_and_zero_rows(cols, layer):
    t, dy = case((7, cols), layer, F32, F32)
    with torch.no_grad():
        t["x"][2], t["x"][4] = 0.0, 3.0
    check(t, dy, layer)
    if cols == 1024:
        with torch.no_grad():
            y = call(t, layer, 0.0)
        assert torch.isnan(y[2]).all() and torch.isfinite(y[[0, 1, 3, 5, 6]]).all()


@pytest.mark.parametrize("layer", [True, False])
@pytest.mark.parametrize("cols", [24, 128, 1024, 6000])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_bad_rows_stay_alone(bad, cols, layer):
    t, dy = case((40, cols), layer)
    y, grads = check(t, dy, layer)
    u = {**t, "x": t["x"].detach().clone()}
    u["x"][17, cols // 2] = bad
    u["x"].requires_grad_()
    z = call(u, layer)
    keep = torch.arange(40, device=DEV) != 17
    same(z[keep], y[keep])
    assert torch.isnan(z[17]).any() and not torch.isinf(z[17]).any()
    got, = torch.autograd.grad(z, u["x"], dy)
    same(got[keep], grads["x"][keep])
    assert torch.isnan(got[17]).any()


@pytest.mark.parametrize("layer", [True, False])
def test_no_rows(layer):
    t, _ = case((3, 40), layer)
    u = {**t, "x": torch.empty(2, 0, 40, dtype=BF16, device=DEV, requires_grad=True)}
    y = call(u, layer, dtype=F32)
    assert y.shape == (2, 0, 40) and y.dtype == F32
    keys = [k for k in u if u[k] is not None]
    for k, g in zip(keys, torch.autograd.grad(y.sum(), [u[k] for k in keys])):
        assert g.shape == u[k].shape and g.dtype == u[k].dtype and not g.any()


# ---------------------------------------------------------------------------- as programs call them


@pytest.mark.parametrize("layer", [True, False])
def test_autocast_changes_nothing(layer):
    t, dy = case((20, 300), layer, F32, F32)
    y, grads = check(t, dy, layer, out=None)
    with torch.autocast("cuda", dtype=BF16):
        z = call(t, layer)
    same(y, z)
    for k, g in zip(grads, torch.autograd.grad(z, [t[k] for k in grads], dy)):
        same(g, grads[k])


@pytest.mark.parametrize("layer", [True, False])
def test_once_and_in_reverse(layer):
    t, dy = case((5, 64), layer, F32, F32)
    y = call(t, layer)
    g, = torch.autograd.grad(y, t["x"], dy.requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|differentiat"):
        torch.autograd.grad(g.sum(), t["x"])
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            call({**t, "x": torch.autograd.forward_ad.make_dual(t["x"].detach(), torch.ones_like(t["x"]))}, layer)


def test_kept_tensors_are_guarded_and_may_move():
    t, dy = case((30, 200), True)
    _, grads = check(t, dy, True)
    with torch.autograd.graph.save_on_cpu():
        y = call(t, True)
    for k, g in zip(grads, torch.autograd.grad(y, [t[k] for k in grads], dy)):
        same(g, grads[k])
    x = t["x"].detach().clone().requires_grad_()
    h = x * 1
    y = call({**t, "x": h}, True)
    with torch.no_grad():
        h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward(dy)
    y = call(t, True)
    y += 1  # the result is its own


@pytest.mark.parametrize("layer", [True, False])
def test_more_elements_than_32_bits(layer):
    x = torch.zeros(1_100_000, 2048, dtype=BF16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(2)
    x[-300:] = torch.randn(300, 2048, generator=g, device=DEV).to(BF16)
    w = torch.randn(2048, generator=g, device=DEV)
    t = {"x": x, "weight": w, "bias": None}
    y = call(t, layer)
    same(y[-300:], call({**t, "x": x[-300:].clone()}, layer))
    assert not y[:-300].any()
    part = x[-300:].clone().requires_grad_()
    dy = torch.zeros_like(x)
    dy[-300:] = torch.randn(300, 2048, generator=g, device=DEV).to(BF16)
    dx, = torch.autograd.grad(call({**t, "x": x.requires_grad_()}, layer), x, dy)
    dp, = torch.autograd.grad(call({**t, "x": part}, layer), part, dy[-300:])
    same(dx[-300:], dp)


@pytest.mark.parametrize("layer", [True, False])
def test_another_stream(layer):
    t, dy = case((400, 1000), layer)
    y, grads = check(t, dy, layer)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s):
            z = call(t, layer)
            got = torch.autograd.grad(z, [t[k] for k in grads], dy)
        s.synchronize()
        same(y, z)
        for k, g in zip(grads, got):
            same(grads[k], g)


@pytest.mark.parametrize("layer", [True, False])
def test_graphs(layer):
    """Two captured passes, of forward and backward, replayed in turn with eager calls between."""
    cases = [case(s, layer, seed=i) for i, s in enumerate(((300, 1000), (5, 5000)))]
    keys = [k for k in cases[0][0] if cases[0][0][k] is not None]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for t, dy in cases:
        with torch.cuda.stream(side):
            torch.autograd.grad(call(t, layer), [t[k] for k in keys], dy)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = call(t, layer)
            grads = torch.autograd.grad(y, [t[k] for k in keys], dy)
        graphs.append(g)
        outs.append((y.detach(), grads))
        del y
    for k in range(3):
        with torch.no_grad():
            for t, dy in cases:
                t["x"].add_(0.25)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for (t, dy), (y, grads) in zip(cases, outs):
            z = call(t, layer)
            same(y, z, f"replay {k}")
            for a, b in zip(grads, torch.autograd.grad(z, [t[k] for k in keys], dy)):
                same(a, b, f"replay {k}")
            del z


def test_refused_by_the_library():
    """What passes Python's checks of types and shapes and cannot run comes back as an error."""
    t, _ = case((4, 64), True)
    with pytest.raises(RuntimeError, match="features"):
        ta.rms_norm(torch.zeros(2, 16385, device=DEV))
    with pytest.raises(RuntimeError, match="features"):
        ta.layer_norm(torch.zeros(2, 0, device=DEV))
    with pytest.raises(RuntimeError, match="weight of shape"):
        ta.rms_norm(t["x"], t["weight"][:1])
    with pytest.raises(NotImplementedError, match="float16"):
        ta.rms_norm(t["x"].half())
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ta.rms_norm(t["x"], t["weight"].cpu())
    with pytest.raises(NotImplementedError, match="dense"):
        ta.rms_norm(torch.eye(64, device=DEV).to_sparse())
    assert _native.layer_host().norm_plain(t["x"], t["weight"], t["bias"], 0)
