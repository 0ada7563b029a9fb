"""The linear layers, the gated feed-forward and the 8-bit activations as programs call them: sizes that
take every tile, split and path, layouts, types under autocast, partial gradients, streams, graphs,
special values, and a block of them trained together. Where two calls must give the same bits, they
are compared bit for bit; against 64 bits, by the bounds of test_gpu_linear."""

from __future__ import annotations

import pytest
import torch

import test_gpu_linear as T
import torchure_amd as ta
from torchure_amd.loss.fused_linear_ce import fused_linear_cross_entropy

pytestmark = pytest.mark.gpu

DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32


def on_device(t):
    return {k: None if v is None else v.to(DEV).requires_grad_() for k, v in t.items()}


def same(a, b, what=""):
    """Bit for bit, NaN included."""
    assert a.dtype == b.dtype and a.shape == b.shape, what
    kind = torch.int16 if a.dtype == BF16 else torch.int32
    assert torch.equal(a.detach().contiguous().view(kind), b.detach().contiguous().view(kind)), what


def linear_grads(t, dy, act=None, checkpoint=None, keys=None):
    y = ta.fused_linear(t["x"], t["weight"], t.get("bias"), t.get("residual"), act, checkpoint)
    keys = keys or [k for k in t if t[k] is not None]
    return y, dict(zip(keys, torch.autograd.grad(y, [t[k] for k in keys], dy)))


def mlp_grads(t, dy, checkpoint=None, keys=None):
    y = ta.swiglu_mlp(t["x"], t["w_gate"], t["w_up"], t["w_down"], t.get("residual"), checkpoint)
    keys = keys or [k for k in t if t[k] is not None]
    return y, dict(zip(keys, torch.autograd.grad(y, [t[k] for k in keys], dy)))


# ---------------------------------------------------------------------------- sizes


@pytest.mark.parametrize("rows,inp,out,act,bias,res", [
    (4096, 256, 4096, None, None, None),  # whole rounds of 256 x 256 tiles
    (2304, 512, 2304, "silu", torch.bfloat16, None),
    (6144, 320, 2000, "gelu", None, torch.float32),  # a last round of tiles, edges on one side
    (3001, 1001, 1237, "gelu_tanh", torch.float32, torch.bfloat16),  # every row unaligned, K ragged
    (300, 6000, 260, None, None, torch.bfloat16),  # long K, few tiles
    (6001, 200, 300, "relu", torch.bfloat16, torch.float32),  # the same for the weight's gradient
    (16, 4864, 640, None, None, torch.float32), (17, 1536, 4096, "silu", torch.float32, None),  # few rows
    (64, 1536, 1000, "gelu", torch.bfloat16, torch.bfloat16), (65, 1024, 2048, None, None, None),
])
def test_linear_sizes(rows, inp, out, act, bias, res):
    t, dy = T.linear_case(rows, inp, out, act, bias, res, None, seed=rows)
    want = T.linear_want(t, dy, act, None)
    y, grads = linear_grads(on_device(t), dy.to(DEV), act)
    T.close(y, *want["y"], "y")
    for k, got in grads.items():
        T.close(got, *want[k], "gradient of " + k)
    again, twice = linear_grads(on_device(t), dy.to(DEV), act)
    same(y, again, "y of two runs")
    for k in grads:
        same(grads[k], twice[k], "two runs: " + k)


@pytest.mark.parametrize("rows,dim,ffn,out,res", [
    (2100, 512, 1400, 520, torch.float32), (4096, 256, 2048, 256, torch.bfloat16), (1999, 333, 777, 401, None),
    (6200, 96, 640, 96, None), (40, 1024, 1024, 512, torch.float32)])
def test_mlp_sizes(rows, dim, ffn, out, res):
    t, dy = T.mlp_case(rows, dim, ffn, out, res, seed=rows)
    want = T.mlp_want(t, dy, None)
    y, grads = mlp_grads(on_device(t), dy.to(DEV))
    T.close(y, *want["y"], "y")
    for k, got in grads.items():
        T.close(got, *want[k], "gradient of " + k)
    again, twice = mlp_grads(on_device(t), dy.to(DEV))
    same(y, again)
    for k in grads:
        same(grads[k], twice[k], "two runs: " + k)


@pytest.mark.parametrize("rows", [1, 7, 16, 17, 32, 33, 64])
@pytest.mark.parametrize("inp,out,act,bias,res", [
    (64, 16, None, None, None), (72, 33, "silu", torch.bfloat16, torch.float32), (1000, 9, "gelu", torch.float32, None),
    (2816, 1024, None, None, torch.bfloat16), (4864, 47, "relu", None, torch.float32), (136, 8200, "gelu_tanh", None, None),
    (9, 15, None, torch.bfloat16, torch.bfloat16)])
def test_few_rows_without_gradients(rows, inp, out, act, bias, res):
    """The forms for single tokens and short ends: every width of a workgroup's columns, to the last and past it."""
    t, dy = T.linear_case(rows, inp, out, act, bias, res, None, seed=rows + out)
    want = T.linear_want(t, dy, act, None)["y"]
    with torch.no_grad():
        d = {k: None if v is None else v.to(DEV) for k, v in t.items()}
        T.close(ta.fused_linear(d["x"], d["weight"], d["bias"], d["residual"], act), *want, "y")


@pytest.mark.parametrize("rows", [1, 16, 17, 33, 64])
@pytest.mark.parametrize("dim,ffn,out", [(64, 16, 40), (72, 47, 33), (1024, 2816, 1024), (2560, 520, 96), (24, 8200, 24)])
def test_few_rows_of_the_feed_forward_without_gradients(rows, dim, ffn, out):
    t, dy = T.mlp_case(rows, dim, ffn, out, torch.bfloat16, seed=rows + ffn)
    want = T.mlp_want(t, dy, None)["y"]
    with torch.no_grad():
        y = ta.swiglu_mlp(*(t[k].to(DEV) for k in ("x", "w_gate", "w_up", "w_down", "residual")))
    T.close(y, *want, "y")


@pytest.mark.parametrize("rows,inp,out", [(2304, 512, 2304), (3001, 333, 1237)])
def test_8_bit_gradients_are_those_of_what_is_held(rows, inp, out):
    """With no activation the weight's gradient reads x as held: the same bits as a call on the held x."""
    t, dy = T.linear_case(rows, inp, out, None, None, None, "e4m3", seed=1)
    t["x"] = torch.randn(rows, inp).to(BF16)
    d, dy = on_device(t), dy.to(DEV)
    y, grads = linear_grads(d, dy, checkpoint="e4m3")
    same(y, linear_grads(d, dy)[0], "the forward result")
    held = ta.dequantize_activation(ta.quantize_activation(d["x"].detach())).requires_grad_()
    same(grads["weight"], linear_grads({**d, "x": held}, dy)[1]["weight"])


def test_more_elements_than_32_bits():
    """Rows past 2^31 elements of x, of y and of what is held in 8 bits equal a small call on them."""
    g = torch.Generator(device=DEV).manual_seed(0)
    w = torch.randint(-4, 5, (64, 8192), generator=g, device=DEV).to(BF16)
    x = torch.zeros(270_001, 8192, dtype=BF16, device=DEV)
    x[-300:] = torch.randint(-4, 5, (300, 8192), generator=g, device=DEV).to(BF16)
    y = ta.fused_linear(x, w)
    same(y[-300:], ta.fused_linear(x[-300:].clone(), w))
    assert not y[:-300].any()
    q = ta.quantize_activation(x)
    back = ta.dequantize_activation(q)
    same(back[-64:], x[-64:])  # small whole numbers: exact
    del q, back, x, y
    tall = torch.randint(-4, 5, (40_000, 64), generator=g, device=DEV).to(BF16)
    wide = torch.randint(-4, 5, (65_536, 64), generator=g, device=DEV).to(BF16)
    y = ta.fused_linear(tall, wide, activation="relu")
    same(y[-300:], ta.fused_linear(tall[-300:].clone(), wide, activation="relu"))


@pytest.mark.parametrize("rows,cols", [(10_000, 8192), (10_300, 8192), (81_000, 1037)])
def test_large_8_bit_matrices(rows, cols):
    """On both sides of the size from which bf16 matrices go past the caches, odd rows among them: as parts of
    the rows are held by themselves."""
    g = torch.Generator(device=DEV).manual_seed(26)
    x = torch.randn(rows, cols, generator=g, device=DEV).to(BF16)
    q = ta.quantize_activation(x)
    back, wide = ta.dequantize_activation(q), ta.dequantize_activation(q, F32)
    assert torch.equal(back.float(), wide)
    for at in (0, 32 * (rows // 64), 32 * (rows // 32) - 64):
        part = x[at: at + 96] if at + 96 > rows else x[at: at + 64]
        p = ta.quantize_activation(part.contiguous())
        n = part.shape[0]
        assert torch.equal(q.values[at: at + n], p.values)
        assert torch.equal(q.exponents[at // 32: at // 32 + p.exponents.shape[0]], p.exponents)
        same(back[at: at + n], ta.dequantize_activation(p))


# ---------------------------------------------------------------------------- layouts, types


def _views():
    """The same 60 x 72 values in other places and orders."""
    g = torch.Generator().manual_seed(3)
    x = T.grid_values(g, (60, 72), 0.25, 6).to(DEV)
    room = torch.full((64, 200), float("nan"), dtype=BF16, device=DEV)
    yield "contiguous", x
    for name, v in (("a slice at an odd element", room[2:62, 3:75]), ("every second row", room.new_zeros(120, 72)[::2]),
                    ("transposed", room.new_zeros(72, 60).t()), ("every second column", room.new_zeros(60, 144)[:, ::2])):
        v.copy_(x)
        yield name, v
    far = torch.zeros(2, (1 << 23) + 8, dtype=BF16, device=DEV)
    v = far.as_strided((2, 72), (1 << 23, 1))
    v.copy_(x[:2])
    yield "rows 2^23 elements apart", v


def test_layouts():
    g = torch.Generator().manual_seed(4)
    w, b = T.grid_values(g, (50, 72), 2.0 ** -6, 12).to(DEV), T.grid_values(g, (50,), 2.0 ** -7, 20).to(DEV)
    views = dict(_views())
    for name, v in views.items():
        base = views["contiguous"][: v.shape[0]].clone().requires_grad_()
        r = torch.randn(v.shape[0], 50, device=DEV)
        dy = torch.randn(v.shape[0], 50, device=DEV)
        x = v.detach().requires_grad_()
        for checkpoint in (None, "e4m3"):
            one, ones_ = linear_grads({"x": base, "weight": w.requires_grad_(), "bias": b.requires_grad_(), "residual": r.requires_grad_()}, dy, "silu", checkpoint)
            two, twos = linear_grads({"x": x, "weight": w, "bias": b, "residual": r}, dy, "silu", checkpoint)
            same(one, two, name)
            for k in ones_:
                same(ones_[k], twos[k], f"{name}: {k}")


def test_layouts_of_the_other_operands():
    t, dy = T.linear_case(70, 96, 80, "silu", BF16, BF16, None, seed=8)
    d, dy = on_device(t), dy.to(DEV)
    y, grads = linear_grads(d, dy, "silu")
    other = {k: torch.empty(tuple(n + 5 for n in v.shape), dtype=v.dtype, device=DEV)[tuple(slice(3, 3 + n) for n in v.shape)]
             for k, v in d.items()}
    other["weight"] = torch.empty(96, 80, dtype=BF16, device=DEV).t()
    for k in other:
        other[k].copy_(d[k].detach())
    other = {k: v.detach().requires_grad_() for k, v in other.items()}
    odd_dy = torch.empty(80, 70, dtype=BF16, device=DEV).t().copy_(dy)
    y2, grads2 = linear_grads(other, odd_dy, "silu")
    same(y, y2)
    for k in grads:
        same(grads[k], grads2[k], k)
    # one value for all of dy, as y.sum() makes it
    a = linear_grads(d, torch.ones((), dtype=BF16, device=DEV).expand(70, 80), "silu")[1]
    b = linear_grads(d, torch.ones(70, 80, dtype=BF16, device=DEV), "silu")[1]
    for k in a:
        same(a[k], b[k], k)
    # a residual that is one row for all
    row = torch.randn(80, device=DEV).to(BF16).requires_grad_()
    y = ta.fused_linear(d["x"], d["weight"], None, row.expand(70, 80))
    same(y, ta.fused_linear(d["x"], d["weight"], None, row.detach().expand(70, 80).contiguous()))
    got, = torch.autograd.grad(y, row, dy)
    T.close(got, dy.double().cpu().sum(0), dy.double().cpu().abs().sum(0) * (70 * 2.0 ** -24 + 2.0 ** -8), "residual")


def test_mlp_layouts():
    t, dy = T.mlp_case(50, 40, 77, 60, BF16, seed=9)
    d, dy = on_device(t), dy.to(DEV)
    y, grads = mlp_grads(d, dy, "e4m3")
    other = {k: torch.empty(v.shape[::-1], dtype=v.dtype, device=DEV).t().copy_(v.detach()).requires_grad_() for k, v in d.items()}
    y2, grads2 = mlp_grads(other, dy.t().contiguous().t(), "e4m3")
    same(y, y2)
    for k in grads:
        same(grads[k], grads2[k], k)


def test_dimensions():
    t, dy = T.linear_case(24, 40, 48, "gelu", BF16, F32, None, seed=2)
    d, dy = on_device(t), dy.to(DEV)
    y, grads = linear_grads(d, dy, "gelu")
    cube = {**d, "x": d["x"].detach().view(2, 3, 4, 40).requires_grad_(),
            "residual": d["residual"].detach().view(2, 3, 4, 48).requires_grad_()}
    y4, grads4 = linear_grads(cube, dy.view(2, 3, 4, 48), "gelu")
    assert y4.shape == (2, 3, 4, 48)
    same(y, y4.reshape(24, 48))
    for k in grads:
        same(grads[k], grads4[k].reshape(grads[k].shape), k)
    one = ta.fused_linear(d["x"][5], d["weight"], d["bias"], d["residual"][5], "gelu")
    assert one.shape == (48,)
    same(one, ta.fused_linear(d["x"][5:6], d["weight"], d["bias"], d["residual"][5:6], "gelu")[0])
    m, mdy = T.mlp_case(6, 40, 56, 40, None, seed=2)
    m, mdy = on_device(m), mdy.to(DEV)
    y, grads = mlp_grads(m, mdy)
    y3, grads3 = mlp_grads({**m, "x": m["x"].detach().view(3, 2, 40).requires_grad_()}, mdy.view(3, 2, 40))
    same(y, y3.reshape(6, 40))
    for k in grads:
        same(grads[k], grads3[k].reshape(grads[k].shape), k)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("copies", [False, True])
def test_fp32_masters_under_autocast(checkpoint, copies):
    """fp32 hidden states and masters give the bits of their bf16 casts, with fp32 gradients whose
    rounding to bf16 is the bf16 call's."""
    g = torch.Generator().manual_seed(6)
    x32, w32, b32 = (torch.randn(s, generator=g).to(DEV).requires_grad_() for s in ((70, 96), (80, 96), (80,)))
    r32, dy = torch.randn(70, 80, generator=g).to(DEV).requires_grad_(), torch.randn(70, 80, generator=g).to(DEV)
    if copies:
        ta.attach_bf16_working_params([w32, b32])
    with torch.autocast("cuda", dtype=BF16):
        y, grads = linear_grads({"x": x32, "weight": w32, "bias": b32, "residual": r32}, dy, "silu", checkpoint)
    low = {k: v.detach().to(BF16).requires_grad_() for k, v in (("x", x32), ("weight", w32))}
    y2, grads2 = linear_grads({**low, "bias": b32, "residual": r32}, dy, "silu", checkpoint)
    assert y.dtype == F32
    same(y, y2)
    for k, v in grads.items():
        assert v.dtype == F32
        if checkpoint is None or k != "weight":  # whose 8 bits are made from the fp32 x
            same(v.to(grads2[k].dtype), grads2[k], k)


def test_mlp_fp32_masters_under_autocast():
    g = torch.Generator().manual_seed(7)
    d = {k: torch.randn(s, generator=g).mul(m).to(DEV).requires_grad_() for k, s, m in (
        ("x", (70, 96), 1.0), ("w_gate", (120, 96), 0.1), ("w_up", (120, 96), 0.1), ("w_down", (96, 120), 0.1),
        ("residual", (70, 96), 1.0))}
    dy = torch.randn(70, 96, generator=g).to(DEV)
    with torch.autocast("cuda", dtype=BF16):
        y, grads = mlp_grads(d, dy)
    low = {k: v if k == "residual" else v.detach().to(BF16).requires_grad_() for k, v in d.items()}
    y2, grads2 = mlp_grads(low, dy)
    same(y, y2)
    for k, v in grads.items():
        assert v.dtype == F32
        same(v.to(grads2[k].dtype), grads2[k], k)
    ta.attach_bf16_working_params([d["w_gate"], d["w_up"], d["w_down"]])
    with torch.autocast("cuda", dtype=BF16):
        y3, grads3 = mlp_grads(d, dy)
    same(y, y3)
    for k in grads:
        same(grads[k], grads3[k], k)
    with torch.no_grad():
        d["w_gate"].mul_(2.0)  # the copy is no longer the master's
    with torch.autocast("cuda", dtype=BF16):
        y4 = mlp_grads(d, dy)[0]
    same(y4, mlp_grads({**low, "w_gate": d["w_gate"].detach().to(BF16).requires_grad_()}, dy)[0])


# ---------------------------------------------------------------------------- autograd


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("act", [None, "silu"])
def test_some_gradients(act, checkpoint):
    t, dy = T.linear_case(70, 96, 80, act, BF16, F32, checkpoint, seed=11)
    d, dy = on_device(t), dy.to(DEV)
    _, every = linear_grads(d, dy, act, checkpoint)
    names = list(d)
    for bits in range(1, 16):
        keys = [k for i, k in enumerate(names) if bits >> i & 1]
        some = {k: v.detach().requires_grad_(k in keys) for k, v in d.items()}
        _, grads = linear_grads(some, dy, act, checkpoint, keys)
        for k in keys:
            same(grads[k], every[k], f"{keys}: {k}")


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_some_mlp_gradients(checkpoint):
    t, dy = T.mlp_case(50, 40, 72, 64, F32, seed=12)
    d, dy = on_device(t), dy.to(DEV)
    _, every = mlp_grads(d, dy, checkpoint)
    names = list(d)
    for bits in range(1, 32):
        keys = [k for i, k in enumerate(names) if bits >> i & 1]
        some = {k: v.detach().requires_grad_(k in keys) for k, v in d.items()}
        _, grads = mlp_grads(some, dy, checkpoint, keys)
        for k in keys:
            same(grads[k], every[k], f"{keys}: {k}")


def test_one_tensor_in_two_places():
    g = torch.Generator().manual_seed(13)
    w = T.grid_values(g, (64, 64), 2.0 ** -6, 12).to(DEV).requires_grad_()
    x = T.grid_values(g, (40, 64), 0.25, 6).to(DEV).requires_grad_()
    dy = torch.randn(40, 64, generator=g).to(BF16).to(DEV)
    y = ta.fused_linear(x, w, None, x, "silu")
    dx, = torch.autograd.grad(y, x, dy)
    parts = linear_grads({"x": x.detach().requires_grad_(), "weight": w, "residual": x.detach().requires_grad_()}, dy, "silu")[1]
    same(dx, parts["x"] + parts["residual"])
    y = ta.swiglu_mlp(x, w, w, w)
    dw, = torch.autograd.grad(y, w, dy)
    p = mlp_grads({"x": x, **{k: w.detach().requires_grad_() for k in ("w_gate", "w_up", "w_down")}}, dy)[1]
    T.close(dw, (p["w_gate"].double() + p["w_up"].double() + p["w_down"].double()).cpu(),
            sum(p[k].double().abs().cpu() for k in ("w_gate", "w_up", "w_down")) * 2.0 ** -7, "shared weight")


def test_no_second_derivative_and_changed_inputs():
    t, dy = T.linear_case(10, 16, 24, "silu", None, None, None, seed=14)
    d, dy = on_device(t), dy.to(DEV).requires_grad_()
    y = ta.fused_linear(d["x"], d["weight"], None, None, "silu")
    dx, = torch.autograd.grad(y, d["x"], dy, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|twice"):
        dx.sum().backward()
    x = d["x"].detach().clone()
    y = ta.fused_linear(x, d["weight"])
    x.add_(1)  # what the weight's gradient needs
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_no_rows():
    w = torch.ones(8, 16, dtype=BF16, device=DEV, requires_grad=True)
    for shape in ((0, 16), (3, 0, 16)):
        x = torch.ones(shape, dtype=BF16, device=DEV, requires_grad=True)
        r = torch.ones((*shape[:-1], 8), device=DEV, requires_grad=True)
        y = ta.fused_linear(x, w, None, r, "gelu", "e4m3")
        assert y.shape == (*shape[:-1], 8) and y.dtype == F32
        dx, dw, dr = torch.autograd.grad(y, (x, w, r), torch.ones_like(y))
        assert dx.shape == x.shape and dr.shape == r.shape and not dw.any()
        v = torch.ones(16, 8, dtype=BF16, device=DEV, requires_grad=True)
        y = ta.swiglu_mlp(x, w, w, v)
        assert y.shape == shape and y.dtype == BF16
        dx, dw, dv = torch.autograd.grad(y, (x, w, v), torch.ones_like(y))
        assert dx.shape == x.shape and not dw.any() and not dv.any()
    for shape in ((0,), (0, 5), (5, 0), (2, 0, 3)):
        x = torch.ones(shape, dtype=F32, device=DEV)
        back = ta.dequantize_activation(ta.quantize_activation(x))
        assert back.shape == x.shape and back.dtype == F32


def test_gradients_against_differences():
    """Central differences of the formulas in 64 bits (no rounding): the kernels' gradients are within
    bf16's roundings of dz (2^-8 of each), of what is held (2^-8 of z, times the slope's slope, at most 1 for
    these) and of the result; and the differences within h^2."""
    g = torch.Generator().manual_seed(15)
    t, dy = T.linear_case(6, 9, 7, "silu", BF16, F32, None, seed=15)
    _, grads = linear_grads(on_device(t), dy.to(DEV), "silu")
    h = 1e-5

    def loss(p):
        z = p["x"] @ p["weight"].t() + p["bias"]
        return ((T.act64("silu", z) + p["residual"]) * dy.double()).sum()

    def differences(p, k):
        out = torch.zeros_like(p[k])
        for i in range(out.numel()):
            v = p[k].view(-1)[i].item()
            p[k].view(-1)[i] = v + h
            up = loss(p)
            p[k].view(-1)[i] = v - h
            out.view(-1)[i] = (up - loss(p)) / (2 * h)
            p[k].view(-1)[i] = v
        return out

    p = {k: v.double() for k, v in t.items()}
    ad = dy.double().abs()
    z = (p["x"] @ p["weight"].t() + p["bias"]).abs()
    err = ad * (1.2 * 2.0 ** -8 + 2.0 ** -8 * z)  # |silu'| < 1.1
    bounds = {"x": err @ p["weight"].abs(), "weight": err.t() @ p["x"].abs(), "bias": err.sum(0), "residual": 0 * ad}
    for k in grads:
        want = differences(p, k)
        T.close(grads[k], want, bounds[k] + 2.0 ** -8 * (want.abs() + bounds[k]) + 1e-8, k)

    t, dy = T.mlp_case(5, 8, 6, 7, None, seed=16)
    _, grads = mlp_grads(on_device(t), dy.to(DEV))
    p = {k: v.double() for k, v in t.items() if v is not None}
    gate, up = p["x"] @ p["w_gate"].t(), p["x"] @ p["w_up"].t()

    def loss(p):  # noqa: F811
        return (((T.act64("silu", p["x"] @ p["w_gate"].t()) * (p["x"] @ p["w_up"].t())) @ p["w_down"].t()) * dy.double()).sum()

    dh = dy.double().abs() @ p["w_down"].abs()
    step = 2.0 ** -8
    dg = dh * up.abs() * (1.2 * 2 * step + step * gate.abs())  # up and dz rounded, the slope at the held gate
    du = dh * gate.abs() * 1.2 * 2 * step
    h_err = gate.abs() * up.abs() * 1.2 * 3 * step  # gate and up as held, the product rounded
    bounds = {"x": dg @ p["w_gate"].abs() + du @ p["w_up"].abs(), "w_gate": dg.t() @ p["x"].abs(),
              "w_up": du.t() @ p["x"].abs(), "w_down": dy.double().abs().t() @ h_err}
    for k in grads:
        want = differences(p, k)
        T.close(grads[k], want, bounds[k] + step * (want.abs() + bounds[k]) + 1e-8, k)


# ---------------------------------------------------------------------------- special values


@pytest.mark.parametrize("rows", [16, 300])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_special_values_stay_in_their_rows(rows, bad, checkpoint):
    t, dy = T.linear_case(rows, 96, 80, "silu", BF16, F32, checkpoint, seed=17)
    d, dy = on_device(t), dy.to(DEV)
    clean, grads = linear_grads(d, dy, "silu", checkpoint)
    keep = torch.arange(rows, device=DEV) != 7
    x = d["x"].detach().clone()
    x[7, 5] = bad
    y, g2 = linear_grads({**d, "x": x.requires_grad_()}, dy, "silu", checkpoint)
    same(y[keep], clean[keep])
    assert not torch.isfinite(y[7]).all()
    rows_of_block = keep if checkpoint is None else torch.arange(rows, device=DEV) >= 32  # a block shares its power of two
    same(g2["x"][rows_of_block], grads["x"][rows_of_block])
    assert not torch.isfinite(g2["weight"][:, 5]).any()
    r = d["residual"].detach().clone()
    r[7] = bad
    y = ta.fused_linear(d["x"], d["weight"], d["bias"], r, "silu")
    same(y[keep], clean[keep])
    assert not torch.isfinite(y[7]).any()
    worse = dy.clone()
    worse[7, 3] = bad
    g3 = linear_grads(d, worse, "silu", checkpoint)[1]
    same(g3["x"][keep], grads["x"][keep])
    m, mdy = T.mlp_case(rows, 40, 72, 64, None, seed=18)
    m, mdy = on_device(m), mdy.to(DEV)
    clean = mlp_grads(m, mdy, checkpoint)[0]
    x = m["x"].detach().clone()
    x[7, 5] = bad
    y = ta.swiglu_mlp(x, m["w_gate"], m["w_up"], m["w_down"], None, checkpoint)
    same(y[keep], clean[keep])
    assert not torch.isfinite(y[7]).all()


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_activations_of_large_values(act):
    """z of up to +-2^13 and 0: the activation's limits and its slope's, no NaN."""
    w = torch.eye(8, dtype=BF16, device=DEV)
    z = torch.tensor([0.0, -0.0, 30.0, -30.0, 100.0, -100.0, 8192.0, -8192.0]).repeat(40, 1)
    x = z.to(BF16).to(DEV).requires_grad_()
    y = ta.fused_linear(x, w, None, None, act)
    T.close(y, T.act64(act, z.double()), z.double().abs() * 2.0 ** -7 + 1e-9, "y")
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    s = torch.sigmoid(z.double())  # the derivative of z / (1 + exp(-z)) by its rule is inf / inf at -8192
    want = s * (1 + z * (1 - s)) if act == "silu" else T.act_grad64(act, z.double())
    T.close(dx, want, torch.full(z.shape, 2.0 ** -8 + 2.0 ** -9, dtype=torch.float64), "slope")


# ---------------------------------------------------------------------------- streams, graphs, memory


def test_another_stream():
    t, dy = T.linear_case(1000, 256, 520, "silu", BF16, F32, None, seed=19)
    d, dy = on_device(t), dy.to(DEV)
    y, grads = linear_grads(d, dy, "silu", "e4m3")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y2, grads2 = linear_grads(d, dy, "silu", "e4m3")
        back = ta.dequantize_activation(ta.quantize_activation(y2))
    torch.cuda.current_stream().wait_stream(side)
    same(y, y2)
    for k in grads:
        same(grads[k], grads2[k], k)
    same(back, ta.dequantize_activation(ta.quantize_activation(y)))


def _step(lin, mlp, dy, checkpoint):
    h, _ = linear_grads(lin, dy, "gelu", checkpoint)
    y, g = linear_grads(lin, dy, "gelu", checkpoint)
    z, m = mlp_grads(mlp, dy, checkpoint)
    return [h, y, z, *g.values(), *m.values()]


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_captured_steps(checkpoint):
    """Forward and backward of both in two graphs whose private pools hold their workspaces, replayed in turn
    with new inputs and eager work between; every replay equals the eager calls."""
    torch.manual_seed(0)

    def inputs(rows):
        lin = {k: torch.randn(s, device=DEV).mul(0.2).to(BF16).requires_grad_() for k, s in (
            ("x", (rows, 136)), ("weight", (264, 136)), ("bias", (264,)))}
        mlp = {"x": lin["x"], **{k: torch.randn(s, device=DEV).mul(0.1).to(BF16).requires_grad_() for k, s in (
            ("w_gate", (200, 136)), ("w_up", (200, 136)), ("w_down", (264, 200)))}}
        return lin, mlp, torch.randn(rows, 264, device=DEV).to(BF16)

    sets = [inputs(1300), inputs(17)]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for lin, mlp, dy in sets:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(lin, mlp, dy, checkpoint)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(_step(lin, mlp, dy, checkpoint))
        graphs.append(g)
    for k in range(3):
        for g, (lin, mlp, dy), out in zip(graphs, sets, outs):
            with torch.no_grad():
                lin["x"].add_(0.1)
                lin["weight"].mul_(1.01)
                dy.mul_(-1)
            g.replay()
            want = _step(lin, mlp, dy, checkpoint)
            torch.cuda.synchronize()
            for i, (a, b) in enumerate(zip(out, want)):
                same(a, b, f"replay {k}, result {i}")


def test_what_is_kept():
    """Between forward and backward, 8 bits keep about half of what bf16 does, and no gradient keeps nothing."""
    x = torch.randn(4096, 1024, device=DEV).to(BF16)
    w = torch.randn(1024, 1024, device=DEV).mul(0.03).to(BF16).requires_grad_()

    def kept(call):
        call()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        y = call()
        return torch.cuda.memory_allocated() - before - y.numel() * y.element_size()

    n = x.numel()
    assert kept(lambda: ta.fused_linear(x, w, activation="silu")) <= 2 * n + (1 << 16)  # z; x is the caller's
    assert kept(lambda: ta.fused_linear(x, w, activation="silu", checkpoint="e4m3")) <= 2 * (n + n // 1024) + (1 << 16)
    assert kept(lambda: ta.fused_linear(x, w.detach(), activation="silu")) <= 1 << 16
    assert kept(lambda: ta.swiglu_mlp(x, w, w, w)) <= 4 * n + (1 << 16)
    assert kept(lambda: ta.swiglu_mlp(x, w, w, w, None, "e4m3")) <= 3 * (n + n // 1024) + (1 << 16)


def test_nothing_behind_the_last_row_or_column_is_written():
    """Through the C ABI, where outputs may be parts of larger rows: what is around them stays."""
    import ctypes

    from torchure_amd import _native
    lib = _native.lib()
    g = torch.Generator().manual_seed(20)
    for rows, inp, out, f32 in ((37, 40, 29, 0), (300, 72, 261, 1), (513, 64, 777, 0), (5, 64, 77, 0)):
        a, b = T.grid_values(g, (rows, inp), 0.25, 6).to(DEV), T.grid_values(g, (out, inp), 2.0 ** -6, 12).to(DEV)
        room = torch.full((rows + 9, out + 15), 7.0, dtype=F32 if f32 else BF16, device=DEV)
        o = room[4: 4 + rows, 5: 5 + out]
        d = _native.TmLin(rows=rows, inp=inp, out=out, a=a.data_ptr(), b0=b.data_ptr(), o0=o.data_ptr(), lda=inp, ldb=inp,
                          ldo=out + 15, op=0, out_f32=f32)
        ws = torch.empty(max(1, lib.tm_lin_workspace_bytes(0, rows, inp, out, 0)), dtype=torch.uint8, device=DEV)
        _native.check(lib.tm_lin(ctypes.byref(d), ws.data_ptr(), ws.numel(), _native.stream_handle(torch.device(DEV, 0))), "tm_lin")
        want = torch.full_like(room, 7.0)
        y = ta.fused_linear(a, b, None, torch.zeros(rows, out, dtype=room.dtype, device=DEV))
        want[4: 4 + rows, 5: 5 + out] = y
        same(room, want, f"{rows} x {inp} -> {out}")


@pytest.mark.parametrize("rows,inp,out,held", [(5, 64, 77, 0), (5, 64, 77, 1), (40, 72, 33, 2), (300, 72, 130, 1), (300, 64, 130, 0)])
def test_the_gate_writes_its_rows_only(rows, inp, out, held):
    import ctypes

    from torchure_amd import _native
    lib = _native.lib()
    g = torch.Generator().manual_seed(23)
    a, b0, b1 = (T.grid_values(g, s, 0.125, 6).to(DEV) for s in ((rows, inp), (out, inp), (out, inp)))
    pad = -(-out // 8) * 8
    room = torch.full((rows + 6, pad + 24), 7.0, dtype=BF16, device=DEV)
    width = pad if held < 2 else -(-out // 32) * 32
    kept = [torch.full((rows + 4, width), 7, dtype=torch.uint8 if held == 2 else BF16, device=DEV) for _ in range(2)]
    exps = [torch.full((-(-rows // 32) * -(-out // 32) + 9,), 7, dtype=torch.uint8, device=DEV) for _ in range(2)]
    d = _native.TmLin(rows=rows, inp=inp, out=out, a=a.data_ptr(), b0=b0.data_ptr(), b1=b1.data_ptr(), o0=room[3:, 8:].data_ptr(),
                      lda=inp, ldb=inp, ldo=pad + 24, op=1, held=held, z0=kept[0].data_ptr(), z1=kept[1].data_ptr(),
                      s0=exps[0].data_ptr(), s1=exps[1].data_ptr(), ldz=width)
    ws = torch.empty(max(1, lib.tm_lin_workspace_bytes(1, rows, inp, out, 0)), dtype=torch.uint8, device=DEV)
    _native.check(lib.tm_lin(ctypes.byref(d), ws.data_ptr(), ws.numel(), _native.stream_handle(torch.device(DEV, 0))), "tm_lin")
    inside = torch.zeros(room.shape, dtype=torch.bool, device=DEV)
    inside[3: 3 + rows, 8: 8 + pad] = True
    assert bool((room[~inside] == 7.0).all())
    assert not room[3: 3 + rows, 8 + out: 8 + pad].any()  # the padding: zeros
    gate, up = a.double() @ b0.double().t(), a.double() @ b1.double().t()
    want = gate / (1 + torch.exp(-gate)) * up
    bound = want.abs() * 2.0 ** -8 + up.abs() * gate.abs().clamp_min(1) * T.ACT_ERR
    T.close(room[3: 3 + rows, 8: 8 + out], want.cpu(), bound.cpu(), "the gate's result")
    n = exps[0].numel() - 9
    for k, e in zip(kept, exps):
        assert bool((k[rows:] == 7).all()) and bool((e[n:] == 7).all())
        if held == 0:
            assert bool((k == 7).all()) and bool((e == 7).all())
        else:
            assert not k[:rows, out:].any()


def test_two_threads_on_two_streams():
    import threading

    t, dy = T.linear_case(700, 256, 520, "silu", BF16, F32, None, seed=24)
    m, mdy = T.mlp_case(130, 128, 320, 128, BF16, seed=24)
    sets = [(on_device(t), dy.to(DEV)), (on_device(m), mdy.to(DEV))]
    want = [linear_grads(*sets[0], "silu", "e4m3"), mlp_grads(*sets[1], "e4m3")]
    torch.cuda.synchronize()
    got = [None, None]

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            for _ in range(20):
                got[i] = linear_grads(*sets[0], "silu", "e4m3") if i == 0 else mlp_grads(*sets[1], "e4m3")
        stream.synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for th in threads:
        th.start()
    for th in threads:
        th.join(60)
        assert not th.is_alive()
    for (y, grads), (y2, grads2) in zip(want, got):
        same(y, y2)
        for k in grads:
            same(grads[k], grads2[k], k)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_saved_elsewhere_and_recomputed(checkpoint):
    """What is kept may be moved to the host between the passes, or made again."""
    from torch.utils.checkpoint import checkpoint as again

    t, dy = T.linear_case(70, 96, 77, "gelu", BF16, F32, None, seed=25)
    d, dy = on_device(t), dy.to(DEV)
    wide = torch.zeros(70, 200, dtype=BF16, device=DEV)
    wide[:, 8:104] = d["x"].detach()
    d["x"] = wide[:, 8:104].requires_grad_()  # strided rows
    m, mdy = T.mlp_case(50, 40, 77, 60, BF16, seed=25)
    m, mdy = on_device(m), mdy.to(DEV)
    y, grads = linear_grads(d, dy, "gelu", checkpoint)
    z, mgrads = mlp_grads(m, mdy, checkpoint)
    with torch.autograd.graph.save_on_cpu():
        y2, grads2 = linear_grads(d, dy, "gelu", checkpoint)
        z2, mgrads2 = mlp_grads(m, mdy, checkpoint)
    y3 = again(ta.fused_linear, d["x"], d["weight"], d["bias"], d["residual"], "gelu", checkpoint, use_reentrant=False)
    grads3 = dict(zip(d, torch.autograd.grad(y3, list(d.values()), dy)))
    z3 = again(ta.swiglu_mlp, *m.values(), checkpoint, use_reentrant=False)
    mgrads3 = dict(zip(m, torch.autograd.grad(z3, list(m.values()), mdy)))
    for a, b in ((y, y2), (z, z2), (y, y3), (z, z3)):
        same(a, b)
    for one, others in ((grads, (grads2, grads3)), (mgrads, (mgrads2, mgrads3))):
        for k in one:
            for o in others:
                same(one[k], o[k], k)
    # twice from what is kept
    y = ta.fused_linear(d["x"], d["weight"], d["bias"], d["residual"], "gelu", checkpoint)
    for _ in range(2):
        for k, v in zip(d, torch.autograd.grad(y, list(d.values()), dy, retain_graph=True)):
            same(grads[k], v, k)


# ---------------------------------------------------------------------------- together


def _block(p, h, labels, checkpoint):
    h = ta.fused_linear(h, p["wo"], None, h, None, checkpoint)
    h = ta.swiglu_mlp(h, p["w_gate"], p["w_up"], p["w_down"], h, checkpoint)
    h = ta.fused_linear(h, p["proj"], p["bias"], None, "gelu_tanh", checkpoint)
    return fused_linear_cross_entropy(h, p["head"], labels)


def _params(g):
    return {k: (torch.randn(s, generator=g) * s[-1] ** -0.5).to(DEV).requires_grad_() for k, s in (
        ("wo", (128, 128)), ("w_gate", (320, 128)), ("w_up", (320, 128)), ("w_down", (128, 320)), ("proj", (128, 128)),
        ("bias", (128,)), ("head", (512, 128)))}


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_a_block_with_its_loss(checkpoint):
    """Chained, the operators pass each other the gradients that calls one by one give."""
    g = torch.Generator().manual_seed(21)
    p, labels = _params(g), torch.randint(0, 512, (2, 33), generator=g).to(DEV)
    h0 = torch.randn(2, 33, 128, generator=g).to(DEV).requires_grad_()
    with torch.autocast("cuda", dtype=BF16):
        loss = _block(p, h0, labels, checkpoint)
        grads = dict(zip([*p, "h"], torch.autograd.grad(loss, [*p.values(), h0])))
        x0, r0 = h0.detach().requires_grad_(), h0.detach().requires_grad_()
        h1 = ta.fused_linear(x0, p["wo"], None, r0, None, checkpoint)
        x1, r1 = h1.detach().requires_grad_(), h1.detach().requires_grad_()
        h2 = ta.swiglu_mlp(x1, p["w_gate"], p["w_up"], p["w_down"], r1, checkpoint)
        x2 = h2.detach().requires_grad_()
        h3 = ta.fused_linear(x2, p["proj"], p["bias"], None, "gelu_tanh", checkpoint)
        x3 = h3.detach().requires_grad_()
        last = fused_linear_cross_entropy(x3, p["head"], labels)
        same(loss, last)
        d3, dhead = torch.autograd.grad(last, (x3, p["head"]))
        d2, dproj, dbias = torch.autograd.grad(h3, (x2, p["proj"], p["bias"]), d3)
        d1, dr1, dg, du, dd = torch.autograd.grad(h2, (x1, r1, p["w_gate"], p["w_up"], p["w_down"]), d2)
        d0, dr0, dwo = torch.autograd.grad(h1, (x0, r0, p["wo"]), d1 + dr1)
    for k, v in (("head", dhead), ("proj", dproj), ("bias", dbias), ("w_gate", dg), ("w_up", du), ("w_down", dd), ("wo", dwo),
                 ("h", d0 + dr0)):
        same(grads[k], v, k)


def test_training_steps_with_working_copies():
    """Three optimizer steps with and without working copies: the same losses, bit for bit."""
    def run(copies):
        g = torch.Generator().manual_seed(22)
        p, labels = _params(g), torch.randint(0, 512, (2, 40), generator=g).to(DEV)
        h = torch.randn(2, 40, 128, generator=g).to(DEV)
        if copies:
            ta.attach_bf16_working_params([v for v in p.values()])
        opt = ta.AdamW(list(p.values()), lr=1e-3)
        losses = []
        for _ in range(3):
            with torch.autocast("cuda", dtype=BF16):
                loss = _block(p, h, labels, "e4m3")
            loss.backward()
            ta.clip_grad_norm(list(p.values()), None, 1.0)
            opt.step()
            opt.zero_grad()
            losses.append(loss.detach())
        return losses, p

    (a, pa), (b, pb) = run(False), run(True)
    for x, y in zip(a, b):
        assert torch.isfinite(x)
        same(x, y)
    for k in pa:
        same(pa[k], pb[k], k)
