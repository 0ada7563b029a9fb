"""The linear layers, the gated feed-forward and 8-bit activations against the same formulas in 64 bits.

Where a product's sums are kept for the backward pass, a sum next to a rounding border would make the
two sides keep different values, so operands are small multiples of powers of two: sums of up to 2^24
of their units are exact in fp32 in any order, and both sides keep the same values. What is left is
derived in ``_bounds``.
"""

from __future__ import annotations

import math

import pytest
import torch

import torchure_amd as ta

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}  # half a step, relative to the value


def grid_values(g, shape, unit, most, dtype=BF16):
    """Whole multiples of ``unit`` up to ``most`` of them either way."""
    return (torch.randint(-most, most + 1, shape, generator=g).double() * unit).to(dtype)


# ---------------------------------------------------------------------------- the definitions, in 64 bits


def act64(name, z):
    if name in (None, "none"):
        return z
    if name == "relu":
        return z.clamp_min(0)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z / math.sqrt(2))
    return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))


def act_grad64(name, z):
    z = z.clone().requires_grad_()
    with torch.enable_grad():
        if name == "relu":
            return (z > 0).double()
        return torch.autograd.grad(act64(name, z).sum() + 0 * z.sum(), z)[0]


def e4m3_64(x):
    """What 8 bits hold of a finite matrix, from the format's definition."""
    n, d = x.shape
    out = torch.zeros_like(x)
    for i in range(0, n, 32):
        for j in range(0, d, 32):
            b = x[i: i + 32, j: j + 32]
            most = float(b.abs().max())
            e = -117
            while e < 119 and 448.0 * 2.0 ** e < most:
                e += 1
            v = (b * 2.0 ** -e).clamp(-448, 448)
            _, ex = torch.frexp(v.abs())
            step = torch.pow(2.0, (ex - 1).clamp_min(-6).double() - 3)
            out[i: i + 32, j: j + 32] = torch.round(v / step) * step * 2.0 ** e
    return out


def held64(checkpoint, x):
    return e4m3_64(x) if checkpoint == "e4m3" else x.to(BF16).double()


ACT_ERR = 2.0 ** -18  # an activation or its derivative on the GPU, relative to max(1, |z|) (7.5e-8 for the
# distribution function, an exponent's argument rounded at up to 2^-24 |z| with |z| < 60 here: 3.6e-6)


def close(got, want, bound, what):
    got, want = got.detach().double().cpu(), want.detach()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - want).abs().max()):.3g}"


def linear_case(rows, inp, out, act, bias, res, checkpoint, seed=0, xt=BF16, wt=BF16):
    g = torch.Generator().manual_seed(seed)
    t = {"x": grid_values(g, (rows, inp), 0.25, 6, xt), "weight": grid_values(g, (out, inp), 2.0 ** -6, 12, wt)}
    t["bias"] = None if bias is None else grid_values(g, (out,), 2.0 ** -7, 20, bias)
    t["residual"] = None if res is None else torch.randn(rows, out, generator=g).to(res)
    dy = torch.randn(rows, out, generator=g).to(F32 if res == F32 else BF16)
    return t, dy


def linear_want(t, dy, act, checkpoint):
    """Results and their bounds. Every product's sums are exact up to fp32 additions, at most one
    rounding of 2^-24 of the sum of magnitudes per addition (here: per K); dz is rounded to bf16."""
    d = {k: None if v is None else v.double() for k, v in t.items()}
    x, w, dy = d["x"], d["weight"], dy.double()
    z = x @ w.t() + (0 if d["bias"] is None else d["bias"])
    assert float((x.abs() @ w.abs().t()).max()) * 2 ** 8 < 2 ** 24  # exact in fp32
    y = act64(act, z) + (0 if d["residual"] is None else d["residual"])
    out_t = F32 if t["residual"] is not None and t["residual"].dtype == F32 else BF16
    sizes = z.abs().clamp_min(1) * (0 if act is None else ACT_ERR)
    want = {"y": (y, sizes + (HALF[out_t] + 2 ** -23) * y.abs() + 2 ** -23 * z.abs())}
    dz = dy * act_grad64(act, held64(checkpoint, z)) if act else dy
    err = (2.0 ** -8) * dz.abs() + (dy.abs() * ACT_ERR * 8 if act else 0)
    xk = held64(checkpoint, x)

    def product(a, a_err, b, dtype, k):
        s = a @ b
        return s, a_err @ b.abs() + (a.abs() @ b.abs()) * k * 2.0 ** -24 + HALF[dtype] * (s.abs() + a_err @ b.abs())

    want["x"] = product(dz, err, w, t["x"].dtype, w.shape[0])
    want["weight"] = product(dz.t(), err.t(), xk, t["weight"].dtype, x.shape[0])
    if t["bias"] is not None:
        b = dz.sum(0)
        e = (dz.abs() * (x.shape[0] * 2.0 ** -24) + (dy.abs() * ACT_ERR * 8 if act else 0)).sum(0)
        want["bias"] = (b, e + HALF[t["bias"].dtype] * (b.abs() + e))
    if t["residual"] is not None:
        want["residual"] = (dy, torch.zeros_like(dy))
    return want


SHAPES = [(1, 64, 64), (1, 8, 8), (2, 1, 1), (31, 72, 40), (128, 64, 128), (130, 136, 264), (37, 33, 29), (300, 200, 77),
          (257, 520, 136), (1, 777, 501)]


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("rows,inp,out", SHAPES)
@pytest.mark.parametrize("act,bias,res", [(None, None, None), ("silu", BF16, F32), ("gelu_tanh", F32, BF16)])
def test_linear_and_gradients(rows, inp, out, act, bias, res, checkpoint):
    t, dy = linear_case(rows, inp, out, act, bias, res, checkpoint, seed=rows + inp + out)
    want = linear_want(t, dy, act, checkpoint)
    dev = {k: None if v is None else v.to(DEV).requires_grad_() for k, v in t.items()}
    y = ta.fused_linear(dev["x"], dev["weight"], dev["bias"], dev["residual"], act, checkpoint)
    close(y, *want["y"], "y")
    with torch.no_grad():
        plain = ta.fused_linear(dev["x"], dev["weight"], dev["bias"], dev["residual"], act, checkpoint)
    assert torch.equal(plain, y)
    keys = [k for k in dev if dev[k] is not None]
    grads = torch.autograd.grad(y, [dev[k] for k in keys], dy.to(DEV))
    for k, got in zip(keys, grads):
        assert got.dtype == dev[k].dtype
        close(got, *want[k], "gradient of " + k)


@pytest.mark.parametrize("act", ["relu", "gelu"])
@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_linear_other_activations(act, checkpoint):
    t, dy = linear_case(70, 96, 80, act, BF16, None, checkpoint, seed=5)
    want = linear_want(t, dy, act, checkpoint)
    dev = {k: None if v is None else v.to(DEV).requires_grad_() for k, v in t.items()}
    y = ta.fused_linear(dev["x"], dev["weight"], dev["bias"], None, act, checkpoint)
    close(y, *want["y"], "y")
    for k, got in zip(("x", "weight", "bias"), torch.autograd.grad(y, [dev[k] for k in ("x", "weight", "bias")], dy.to(DEV))):
        close(got, *want[k], "gradient of " + k)


def mlp_case(rows, dim, ffn, out, res, seed, xt=BF16, wt=BF16):
    g = torch.Generator().manual_seed(seed)
    t = {"x": grid_values(g, (rows, dim), 0.25, 6, xt), "w_gate": grid_values(g, (ffn, dim), 2.0 ** -6, 12, wt),
         "w_up": grid_values(g, (ffn, dim), 2.0 ** -6, 12, wt), "w_down": torch.randn(out, ffn, generator=g).mul(0.1).to(wt)}
    t["residual"] = None if res is None else torch.randn(rows, out, generator=g).to(res)
    return t, torch.randn(rows, out, generator=g).to(F32 if res == F32 else BF16)


def mlp_want(t, dy, checkpoint):
    """As ``linear_want``. h is a bf16 matrix: a value next to a border may differ by a whole step,
    2^-7 of it, between the two sides."""
    x, wg, wu, wd = (t[k].to(BF16).double() for k in ("x", "w_gate", "w_up", "w_down"))
    dyb = dy.to(BF16).double()
    res = 0 if t["residual"] is None else t["residual"].double()
    out_t = F32 if t["residual"] is not None and t["residual"].dtype == F32 else BF16
    gate, up = x @ wg.t(), x @ wu.t()
    h = (act64("silu", gate) * up)
    h_err = h.abs() * 2.0 ** -8 + up.abs() * gate.abs().clamp_min(1) * ACT_ERR  # against the unrounded h
    y = h @ wd.t() + res
    e = h_err @ wd.abs().t() + (h.abs() @ wd.abs().t()) * wd.shape[1] * 2.0 ** -24
    want = {"y": (y, e + HALF[out_t] * (y.abs() + e))}
    gate, up = held64(checkpoint, gate), held64(checkpoint, up)
    a, slope = act64("silu", gate), act_grad64("silu", gate)
    dh = dyb @ wd
    dh_err = (dyb.abs() @ wd.abs()) * wd.shape[0] * 2.0 ** -24
    dg, du = dh * up * slope, dh * a
    act_e = ACT_ERR * 8
    dg_err = 2.0 ** -8 * dg.abs() + up.abs() * (dh_err * 1.2 + dh.abs() * act_e)
    du_err = 2.0 ** -8 * du.abs() + dh_err * a.abs() + dh.abs() * act_e * gate.abs().clamp_min(1)
    hk = a * up
    hk_err = hk.abs() * 2.0 ** -8 + up.abs() * gate.abs().clamp_min(1) * act_e
    xk = held64(checkpoint, x)

    def product(a, a_err, b, dtype, k):
        s, e = a @ b, a_err @ b.abs() + (a.abs() @ b.abs()) * k * 2.0 ** -24
        return s, e + HALF[dtype] * (s.abs() + e)

    dyf = dyb if dy.dtype == BF16 else dy.double()  # an fp32 gradient is rounded to bf16 for the products
    dy_err = dyf.abs() * (0 if dy.dtype == BF16 else 2.0 ** -8)
    n, ffn = dg.shape
    xa, xb = product(dg, dg_err, wg, F32, 2 * ffn), product(du, du_err, wu, F32, 2 * ffn)
    s, e = xa[0] + xb[0], xa[1] + xb[1]
    want["x"] = (s, e + HALF[t["x"].dtype] * (s.abs() + e))
    want["w_gate"] = product(dg.t(), dg_err.t(), xk, t["w_gate"].dtype, n)
    want["w_up"] = product(du.t(), du_err.t(), xk, t["w_up"].dtype, n)
    s, e = dyb.t() @ hk, dyb.abs().t() @ hk_err + dy_err.t() @ hk.abs() + (dyb.abs().t() @ hk.abs()) * n * 2.0 ** -24
    want["w_down"] = (s, e + HALF[t["w_down"].dtype] * (s.abs() + e))
    if t["residual"] is not None:
        want["residual"] = (dy.double(), torch.zeros_like(dyb))
    return want


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("rows,dim,ffn,out,res", [
    (1, 64, 128, 64, BF16), (5, 8, 8, 16, None), (33, 72, 100, 72, F32), (130, 128, 320, 128, BF16), (50, 37, 45, 37, BF16),
    (300, 136, 77, 40, None), (257, 64, 200, 64, None)])
def test_mlp_and_gradients(rows, dim, ffn, out, res, checkpoint):
    t, dy = mlp_case(rows, dim, ffn, out, res, seed=rows + ffn)
    want = mlp_want(t, dy, checkpoint)
    dev = {k: None if v is None else v.to(DEV).requires_grad_() for k, v in t.items()}
    args = (dev["x"], dev["w_gate"], dev["w_up"], dev["w_down"], dev["residual"], checkpoint)
    y = ta.swiglu_mlp(*args)
    close(y, *want["y"], "y")
    with torch.no_grad():
        assert torch.equal(ta.swiglu_mlp(*args), y)
    keys = [k for k in dev if dev[k] is not None]
    for k, got in zip(keys, torch.autograd.grad(y, [dev[k] for k in keys], dy.to(DEV))):
        assert got.dtype == dev[k].dtype
        close(got, *want[k], "gradient of " + k)


# ---------------------------------------------------------------------------- 8 bits


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape", [(1,), (7,), (1, 1), (32, 32), (33, 65), (5, 3, 40), (100, 257), (64, 8)])
def test_quantize_equals_the_format(shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * torch.exp2(torch.randint(-20, 20, shape, generator=g).float())).to(dtype)
    q = ta.quantize_activation(x.to(DEV))
    got = ta.dequantize_activation(q)
    assert got.dtype == dtype and got.shape == x.shape
    want = e4m3_64(x.double().reshape(-1, shape[-1])).reshape(shape)
    assert torch.equal(got.double().cpu(), want)
    assert torch.equal(ta.dequantize_activation(q, F32).double().cpu(), want)
    assert torch.equal(ta.dequantize_activation(q, BF16).double().cpu(), want)
    rows, cols = x.reshape(-1, shape[-1]).shape
    assert q.nbytes == rows * (-(-cols // 32) * 32) + -(-rows // 32) * -(-cols // 32)
    assert int(q.values[:, cols:].count_nonzero()) == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_quantize_every_bit_pattern(dtype):
    """All 65,536 bf16 values (as bf16 and widened), 32 x 32 at a time: special values, subnormals, the
    largest."""
    bits = torch.arange(65536, dtype=torch.int32).to(torch.int16)
    x = bits.view(BF16).reshape(256, 256).to(dtype)
    got = ta.dequantize_activation(ta.quantize_activation(x.to(DEV))).cpu()
    fine = torch.isfinite(x.float())
    assert torch.isnan(got.float())[~fine].all()
    want = e4m3_64(torch.where(fine, x.double(), 0.0))
    assert torch.equal(torch.where(fine, got.double(), 0.0), want)


def test_quantize_zeros_and_tiny():
    x = torch.zeros(64, 64, dtype=F32)
    x[40, 40] = 1e-38
    x[3, 3] = -0.0
    got = ta.dequantize_activation(ta.quantize_activation(x.to(DEV))).cpu()
    assert torch.equal(got.double(), e4m3_64(x.double()))
    e = ta.quantize_activation(x.to(DEV)).exponents
    assert int(e.min()) >= 10 and int(e.max()) <= 246


def test_quantize_strided_rows_and_columns():
    x = torch.randn(70, 200, device=DEV).to(BF16)
    for v in (x[:, 3:100], x[::2], x.t(), x[:, ::3], x[5:6].expand(40, 200)):
        a, b = ta.dequantize_activation(ta.quantize_activation(v)), ta.dequantize_activation(
            ta.quantize_activation(v.contiguous()))
        assert torch.equal(a, b) and a.shape == v.shape
