"""The activations and their slopes over the whole range of z, tails and limits among it, each value against
64 bits by a bound relative to itself. Through an identity weight, so that z is x to the bit."""

from __future__ import annotations

import math

import pytest
import torch

import torchure_amd as ta

pytestmark = pytest.mark.gpu

DEV, BF16 = "cuda", torch.bfloat16
ULP = 2.0 ** -24  # half a step of fp32, relative to the value
TINY = 2.0 ** -116  # what becomes zero where exp2's or the reciprocal's result leaves fp32's normal range, times z < 2^7


def cdf64(z):
    return 0.5 * torch.special.erfc(-z / math.sqrt(2))


def published_tail(z):
    """Formula 7.1.26 of Abramowitz and Stegun for erfc(|z| / sqrt 2) / 2, in 64 bits."""
    t = 1 / (1 + 0.3275911 / math.sqrt(2) * z.abs())
    c = (0.254829592, -0.284496736, 1.421413741, -1.453152027, 1.061405429)
    return 0.5 * sum(k * t ** (i + 1) for i, k in enumerate(c)) * torch.exp(-0.5 * z * z)


def wanted(act, z):
    """(value, its bound, slope, its bound) without the bf16 rounding. Of each: its relative error in fp32 from
    the number of roundings on the way, an exponent's argument a counting |a| times its own, and of a sum the
    errors of its terms."""
    zero = torch.zeros_like(z)
    if act == "relu":
        return z.clamp_min(0), zero, (z > 0).double(), zero
    if act == "gelu":
        tail = published_tail(z)
        cdf = torch.where(z < 0, tail, 1 - tail)
        bell = torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
        # Horner's five steps cancel at most 5-fold, t's three roundings count up to five times; the exponent is z^2 / 2
        rel = (130 + z * z) * ULP * tail + ULP * cdf
        off = (cdf - cdf64(z)).abs()  # the formula's own error: at most 7.5e-8
        assert float(off.max()) <= 7.6e-8
        return (z * cdf64(z), z.abs() * (rel + off + 2 * ULP * cdf),
                cdf64(z) + z * bell, rel + off + 2 * ULP * cdf + (z * z + 6) * ULP * z.abs() * bell)
    k = 1.0 + 0.044715 * z * z if act == "gelu_tanh" else 1.0
    c = 2 * math.sqrt(2 / math.pi) if act == "gelu_tanh" else 1.0
    a = c * z * k
    s, r = torch.sigmoid(a), torch.sigmoid(-a)
    rel = (6 * a.abs().clamp_max(200) + 8) * ULP
    more = c * (1.0 + 0.134145 * z * z) if act == "gelu_tanh" else 1.0
    # 1 - s in fp32 is off by s's rounding where it is not zero on both sides
    near = torch.where(r > 2.0 ** -26, z.abs() * s * more * 2 * ULP, zero)
    # the second term vanishes with s or 1 - s, however large z
    second = torch.where(s * r > 0, z * s * r * more, zero)
    return z * s, (z * s).abs() * rel, s + second, s * rel + second.abs() * (rel + 6 * ULP) + near


@pytest.mark.parametrize("rows", [16, 40, 300])
@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_values_and_slopes(act, rows):
    """z from 2^-20 to 2^13 either way, 3 to 9 below zero closely, and zeros."""
    near = -torch.arange(3, 9, 1 / 32)
    wide = torch.exp2(torch.linspace(-20, 13, 200))
    z = torch.cat([near, wide, -wide, torch.tensor([0.0, -0.0, 30.0, -30.0, 100.0, -100.0, 8192.0, -8192.0])]).to(BF16)
    w = torch.eye(z.numel(), dtype=BF16, device=DEV)
    x = z.repeat(rows, 1).to(DEV).requires_grad_()
    y = ta.fused_linear(x, w, None, None, act)
    dx, = torch.autograd.grad(y, x, torch.ones_like(y))
    value, e_value, slope, e_slope = wanted(act, z.double())
    for got, want, e, what in ((y, value, e_value, "value"), (dx, slope, e_slope, "slope")):
        assert bool((got == got[:1]).all())
        got = got[0].detach().double().cpu()
        bound = 2.0 ** -8 * (want.abs() + e) + e + TINY * (act != "relu")
        bad = ~((got - want).abs() <= bound)
        assert not bad.any(), [(float(a), float(b), float(c), float(d)) for a, b, c, d in
                               zip(z[bad].double(), got[bad], want[bad], bound[bad])][:8]


@pytest.mark.parametrize("largest", [448.0, 225.0, 224.5, 300.0])
@pytest.mark.parametrize("e", [0, -30, 60])
def test_8_bits_are_off_by_no_more_than_stated(largest, e):
    """At most 2^-4 of the value, or 2^-10 of the block's power of two; zero from there down; and 2^-4 alone
    is too little from 2^-13.8 of the block's largest on."""
    x = torch.exp2(torch.linspace(-24, 0, 32 * 32).double()) * largest * torch.tensor([1.0, -1.0]).double().repeat(512)
    x = (x * 2.0 ** e).float().reshape(32, 32)
    assert float(x.abs().max()) == largest * 2.0 ** e
    q = ta.quantize_activation(x.to(DEV))
    assert int(q.exponents) == e + 127
    off = (ta.dequantize_activation(q).cpu().double() - x.double()).abs()
    size, power = x.double().abs(), 2.0 ** e
    assert bool((off <= torch.maximum(2.0 ** -4 * size, torch.full_like(size, 2.0 ** -10 * power))).all())
    assert bool((off == size)[size <= 2.0 ** -10 * power].all())
    fine = size >= 2.0 ** -6 * power
    assert bool((off <= 2.0 ** -4 * size)[fine].all()) and not bool((off <= 2.0 ** -4 * size)[~fine].all())
