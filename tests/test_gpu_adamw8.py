"""AdamW on 8-bit moments against the same step in 64 bits, from what is held before it, and what a
program does with it: lists, clips, working copies, checkpoints of both widths, streams, graphs.

The oracle reads the held bytes by the format's definition. A moment that lies within the fp32 step's error of
the border at which its random bits turn it up may go either way; every other one has to be the oracle's."""

from __future__ import annotations

import copy
import io
import math

import pytest
import torch

import torchure_amd as ta
from torchure_amd.optimizer.adamw import held_bytes

pytestmark = pytest.mark.gpu

DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32
LR, BETAS, EPS, WD, SEED = 3e-4, (0.9, 0.95), 1e-8, 0.1, 0x1234567890ABCDEF
MASK = (1 << 32) - 1


# ---------------------------------------------------------------------------- the definition


def mix(z):
    z = ((z ^ (z >> 16)) * 0x8C2549D1) & MASK
    z = ((z ^ (z >> 15)) * 0xD406A25D) & MASK
    return z ^ (z >> 16)


def element_bits(i, seed, step):
    key = mix((step + mix(((seed >> 32) + mix(seed & MASK)) & MASK)) & MASK)
    z = (i * 0x9E3779B1 + key) & MASK
    z = ((z ^ (z >> 16)) * 0x8C2549D1) & MASK
    return z ^ (z >> 15)


E4M3 = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
ROOT = torch.tensor([float(c) if c < 16 else (16 + c % 16) * 2.0 ** (c // 16 - 1) for c in range(255)] + [math.nan],
                    dtype=torch.float64)


def spread(per_block, n):
    return per_block.repeat_interleave(64)[:n]


def held_values(m_bytes, r_bytes, n):
    """(m, r) in 64 bits of a tensor's bytes."""
    codes = -(-n // 256) * 256
    m, r = m_bytes.cpu(), r_bytes.cpu()
    em, er = m[codes:].double() - 127, r[codes:].double() - 145
    return (E4M3[m[:n].long()] * torch.pow(2.0, spread(em, n)), ROOT[r[:n].long()] * torch.pow(2.0, spread(er, n)))


def scales(x, top, low):
    """2^e of each element's block, by trying."""
    n = x.numel()
    padded = torch.zeros(-(-n // 64) * 64, dtype=torch.float64)
    padded[:n] = torch.where(torch.isfinite(x), x.abs(), 0.0)
    out = []
    for most in padded.view(-1, 64).amax(1).tolist():
        e = low if most == 0 else max(low, math.frexp(most)[1] - 30)
        while top * 2.0 ** e < most:
            e += 1
        out.append(2.0 ** e)
    return spread(torch.tensor(out, dtype=torch.float64), n)


def neighbours(x, scale, mantissa, least):
    """(lower, step) of magnitudes on the format's places."""
    y = x / scale
    step = torch.pow(2.0, torch.frexp(y)[1].double() - 1 - mantissa).clamp_min(least)
    return torch.floor(y / step) * step * scale, step * scale


def check_held(got, x, err, top, low, mantissa, least, smallest, u, what):
    """``got`` is within a step of x, and the right neighbour of it where the border is further than ``err``."""
    scale = scales(x, top, low)
    lower, step = neighbours(x.abs(), scale, mantissa, least)
    part = (x.abs() - lower) / step
    up = part + u >= 1
    want = lower + up * step
    if smallest:
        want = torch.where(x > 0, torch.maximum(want, scale * smallest), want)
    # x moves by up to err: what is held changes only where part + u passes a whole number (0 and 2 where x passes a place)
    sure = (part + u - torch.round(part + u)).abs() > err / step + 2.0 ** -19
    want = torch.copysign(want, x)
    off = (got - want).abs()
    assert bool((off[sure] == 0).all()), f"{what}: {int((off[sure] != 0).sum())} of {int(sure.sum())} held otherwise"
    assert bool((off <= step * (1 + 2.0 ** -20)).all()), f"{what}: over a step off"
    assert float(sure.double().mean()) > 0.99


def check_step(p, was_p, was, now, g, step, decay, seed=SEED, betas=BETAS, eps=EPS, lr=LR, wd=WD, copy_=None, first=0):
    """One step of one tensor: p after against p before, the held values before and after, the (scaled) grad."""
    m, r = was
    m2 = betas[0] * m + (1 - betas[0]) * g
    r2 = torch.sqrt(betas[1] * r * r + (1 - betas[1]) * g * g)
    b1, b2 = 1 - betas[0] ** step, 1 - betas[1] ** step
    denom = r2 / math.sqrt(b2) + eps
    d = was_p * (1 - lr * wd) if decay else was_p
    u = lr / b1 * m2 / denom
    want = d - u
    # each fp32 result is off by half a step: the constants (2^-24 each) and the sums of m and r, a
    # product, the quotient; p's own multiply-add and difference
    err_m = 2.0 ** -24 * (4 * betas[0] * m.abs() + 5 * (1 - betas[0]) * g.abs())
    err_p = 2.0 ** -24 * (2 * d.abs() + 16 * u.abs() + want.abs()) + lr / b1 * err_m / denom
    bad = ~((p - want).abs() <= err_p)
    assert not bad.any(), f"master: {int(bad.sum())} off, {float((p - want).abs().max()):.3g}"
    i = torch.arange(first, first + p.numel())
    bits = element_bits(i, seed, step)
    check_held(now[0], m2, err_m, 448.0, -117, 3, 2.0 ** -9, 0, ((bits & 0xFFFF) + 0.5) / 65536, "exp_avg")
    check_held(now[1], r2, 2.0 ** -24 * 5 * r2, 30.0 * 2 ** 14, -105, 4, 1.0, 1, ((bits >> 16) + 0.5) / 65536, "root")
    if copy_ is not None:
        assert torch.equal(copy_, p.float().to(BF16))


def f64(t):
    return t.detach().double().cpu().reshape(-1)


def moments(opt, p):
    st = opt.state[p]
    return held_values(st["exp_avg"], st["exp_avg_sq"], p.numel())


def make(sizes, grads="fp32", seed=0, **kw):
    g = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(s, generator=g).mul(0.02).to(DEV)) for s in sizes]
    decay = [p for p in params if p.dim() >= 2]
    rest = [p for p in params if p.dim() < 2]
    groups = [{"params": ps, "weight_decay": w} for ps, w in ((decay, WD), (rest, 0.0)) if ps]
    opt = ta.AdamW(groups, lr=LR, betas=BETAS, eps=EPS, state_bits=8, seed=SEED, **kw)
    works = ta.attach_bf16_working_params(params) if grads == "bf16" else None
    return params, opt, works, g


def set_grads(params, works, g, std=1e-3):
    out = []
    for i, p in enumerate(params):
        v = torch.randn(p.shape, generator=g) * std * torch.exp2(torch.randint(-8, 9, p.shape, generator=g).float())
        if works is None:
            p.grad = v.to(DEV)
            out.append(f64(p.grad))
        else:
            works[i].grad = v.to(DEV).to(BF16)
            out.append(f64(works[i].grad))
    return out


SIZES = [(1,), (2,), (3, 1), (1, 63), (64,), (5, 13), (255,), (1, 256), (257,), (7, 100), (2, 2049), (4095,), (3, 11000)]


@pytest.mark.parametrize("grads", ["fp32", "bf16"])
def test_steps(grads):
    params, opt, works, g = make(SIZES, grads)
    for step in range(1, 5):
        gs = set_grads(params, works, g)
        before = [f64(p) for p in params]
        was = [moments(opt, p) if opt.state.get(p) else (torch.zeros(p.numel()).double(),) * 2 for p in params]
        opt.step()
        for i, p in enumerate(params):
            assert float(opt.state[p]["step"]) == step
            assert opt.state[p]["exp_avg"].numel() == held_bytes(p.numel())
            check_step(f64(p), before[i], was[i], moments(opt, p), gs[i], step, p.dim() >= 2,
                       copy_=None if works is None else works[i].detach().cpu().reshape(-1))


def test_flat_moments():
    params, opt, works, g = make(SIZES)
    for _ in range(3):
        set_grads(params, works, g)
        opt.step()
    m, r = opt.flat_moments()
    order = [p for p in params if p.dim() >= 2] + [p for p in params if p.dim() < 2]
    want = [moments(opt, p) for p in order]
    assert m.dtype == r.dtype == BF16
    assert torch.equal(f64(m), torch.cat([w[0] for w in want]))
    assert torch.equal(f64(r), torch.cat([w[1] for w in want]))


@pytest.mark.parametrize("defer", [True, False])
def test_clip(defer):
    """A deferred clip scales the grads inside the step, the other before it: the same fp32 product."""
    params, opt, _, g = make(SIZES, defer_clip=defer)
    for step in (1, 2):
        gs = set_grads(params, None, g, 0.5)
        before = [f64(p) for p in params]
        was = [moments(opt, p) if step > 1 else (torch.zeros(p.numel()).double(),) * 2 for p in params]
        norm = ta.clip_grad_norm(params, None, 1.0)
        coef = torch.clamp(1.0 / (norm + 1e-6), max=1.0).double().cpu()
        opt.step()
        for i, p in enumerate(params):
            check_step(f64(p), before[i], was[i], moments(opt, p), gs[i] * coef, step, p.dim() >= 2)


def test_the_mean_is_kept():
    """Constant grads for 600 steps at beta2 = 0.999, where to the nearest no root would move. Over 16,384 elements the means are
    those of unrounded moments: m wanders by under 1.2 steps (an eighth of it) and the root by under a step's root, 0.25 of it, an element, so
    the means by under 0.002 of themselves at one deviation; 5 of them are allowed."""
    n = 16384
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    opt = ta.AdamW([p], lr=1e-4, betas=(0.9, 0.999), weight_decay=0.0, state_bits=8, seed=7)
    p.grad = torch.full((n,), 0.011, device=DEV)
    for _ in range(600):
        opt.step()
    m, r = (v.double() for v in opt.flat_moments())
    assert abs(float(m.mean()) / 0.011 - 1) < 0.01
    assert abs(float(r.mean()) / (0.011 * math.sqrt(1 - 0.999 ** 600)) - 1) < 0.01
    p.grad = torch.full((n,), -0.002, device=DEV)
    for _ in range(600):
        opt.step()
    m, r = (v.double() for v in opt.flat_moments())
    want = math.sqrt(0.011 ** 2 * (1 - 0.999 ** 600) * 0.999 ** 600 + 0.002 ** 2 * (1 - 0.999 ** 600))
    assert abs(float(m.mean()) / -0.002 - 1) < 0.01
    assert abs(float(r.mean()) / want - 1) < 0.01


def test_seeds():
    def run(seed):
        params, opt, _, g = make([(3, 700)])
        opt.seed = seed
        for _ in range(2):
            set_grads(params, None, g)
            opt.step()
        return opt.flat_moments()[0]

    a, b, c = run(5), run(5), run(6 << 40)
    assert torch.equal(a, b) and not torch.equal(a, c)
    assert float((a != c).double().mean()) > 0.2


def test_wide_range_in_a_block():
    """Values from 2^-40 of the block's largest on: a root is held as at least the smallest, m may vanish."""
    p = torch.nn.Parameter(torch.zeros(640, device=DEV))
    opt = ta.AdamW([p], lr=LR, betas=BETAS, eps=EPS, weight_decay=0.0, state_bits=8, seed=SEED)
    p.grad = torch.exp2(-torch.arange(640, device=DEV).float() % 64)
    zero = torch.zeros(640).double()
    opt.step()
    now = moments(opt, p)
    assert bool((now[1] > 0).all())
    check_step(f64(p), zero, (zero, zero), now, f64(p.grad), 1, False)
    before = f64(p)
    p.grad = torch.zeros_like(p)  # nothing comes for these any more
    opt.step()
    check_step(f64(p), before, now, moments(opt, p), zero, 2, False)
    assert bool((moments(opt, p)[1] > 0).all())
    assert float(f64(p).abs().max()) < 3 * LR


@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-18, 1e15])
def test_small_and_large_grads(size):
    p = torch.nn.Parameter(torch.zeros(300, device=DEV))
    opt = ta.AdamW([p], lr=LR, betas=BETAS, eps=EPS, weight_decay=0.0, state_bits=8, seed=SEED)
    g = torch.Generator().manual_seed(1)
    for step in range(1, 4):
        p.grad = (torch.rand(300, generator=g) + 0.5).mul(size).to(DEV)
        opt.step()
        m, r = moments(opt, p)
        assert torch.isfinite(m).all() and torch.isfinite(p).all()
        if size * size < 2.0 ** -150:
            assert not r.any()  # the squares are below fp32
        else:
            assert bool((r > 0.05 * size).all() and (r < 2 * size).all())


def test_zero_grads_and_state():
    params, opt, works, _ = make([(3, 100), (70,)], "bf16")
    for w in works:
        w.grad = torch.zeros_like(w)
    before = [p.detach().clone() for p in params]
    opt.step()
    for p, b in zip(params, before):
        assert not any(v.any() for v in moments(opt, p))
        want = b.double() * (1 - LR * WD) if p.dim() == 2 else b.double()
        assert bool(((p.double() - want).abs() <= 2.0 ** -23 * want.abs()).all())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_one_bad_element(bad):
    """It is NaN from then on, alone: its block's other elements are as they were."""
    params, opt, _, g = make([(1, 700)])
    p, = params
    twin = torch.nn.Parameter(p.detach().clone())
    other = ta.AdamW([twin], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=8, seed=SEED)
    for step in range(3):
        set_grads(params, None, g)
        twin.grad = p.grad.clone()
        if step == 1:
            p.grad[0, 333] = bad
        twin.grad[0, 333] = 0.0
        opt.step()
        other.step()
    m, r = moments(opt, p)
    assert math.isnan(m[333]) and math.isnan(r[333]) and math.isnan(p[0, 333])
    keep = torch.arange(700) // 64 != 333 // 64
    for a, b in zip((m, r, f64(p)), (*moments(other, twin), f64(twin))):
        assert torch.equal(a[keep], b[keep])
        assert bool(torch.isfinite(a[torch.arange(700) != 333]).all())


# ---------------------------------------------------------------------------- layouts


@pytest.mark.parametrize("chunk", [2048, 6144, 16384])
def test_places_and_chunks(chunk):
    """Masters, grads and copies at odd elements, other chunks: the same bits."""
    params, opt, _, g = make([(3, 5000), (901,)])
    twins = []
    for p in params:
        room = torch.zeros(p.numel() + 9, device=DEV)
        twins.append(torch.nn.Parameter(room[5: 5 + p.numel()].view(p.shape).copy_(p.detach())))
    other = ta.AdamW([{"params": twins[:1], "weight_decay": WD}, {"params": twins[1:], "weight_decay": 0.0}], lr=LR,
                     betas=BETAS, eps=EPS, state_bits=8, seed=SEED, chunk_elems=chunk)
    for _ in range(3):
        set_grads(params, None, g)
        for p, t in zip(params, twins):
            room = torch.zeros(p.numel() + 3, device=DEV)
            t.grad = room[1: 1 + p.numel()].view(p.shape).copy_(p.grad)
        opt.step()
        other.step()
    for p, t in zip(params, twins):
        assert torch.equal(p, t)
        for k in ("exp_avg", "exp_avg_sq"):
            assert torch.equal(opt.state[p][k], other.state[t][k])


def test_more_elements_than_32_bits():
    """The last elements of a tensor of 2^31 + 12,345 step by their own places' bits."""
    n, tail = (1 << 31) + 12345, 4096 + 12345 % 64
    p = torch.nn.Parameter(torch.zeros(n, device=DEV))
    p.grad = torch.zeros(n, device=DEV)
    g = torch.Generator().manual_seed(3)
    first = n - tail
    assert first % 64 == 0
    p.data[first:] = torch.randn(tail, generator=g).to(DEV)
    opt = ta.AdamW([p], lr=LR, betas=BETAS, eps=EPS, weight_decay=WD, state_bits=8, seed=SEED)
    codes = -(-n // 256) * 256
    was = (torch.zeros(tail).double(),) * 2
    for step in (1, 2):
        p.grad[first:] = torch.randn(tail, generator=g).to(DEV)
        before = f64(p[first:])
        opt.step()
        st = opt.state[p]
        parts = []
        for k in ("exp_avg", "exp_avg_sq"):
            b = torch.zeros(held_bytes(tail), dtype=torch.uint8)
            b[:tail] = st[k][first:n].cpu()
            exps = st[k][codes + first // 64: codes + -(-n // 64)].cpu()
            at = -(-tail // 256) * 256
            b[at: at + len(exps)] = exps
            parts.append(b)
        now = held_values(*parts, tail)
        check_step(f64(p[first:]), before, was, now, f64(p.grad[first:]), step, True, first=first)
        was = now
    assert not p[:first].any() and not opt.state[p]["exp_avg"][:first].any()


def test_empty_and_frozen_params():
    a, b, c = (torch.nn.Parameter(torch.ones(s, device=DEV)) for s in ((0,), (5,), (7,)))
    opt = ta.AdamW([a, b, c], state_bits=8)
    a.grad, b.grad = torch.ones_like(a), torch.ones_like(b)
    opt.step()
    assert c not in opt.state and bool((c == 1).all()) and bool((b < 1).all())
    m, r = opt.flat_moments()
    assert m.shape == r.shape == (5,)


# ---------------------------------------------------------------------------- checkpoints


def trained(steps=3, **kw):
    params, opt, works, g = make([(3, 700), (65,), (2, 256)], **kw)
    for _ in range(steps):
        set_grads(params, works, g)
        opt.step()
    return params, opt, g


def resumed(params, state, **kw):
    twins = [torch.nn.Parameter(p.detach().clone()) for p in params]
    groups = [{"params": [twins[0], twins[2]], "weight_decay": WD}, {"params": [twins[1]], "weight_decay": 0.0}]
    opt = ta.AdamW(groups, lr=LR, betas=BETAS, eps=EPS, **{"state_bits": 8, "seed": SEED, **kw})
    opt.load_state_dict(copy.deepcopy(state))  # (torch keeps the given step tensors)
    return twins, opt


@pytest.mark.parametrize("through", ["memory", "file", "cpu"])
def test_resume(through):
    """A resumed run goes on with the same bits."""
    params, opt, g = trained()
    state = copy.deepcopy(opt.state_dict())
    assert state["state"][0]["exp_avg"].dtype == torch.uint8
    if through == "file":
        f = io.BytesIO()
        torch.save(state, f)
        f.seek(0)
        state = torch.load(f, weights_only=True)
    elif through == "cpu":
        state["state"] = {i: {k: v.cpu() for k, v in s.items()} for i, s in state["state"].items()}
    twins, other = resumed(params, state)
    set_grads(params, None, g)
    for p, t in zip(params, twins):
        t.grad = p.grad.clone()
    opt.step()
    other.step()
    for p, t in zip(params, twins):
        assert torch.equal(p, t) and float(other.state[t]["step"]) == 4.0
        for k in ("exp_avg", "exp_avg_sq"):
            assert other.state[t][k].dtype == torch.uint8
            assert torch.equal(opt.state[p][k], other.state[t][k])


def test_8_bits_into_32():
    params, opt, _ = trained()
    twins, wide = resumed(params, opt.state_dict(), state_bits=32)
    for p, t in zip(params, twins):
        m, r = moments(opt, p)
        st = wide.state[t]
        assert st["exp_avg"].dtype == F32 and st["exp_avg"].shape == t.shape
        assert torch.equal(f64(st["exp_avg"]), m)
        assert torch.equal(f64(st["exp_avg_sq"]), r * r)
        t.grad = torch.ones_like(t)
    wide.step()
    with pytest.raises(RuntimeError, match="state_bits=32"):
        wide.flat_moments()


def nearest(x, top, low, mantissa, least):
    scale = scales(x, top, low)
    lower, step = neighbours(x.abs(), scale, mantissa, least)
    part = (x.abs() - lower) / step
    return torch.copysign(lower + (part + 32768.5 / 65536 >= 1) * step, x), (part - 0.5).abs() > 2.0 ** -14


@pytest.mark.parametrize("kind", ["torch", "this"])
def test_32_bits_into_8(kind):
    """Moments of a 32-bit checkpoint are held to the nearest."""
    g = torch.Generator().manual_seed(5)
    params = [torch.nn.Parameter(torch.randn(s, generator=g).to(DEV)) for s in ((3, 700), (65,), (2, 256))]
    groups = [{"params": [params[0], params[2]], "weight_decay": WD}, {"params": [params[1]], "weight_decay": 0.0}]
    cls = torch.optim.AdamW if kind == "torch" else ta.AdamW
    wide = cls(groups, lr=LR, betas=BETAS, eps=EPS, fused=True)
    for _ in range(3):
        set_grads(params, None, g)
        wide.step()
    twins, opt = resumed(params, wide.state_dict())
    for p, t in zip(params, twins):
        m, r = moments(opt, t)
        want, sure = nearest(f64(wide.state[p]["exp_avg"]), 448.0, -117, 3, 2.0 ** -9)
        assert torch.equal(m[sure], want[sure]) and float(sure.double().mean()) > 0.99
        want, sure = nearest(f64(wide.state[p]["exp_avg_sq"]).sqrt(), 30.0 * 2 ** 14, -105, 4, 1.0)
        sure &= want > 0
        assert torch.equal(r[sure], want[sure]) and float(sure.double().mean()) > 0.99
        assert float(opt.state[t]["step"]) == 3.0
        t.grad = torch.ones_like(t)
    opt.step()


def test_state_put_in_by_hand():
    p = torch.nn.Parameter(torch.ones(100, device=DEV))
    opt = ta.AdamW([p], lr=LR, betas=BETAS, weight_decay=0.0, state_bits=8)
    opt.state[p] = {"step": torch.tensor(5.0), "exp_avg": torch.full((100,), 0.5), "exp_avg_sq": torch.full((100,), 0.25)}
    p.grad = torch.full_like(p, 0.5)
    opt.step()
    assert float(opt.state[p]["step"]) == 6.0 and opt.state[p]["step"].is_cuda
    m, r = opt.flat_moments()
    assert bool((m == 0.5).all() and (r == 0.5).all())
    opt.state[p]["exp_avg"] = torch.zeros(7, device=DEV)
    with pytest.raises(RuntimeError, match="moments"):
        opt.step()


def test_pickled_and_copied():
    params, opt, _ = trained()
    both = copy.deepcopy((params, opt))
    assert both[1].state_bits == 8 and both[1].seed == SEED
    for a, b in zip(opt.flat_moments(), both[1].flat_moments()):
        assert torch.equal(a, b)


# ---------------------------------------------------------------------------- streams, graphs, C calls


def test_another_stream_and_replanned():
    params, opt, g = trained()
    twins, other = resumed(params, opt.state_dict())
    set_grads(params, None, g)
    for p, t in zip(params, twins):
        t.grad = p.grad.clone()
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        other.step()
        m, r = other.flat_moments()
    opt.step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(opt.flat_moments(), (m, r)):
        assert torch.equal(a, b)
    for p, t in zip(params, twins):
        assert torch.equal(p, t)


def test_graph():
    """A step captured once and replayed steps on: its counter and random bits are made on the device."""
    params, opt, g = trained()
    twins, other = resumed(params, opt.state_dict())
    set_grads(params, None, g)
    for p, t in zip(params, twins):
        t.grad = p.grad
    launch, = other.plan_step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch()
    for k in range(3):
        graph.replay()
        opt.step()
        torch.cuda.synchronize()
        for p, t in zip(params, twins):
            assert torch.equal(p, t), k
        for a, b in zip(opt.flat_moments(), other.flat_moments()):
            assert torch.equal(a, b)


def test_record_with_unknown_group_is_poisoned():
    params, opt, g = trained()
    set_grads(params, None, g)
    launch, = opt.plan_step()
    launch.n_groups = 1  # the second group's tensor now names a group that the call does not have
    launch()
    assert torch.isnan(params[1]).all() and torch.isnan(opt.state[params[1]]["step"])
    assert all(torch.isnan(v).all() for v in moments(opt, params[1]))
    assert torch.isfinite(params[0]).all() and torch.isfinite(params[2]).all()


def test_built_from_a_config():
    model = torch.nn.Linear(40, 30).to(DEV)
    opt = ta.build_optimizer(model, "adamw", {"lr": LR, "weight_decay": WD, "betas": BETAS, "fused": True, "state_bits": 8,
                                              "seed": 3})
    sched = ta.build_scheduler(opt, {"type": "wsd", "total_steps": 10, "warmup_ratio": 0.2, "decay_ratio": 0.2})
    for _ in range(3):
        model(torch.randn(8, 40, device=DEV)).square().mean().backward()
        ta.clip_grad_norm(model.parameters(), None, 1.0)
        opt.step()
        opt.zero_grad()
        sched.step()
    assert opt.state[model.weight]["exp_avg"].dtype == torch.uint8
    assert opt.flat_moments()[0].numel() == 40 * 30 + 30
