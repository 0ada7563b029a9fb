"""Performance cases of what a training step does around the block's products: norms, the token embedding
with its gradient, and the optimizer step on moments held in 8 bits.

Three families, each with listed cases and a generator of further cases of the same ranges:

- ``norm``: layer norm and RMS norm over the last dimension, forward alone or with all gradients;
- ``embed``: ``y = scale * weight[ids]``, forward alone, with the weight's gradient (the tokens' gradients summed
  by id), or that gradient added into one that is there already (a head tied to the embedding);
- ``adamw8``: one AdamW step over a list of tensors whose moments are held in 8 bits, and the moments as
  they are held after it.

Definitions of the 8-bit moments, for both sides. Each tensor's elements, in order, are cut into blocks of 64; the
first moment m is held as e4m3 values with one power of two for each block, ``2^e``, e the least with which the block's
largest finite magnitude is at most 448, clamped to [-117, 119]. Of the second moment its root r is held, as
``n(c) 2^x``: c is 8 bits, n(c) = c below 16, else (16 + c % 16) 2^(c / 16 - 1), 254 the largest code of a number (255 is
NaN), x the least with which the block's largest finite r is at most n(254) 2^x, at least -105. A value between two that
can be held becomes the upper one (in magnitude) if the part of the step that it lies above the lower one, plus u, is at least 1;
u is (16 bits of a 32-bit hash + 1/2) / 2^16. A nonzero r is held as at least n(1). The hash of element i in step s
of a run with the seed k is ``_element(i * A + key)``, its low half for m and its high one for r, the key
``_mix(s + _mix(k >> 32 + _mix(k)))``, all modulo 2^32. The step itself uses the moments before they are rounded.

``listed()`` and ``draw(rng)`` give cases (plain dicts), ``prepare`` what a program has in hand before the call, ``run``
one pass, ``exact`` the same outputs in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

LR, BETAS, EPS, WEIGHT_DECAY, SEED = 3e-4, (0.9, 0.95), 1e-8, 0.1, 2024
STEPS_DONE = 1000  # the optimizer is in its steady state
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


def listed():
    return [
        # One token's hidden state before a projection: a generated sample. Latency.
        {"name": "norm-token", "family": "norm", "kind": "rms", "rows": 1, "dim": 1024, "x": "bf16", "out": "bf16",
         "weight": "bf16", "bias": False, "grad": False},
        # Query and key heads of the 0.6B shape, 8192 tokens: many short rows.
        {"name": "norm-heads", "family": "norm", "kind": "rms", "rows": 8192 * 24, "dim": 128, "x": "bf16", "out": "bf16",
         "weight": "fp32", "bias": False, "grad": True},
        # A training batch at the 4B shape's width, bf16 residual stream, weight and bias.
        {"name": "norm-4b-layer", "family": "norm", "kind": "layer", "rows": 8192, "dim": 2560, "x": "bf16",
         "out": "bf16", "weight": "bf16", "bias": True, "grad": True},
        # A packed batch, odd width, fp32 residual stream whose norm feeds a bf16 product.
        {"name": "norm-odd-fp32", "family": "norm", "kind": "layer", "rows": 6001, "dim": 1237, "x": "fp32",
         "out": "bf16", "weight": "fp32", "bias": True, "grad": True},
        # One token's row of the 0.6B table.
        {"name": "embed-token", "family": "embed", "tokens": 1, "vocab": 151936, "dim": 1024, "weight": "fp32",
         "out": "bf16", "scale": 1.0, "padding": False, "mode": "forward"},
        # A training batch of the 0.6B shape on its fp32 master.
        {"name": "embed-0.6b", "family": "embed", "tokens": 8192, "vocab": 151936, "dim": 1024, "weight": "fp32",
         "out": "fp32", "scale": 1.0, "padding": False, "mode": "train"},
        # Many tokens of a small vocabulary, scaled, a third of the batch padding: few rows, long sums.
        {"name": "embed-small-vocab", "family": "embed", "tokens": 50001, "vocab": 4096, "dim": 777, "weight": "bf16",
         "out": "bf16", "scale": 27.875, "padding": True, "mode": "train"},
        # The 4B shape's tied head: its gradient is there, the embedding's is added.
        {"name": "embed-4b-tied", "family": "embed", "tokens": 8192, "vocab": 151936, "dim": 2560, "weight": "fp32",
         "out": "fp32", "scale": 1.0, "padding": False, "mode": "accumulate"},
        # The tiny configuration: launches and host work.
        {"name": "adamw8-tiny", "family": "adamw8", "params": "decoder", "vocab": 4096, "dim": 256, "layers": 2,
         "ffn": 768, "heads": 4, "kv": 2, "head_dim": 64, "grads": "bf16"},
        # An irregular list (adapters, biases, odd lengths) on plain fp32 gradients.
        {"name": "adamw8-irregular", "family": "adamw8", "params": "list", "tensors": 400, "log2_max": 20, "list_seed": 5,
         "grads": "fp32"},
        # The 0.6B shape with bf16 working copies: the largest.
        {"name": "adamw8-0.6b", "family": "adamw8", "params": "decoder", "vocab": 151936, "dim": 1024, "layers": 28,
         "ffn": 2816, "heads": 16, "kv": 8, "head_dim": 128, "grads": "bf16"},
    ]


def _log_uniform(rng: random.Random, lo: float, hi: float) -> int:
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _width(rng, lo, hi):
    """A hidden width: mostly whole vectors, some anything."""
    n, kind = _log_uniform(rng, lo, hi), rng.random()
    return n if kind < 0.25 else max(8, n // 8 * 8) if kind < 0.5 else max(64, n // 64 * 64)


def draw(rng: random.Random):
    family = rng.choice(["norm", "norm", "embed", "embed", "adamw8"])
    if family == "norm":
        dim, grad, x = _width(rng, 24, 9728), rng.random() < 0.7, rng.choice(["bf16", "bf16", "fp32"])
        return {"family": family, "kind": rng.choice(["rms", "layer"]),
                "rows": min(_log_uniform(rng, 1, 200_000), max(1, 40_000_000 // dim)), "dim": dim, "x": x,
                "out": rng.choice([x, "bf16"]), "weight": rng.choice(["bf16", "fp32"]), "bias": rng.random() < 0.5,
                "grad": grad}
    if family == "embed":
        weight = rng.choice(["bf16", "fp32"])
        return {"family": family, "tokens": _log_uniform(rng, 1, 50_000), "vocab": _log_uniform(rng, 300, 151936),
                "dim": _width(rng, 32, 2560), "weight": weight, "out": rng.choice([weight, "bf16"]),
                "scale": rng.choice([1.0, 1.0, 16.0, 27.875]), "padding": rng.random() < 0.4,
                "mode": rng.choice(["forward", "train", "train", "accumulate"])}
    return {"family": family, "params": "list", "tensors": _log_uniform(rng, 10, 1000), "log2_max": rng.randint(12, 21),
            "list_seed": rng.randrange(1 << 20), "grads": rng.choice(["bf16", "fp32"])}


# ---------------------------------------------------------------------------- norms


def _norm_inputs(case, seed):
    """Hidden states whose channels differ in spread and place and of which a few rows are large; weights near
    one; the gradient of a mean loss's size."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device=dev).normal_(0.0, std, generator=g)

    n, d = case["rows"], case["dim"]
    x = normal(n, d) * normal(d, std=0.5).exp_() + normal(d, std=0.3)
    x[torch.randint(0, n, (max(1, n // 1000),), device=dev, generator=g)] *= 30.0
    t = {"x": x.to(TYPES[case["x"]]), "weight": (1.0 + normal(d, std=0.2)).to(TYPES[case["weight"]]),
         "bias": normal(d, std=0.1).to(TYPES[case["weight"]]) if case["bias"] and case["kind"] == "layer" else None}
    if case["grad"]:
        t["dy"] = normal(n, d, std=1e-3).to(TYPES[case["out"]])
    return t


NORM_EPS = {"rms": 1e-6, "layer": 1e-5}


def _norm_own(state):
    import torchure_amd as ta

    case, t = state["case"], state["t"]
    kind, out = case["kind"], TYPES[case["out"]]
    with torch.set_grad_enabled(case["grad"]):
        if kind == "rms":
            y = ta.rms_norm(t["x"], t["weight"], eps=NORM_EPS[kind], dtype=out)
        else:
            y = ta.layer_norm(t["x"], t["weight"], t["bias"], eps=NORM_EPS[kind], dtype=out)
    if not case["grad"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [t[k] for k in state["wanted"]], state["dy"])
    return {"y": y.detach(), **{"d_" + k: v for k, v in zip(state["wanted"], grads)}}


def _norm_plain(state):
    case, t, dy = state["case"], state["t"], state["dy"]
    with torch.no_grad():
        x, w = t["x"].float(), t["weight"].float()
        if case["kind"] == "layer":
            x = x - x.mean(-1, keepdim=True)
        rstd = (x.square().mean(-1, keepdim=True) + NORM_EPS[case["kind"]]).rsqrt()
        xhat = x * rstd
        y = xhat * w
        if t["bias"] is not None:
            y = y + t["bias"].float()
        out = {"y": y.to(TYPES[case["out"]])}
        if not case["grad"]:
            return out
        dy = dy.float()
        dw = dy * w
        dx = dw - xhat * (dw * xhat).mean(-1, keepdim=True)
        if case["kind"] == "layer":
            dx = dx - dw.mean(-1, keepdim=True)
        out["d_x"] = (dx * rstd).to(t["x"].dtype)
        out["d_weight"] = (dy * xhat).sum(0).to(t["weight"].dtype)
        if t["bias"] is not None:
            out["d_bias"] = dy.sum(0).to(t["bias"].dtype)
        return out


def _norm_exact(case, seed):
    t = {k: v if v is None else v.double() for k, v in _norm_inputs(case, seed).items()}
    x, w, b = t["x"], t["weight"], t["bias"]
    n, d = x.shape
    ones = torch.ones(d, dtype=torch.float64, device=x.device)
    mean = torch.mv(x, ones) / d if case["kind"] == "layer" else torch.zeros(n, dtype=torch.float64, device=x.device)
    centred = x - mean[:, None]
    size = torch.sqrt((centred * centred).sum(1) / d + NORM_EPS[case["kind"]])
    unit = centred / size[:, None]
    out = {"y": unit * w[None, :] + (0.0 if b is None else b[None, :])}
    if case["grad"]:
        dy = t["dy"]
        dunit = dy * w[None, :]
        along = (dunit * unit).sum(1) / d
        dx = (dunit - unit * along[:, None]) / size[:, None]
        if case["kind"] == "layer":
            dx -= (torch.mv(dunit, ones) / d / size)[:, None]
        out["d_x"], out["d_weight"] = dx, (dy * unit).sum(0)
        if b is not None:
            out["d_bias"] = torch.mv(dy.t(), torch.ones(n, dtype=torch.float64, device=x.device))
    return out


# ---------------------------------------------------------------------------- embedding


PAD = 3  # the padding token's id


def _embed_inputs(case, seed):
    """Ids as text has them (a few are most of the tokens), a third of the places padding where there is any; weights
    at their usual spread; the gradient of a mean loss's size."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    n, v, d = case["tokens"], case["vocab"], case["dim"]
    ids = (torch.rand(n, device=dev, generator=g).pow_(4) * v).long().clamp_(max=v - 1)
    if case["padding"]:
        ids[n - n // 3:] = PAD
    t = {"ids": ids, "weight": torch.empty(v, d, device=dev).normal_(0.0, 0.02, generator=g).to(TYPES[case["weight"]])}
    if case["mode"] != "forward":
        t["dy"] = torch.empty(n, d, device=dev).normal_(0.0, 1e-3, generator=g).to(TYPES[case["out"]])
    if case["mode"] == "accumulate":
        t["grad"] = torch.empty(v, d, device=dev).normal_(0.0, 1e-3, generator=g).to(TYPES[case["weight"]])
    return t


def _embed_own(state):
    import torchure_amd as ta

    case, t = state["case"], state["t"]
    pad = PAD if case["padding"] else None
    out = TYPES[case["out"]]
    if case["mode"] == "accumulate":
        with torch.no_grad():
            y = ta.embedding(t["ids"], t["weight"], scale=case["scale"], padding_idx=pad, dtype=out)
        ta.embedding_grad_(t["grad"], t["ids"], state["dy"], scale=case["scale"], padding_idx=pad)
        return {"y": y, "grad": t["grad"]}
    with torch.set_grad_enabled(case["mode"] == "train"):
        y = ta.embedding(t["ids"], t["weight"], scale=case["scale"], padding_idx=pad, dtype=out)
    if case["mode"] == "forward":
        return {"y": y}
    grad, = torch.autograd.grad(y, t["weight"], state["dy"])
    return {"y": y.detach(), "d_weight": grad}


def _embed_plain(state):
    case, t, dy = state["case"], state["t"], state["dy"]
    with torch.no_grad():
        ids, weight = t["ids"], t["weight"]
        out = {"y": (weight[ids].float() * case["scale"]).to(TYPES[case["out"]])}
        if case["mode"] == "forward":
            return out
        dy = dy.float()
        if case["padding"]:
            dy = torch.where((ids == PAD)[:, None], 0.0, dy)
        sums = torch.zeros(weight.shape, device=ids.device).index_add_(0, ids, dy) * case["scale"]
        if case["mode"] == "train":
            out["d_weight"] = sums.to(weight.dtype)
        else:
            out["grad"] = t["grad"].copy_(t["grad"].float() + sums)
        return out


def _embed_exact(case, seed):
    t = _embed_inputs(case, seed)
    ids, scale = t["ids"], float(torch.tensor(case["scale"]))
    out = {"y": torch.index_select(t["weight"], 0, ids).double() * scale}
    if case["mode"] == "forward":
        return out
    order = torch.argsort(ids, stable=True)
    found, count = torch.unique_consecutive(ids[order], return_counts=True)
    sums = torch.zeros(t["weight"].shape, dtype=torch.float64, device=ids.device)
    ends = torch.cumsum(count, 0)
    rows = t["dy"][order].double()
    group = torch.repeat_interleave(torch.arange(len(found), device=ids.device), count)
    each = torch.zeros(len(found), case["dim"], dtype=torch.float64, device=ids.device)
    each.index_put_((group,), rows, accumulate=True)
    assert int(ends[-1]) == len(ids)
    if case["padding"]:
        each[found == PAD] = 0.0
    sums[found] = each * scale
    out.update({"d_weight": sums} if case["mode"] == "train" else {"grad": t["grad"].double() + sums})
    return out


# ---------------------------------------------------------------------------- AdamW on 8-bit moments


BLOCK = 64
ALIGN = 256  # elements from one tensor's start to the next one's, a multiple of this
A, B, C = 0x9E3779B1, 0x8C2549D1, 0xD406A25D
MASK = (1 << 32) - 1


def _element(z):
    z = z ^ (z >> 16)
    z = (z * B) & MASK
    return z ^ (z >> 15)


def _mix(z):
    z = (((z ^ (z >> 16)) * B) & MASK)
    z = (((z ^ (z >> 15)) * C) & MASK)
    return z ^ (z >> 16)


def _key(seed, step):
    return _mix((step + _mix(((seed >> 32) + _mix(seed & MASK)) & MASK)) & MASK)


def _shapes(case):
    """The list's shapes, those with weight decay (two dimensions) before the others."""
    if case["params"] == "list":
        r = random.Random(case["list_seed"])
        out = []
        for _ in range(case["tensors"]):
            n = max(1, int(2.0 ** r.uniform(3.0, case["log2_max"])))
            if case["grads"] == "bf16" or r.random() < 0.6:  # whole vectors, the rest anything
                n = -(-n // 8) * 8
            out.append((n,) if r.random() < 0.4 else (1, n))
    else:
        d, f, h = case["dim"], case["ffn"], case["head_dim"]
        q, kv = case["heads"] * h, case["kv"] * h
        block = [(q, d), (kv, d), (kv, d), (d, q), (h,), (h,), (d,), (d,), (f, d), (f, d), (d, f)]
        out = [(case["vocab"], d)] + block * case["layers"] + [(d,)]
    return [s for s in out if len(s) == 2] + [s for s in out if len(s) == 1]


def _layout(case):
    """(offset, elements, shape) of each tensor, and the length of all."""
    places, pos = [], 0
    for s in _shapes(case):
        n = math.prod(s)
        places.append((pos, n, s))
        pos += -(-n // ALIGN) * ALIGN
    return places, pos


def _exponents(x, top, low):
    """For each block of 64 the least e with which its largest finite magnitude is at most ``top`` 2^e, at least ``low``."""
    size = x.view(-1, BLOCK).abs()
    most = torch.where(torch.isfinite(size), size, 0.0).amax(1)
    frac, ex = torch.frexp(most)
    f, t = math.frexp(top)
    return torch.where(most > 0, ex - t + (frac > f), low).clamp(min=low).int()


def _two_to(e):
    return ((e + 127) << 23).view(torch.float32)


def _encode(m, r, bits):
    """(m's codes, exponents, r's codes, exponents) of two fp32 vectors, ``bits`` the hash of each element."""
    e = _exponents(m, 448.0, -117).clamp(max=119)
    y = (m.view(-1, BLOCK) * _two_to(-e)[:, None]).view(-1)
    size = y.abs().clamp(max=448.0)
    base = torch.where(size < 2.0 ** -6, 2.0 ** -6, 0.0)
    raised = (size + base).view(torch.int32) + ((bits & 0xFFFF) * 16 + 8).int()
    size = (raised & ~0xFFFFF).view(torch.float32) - base
    m_codes = torch.where(y < 0, -size, size).to(torch.float8_e4m3fn).view(torch.uint8)
    x = _exponents(r, 30.0 * 2.0 ** 14, -105)
    y = (r.view(-1, BLOCK) * _two_to(-x)[:, None]).view(-1)
    low = y < 16.0
    raised = torch.where(low, y + 16.0, y).view(torch.int32) + ((bits >> 16) * 8 + 4).int()
    codes = (raised >> 19) - torch.where(low, 131 * 16, 130 * 16)
    codes = torch.where(r > 0, codes.clamp(min=1), 0)
    return m_codes, (e + 127).byte(), torch.where(torch.isfinite(r), codes, 255).byte(), (x + 145).byte()


def _decode(m_codes, m_exps, r_codes, r_exps):
    """(m, r) in fp32 of what is held."""
    m = (m_codes.view(torch.float8_e4m3fn).float().view(-1, BLOCK) * _two_to(m_exps.int() - 127)[:, None]).view(-1)
    c = r_codes.int()
    n = torch.where(c < 16, c, (16 + (c & 15)) << ((c >> 4) - 1).clamp(min=0)).float()
    r = (n.view(-1, BLOCK) * _two_to(r_exps.int() - 145)[:, None]).view(-1)
    return m, torch.where(c == 255, math.nan, r)


def _positions(places, total):
    """Each element's place in its own tensor."""
    starts = torch.tensor([o for o, _, _ in places], device="cuda")
    lengths = torch.diff(starts, append=torch.tensor([total], device="cuda"))
    return torch.arange(total, device="cuda") - torch.repeat_interleave(starts, lengths)


def _adamw_inputs(case, seed):
    """Masters, gradients and the moments of the steady state, each in one buffer with zeros between tensors."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    places, total = _layout(case)
    used = torch.zeros(total // 8, 8, dtype=torch.bool, device=dev)
    for o, n, _ in places:
        used.view(-1)[o: o + n] = True
    used = used.view(-1)

    def normal(std):
        return torch.empty(total, device=dev).normal_(0.0, std, generator=g).mul_(used)

    t = {"master": normal(0.02), "grad": normal(1e-3).to(TYPES[case["grads"]])}
    m, r = normal(1e-4), normal(1e-3).abs_().add_(3e-5).mul_(used)
    held = torch.randint(0, 1 << 32, (total,), device=dev, generator=g)
    t["held"] = _encode(m, r, held)
    return t


def _view(flat, offset, shape):
    """A tensor of its own (not an autograd view) over part of ``flat``."""
    return torch.empty(0, dtype=flat.dtype, device=flat.device).set_(flat.untyped_storage(), offset, shape)


def _adamw_optimizer(state):
    """The optimizer that a program keeps, on the prepared tensors."""
    import torchure_amd as ta

    case, t = state["case"], state["t"]
    params = [torch.nn.Parameter(_view(t["master"], o, s)) for o, _, s in state["places"]]
    opt = ta.build_optimizer(torch.nn.ParameterList(params), "adamw",
                             {"lr": LR, "weight_decay": WEIGHT_DECAY, "betas": BETAS, "eps": EPS, "state_bits": 8,
                              "seed": SEED})
    saved = opt.state_dict()
    codes, exps, roots, root_exps = t["held"]
    for i, (o, n, _) in enumerate(state["places"]):
        end = o + -(-n // ALIGN) * ALIGN
        saved["state"][i] = {"step": torch.tensor(float(STEPS_DONE)),
                             "exp_avg": torch.cat([codes[o:end], exps[o // BLOCK: end // BLOCK]]),
                             "exp_avg_sq": torch.cat([roots[o:end], root_exps[o // BLOCK: end // BLOCK]])}
    opt.load_state_dict(saved)
    grads = [_view(t["grad"], o, s) for o, _, s in state["places"]]
    copies = None
    if case["grads"] == "bf16":
        works = ta.attach_bf16_working_params(params)
        for w, g in zip(works, grads):
            w.grad = g
        copies = _view(works[0], 0, (sum(n for _, n, _ in state["places"]),))
    else:
        for p, g in zip(params, grads):
            p.grad = g
    return {"opt": opt, "params": params, "copies": copies}


def _adamw_own(state):
    if "program" not in state:  # built once, kept by the program
        state["program"] = _adamw_optimizer(state)
    program = state["program"]
    program["opt"].step()
    m, r = program["opt"].flat_moments()
    out = {"master": state["t"]["master"], "exp_avg": m, "root": r}
    if program["copies"] is not None:
        out["copies"] = program["copies"]
    return out


def _adamw_plain(state):
    case, t, places = state["case"], state["t"], state["places"]
    with torch.no_grad():
        state["step"] += 1
        step = state["step"]
        bias1, bias2 = 1.0 - BETAS[0] ** step, 1.0 - BETAS[1] ** step
        p, g = t["master"], t["grad"].float()
        decayed = sum(-(-n // ALIGN) * ALIGN for _, n, s in places if len(s) == 2)  # they lie first
        p[:decayed] *= 1.0 - LR * WEIGHT_DECAY
        m, r = _decode(*t["held"])
        m = BETAS[0] * m + (1.0 - BETAS[0]) * g
        r = torch.sqrt(BETAS[1] * (r * r) + (1.0 - BETAS[1]) * (g * g))
        p -= (LR / bias1) * m / (r / math.sqrt(bias2) + EPS)
        bits = _element((state["positions"] * A + _key(SEED, step)) & MASK)
        t["held"] = _encode(m, r, bits)
        m, r = (v.bfloat16() for v in _decode(*t["held"]))
        out = {"master": p, "exp_avg": torch.cat([m[o: o + n] for o, n, _ in places]),
               "root": torch.cat([r[o: o + n] for o, n, _ in places])}
        if case["grads"] == "bf16":
            out["copies"] = torch.cat([p[o: o + n] for o, n, _ in places]).bfloat16()
        return out


def _two_to64(e):
    """2^e in 64 bits to the bit (a power function may be off in its last place)."""
    return ((e.long() + 1023) * (1 << 52)).view(torch.float64)


def _scale64(most, top, low, high):
    """2^e for each block, e the least with most <= top 2^e within [low, high]."""
    e = torch.ceil(torch.log2(most.clamp_min(1e-300) / top)).clamp(-500, 500)
    e = torch.where(_two_to64(e - 1) * top >= most, e - 1, e)  # a logarithm next to a whole number
    e = torch.where(_two_to64(e) * top < most, e + 1, e)
    return _two_to64(e.clamp(low, high))[:, None]


def _hold64(x, scale, mantissa, least, low, u):
    """Magnitudes ``x`` in 64 bits, as blocks, at the places that a format with ``mantissa`` bits and the smallest step
    ``least`` (relative to its block's ``scale``) has, by ``u``."""
    y = x / scale
    _, ex = torch.frexp(y)
    step = _two_to64(ex - 1 - mantissa).clamp_min(least)
    held = torch.floor(y / step + u) * step
    if low:
        held = torch.where(y > 0, held.clamp_min(low), held)
    return held * scale


def _adamw_exact(case, seed):
    t = _adamw_inputs(case, seed)
    places, total = _layout(case)
    codes, exps, roots, root_exps = t["held"]
    step = STEPS_DONE + 1
    bias1, bias2 = 1.0 - BETAS[0] ** step, 1.0 - BETAS[1] ** step
    key = _key(SEED, step)
    out = {"master": torch.zeros(total, dtype=torch.float64, device="cuda"), "exp_avg": [], "root": []}
    e4m3 = torch.arange(256, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn).double()
    lattice = torch.tensor([float(c) if c < 16 else (16.0 + c % 16) * 2.0 ** (c // 16 - 1) for c in range(256)],
                           dtype=torch.float64, device="cuda")
    pieces = [(o, i, min(n, i + (1 << 26)), len(s) == 2) for o, n, s in places for i in range(0, n, 1 << 26)]
    for o, first, last, decay in pieces:
        a, b = o + first, o + -(-last // BLOCK) * BLOCK  # whole blocks; the zeros behind a tensor change none
        m = e4m3[codes[a:b].long()].view(-1, BLOCK) * _two_to64(exps[a // BLOCK: b // BLOCK].long() - 127)[:, None]
        r = lattice[roots[a:b].long()].view(-1, BLOCK) * _two_to64(root_exps[a // BLOCK: b // BLOCK].long() - 145)[:, None]
        g, p = t["grad"][a:b].double().view(-1, BLOCK), t["master"][a:b].double().view(-1, BLOCK)
        m = m + (1.0 - BETAS[0]) * (g - m)
        r = torch.sqrt(r * r + (1.0 - BETAS[1]) * (g * g - r * r))
        if decay:
            p = p - LR * WEIGHT_DECAY * p
        p = p - LR / bias1 * m / (r / math.sqrt(bias2) + EPS)
        out["master"][a: o + last] = p.view(-1)[: last - first]
        where = torch.arange(first, first + b - a, device="cuda")
        bits = _element((where * A + key) & MASK).view(-1, BLOCK)
        del where, p, g
        m = torch.sign(m) * _hold64(m.abs(), _scale64(m.abs().amax(1), 448.0, -117, 119), 3, 2.0 ** -9, 0.0,
                                    ((bits & 0xFFFF) + 0.5) / 65536.0)
        r = _hold64(r, _scale64(r.amax(1), 30.0 * 2.0 ** 14, -105, 500), 4, 1.0, 1.0, ((bits >> 16) + 0.5) / 65536.0)
        out["exp_avg"].append(m.view(-1)[: last - first].clone())
        out["root"].append(r.view(-1)[: last - first].clone())
    out["exp_avg"], out["root"] = torch.cat(out["exp_avg"]), torch.cat(out["root"])
    if case["grads"] == "bf16":
        out["copies"] = torch.cat([out["master"][o: o + n] for o, n, _ in places])
    return out


# ---------------------------------------------------------------------------- the interface


def prepare(case, seed):
    if case["family"] == "adamw8":
        places, total = _layout(case)
        return {"case": case, "t": _adamw_inputs(case, seed), "places": places, "step": STEPS_DONE,
                "positions": _positions(places, total)}
    t = (_norm_inputs if case["family"] == "norm" else _embed_inputs)(case, seed)
    state = {"case": case, "dy": t.pop("dy", None), "t": t, "wanted": []}
    if case["family"] == "norm" and case["grad"]:
        state["wanted"] = [k for k, v in t.items() if v is not None]
        for k in state["wanted"]:
            t[k].requires_grad_()
    elif case["family"] == "embed" and case["mode"] == "train":
        t["weight"].requires_grad_()
    return state


def run(state):
    family = state["case"]["family"]
    if own:
        return {"norm": _norm_own, "embed": _embed_own, "adamw8": _adamw_own}[family](state)
    return {"norm": _norm_plain, "embed": _embed_plain, "adamw8": _adamw_plain}[family](state)


def exact(case, seed):
    return {"norm": _norm_exact, "embed": _embed_exact, "adamw8": _adamw_exact}[case["family"]](case, seed)


SIZE = {"bf16": 2, "fp32": 4}


def _different(case):
    """How many ids occur, on average."""
    n, v = case["tokens"], case["vocab"]
    edges = torch.arange(v + 1, dtype=torch.float64).div_(v).pow_(0.25)
    drawn = n - n // 3 if case["padding"] else n
    return int(round(float((1.0 - (1.0 - edges.diff()).pow(drawn)).sum())))


def work(case):
    if case["family"] == "norm":
        n, d = case["rows"], case["dim"]
        x, y, w = SIZE[case["x"]], SIZE[case["out"]], SIZE[case["weight"]]
        params = d * w * (2 if case["bias"] and case["kind"] == "layer" else 1)
        moved = n * d * (x + y) + params
        if case["grad"]:  # the output's gradient in, the others out
            moved += n * d * (y + x) + params
        return {"bytes": moved, "flops": n * d * (20 if case["grad"] else 7)}
    if case["family"] == "embed":
        n, d, v = case["tokens"], case["dim"], case["vocab"]
        w, y = SIZE[case["weight"]], SIZE[case["out"]]
        rows = _different(case) * d * w
        moved = 8 * n + rows + n * d * y
        if case["mode"] != "forward":  # the gradients in, the table's out (only the rows that occur, where it is added to)
            moved += n * d * y + (v * d * w if case["mode"] == "train" else 2 * rows)
        return {"bytes": moved, "flops": n * d * (1 if case["mode"] == "forward" else 2)}
    n = sum(math.prod(s) for s in _shapes(case))
    # gradients in, masters and both moments in and out, the copies out, the moments' values out
    held = 4 * (1 + 1 / BLOCK)
    per = SIZE[case["grads"]] + 8 + held + (2 if case["grads"] == "bf16" else 0) + 4
    return {"bytes": int(n * per), "flops": 30 * n}
