"""Performance cases of the block's products: linear layers with everything that follows them, the
gated feed-forward, and activations held in 8 bits between forward and backward.

Three families, each with listed cases and a generator of further cases of the same ranges:

- ``linear``: ``y = act(x W^T + b) + r``, forward alone or with all its gradients;
- ``mlp``: ``y = (silu(x Wg^T) * (x Wu^T)) Wd^T + r``, forward alone or with all its gradients;
- ``held``: a tensor put into 8 bits and read back, as those two do with what they keep for the
  backward pass.

Definitions, for both sides. Operands are bf16. ``held="e4m3"`` keeps a matrix as e4m3 values with one
power of two for each 32 x 32 block: ``2^e``, e the least exponent with which the block's largest
finite magnitude is at most 448, clamped to [-117, 119]; values round to nearest even, and values
past 448 * 2^e are held as that. ``held="bf16"`` rounds to bf16. The forward pass uses the values
themselves; the gradients use what was held: the linear layer's input and pre-activation, the
feed-forward's input, gate and up products, and the product of the activated gate with up made from
those two again. That product is a bf16 matrix, also in the forward pass.

``listed()`` and ``draw(rng)`` give cases (plain dicts), ``prepare`` what a program has in hand before
the call, ``run`` one pass, ``exact`` the same outputs in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")


def listed():
    return [
        # One token through a projection: a generated sample or a probe during evaluation. Latency.
        {"name": "linear-token", "family": "linear", "rows": 1, "inp": 1024, "out": 2816, "act": "silu", "bias": True,
         "residual": "none", "held": "bf16", "grad": False},
        # The attention output projection of the 0.6B shape, training: fp32 residual stream.
        {"name": "linear-o-0.6b", "family": "linear", "rows": 8192, "inp": 2048, "out": 1024, "act": "none",
         "bias": False, "residual": "fp32", "held": "bf16", "grad": True},
        # A plain two-layer feed-forward's first product, sizes that no tile divides, odd width.
        {"name": "linear-odd-gelu", "family": "linear", "rows": 1237, "inp": 1000, "out": 777, "act": "gelu_tanh",
         "bias": True, "residual": "bf16", "held": "bf16", "grad": True},
        # The 4B shape's widening product with what it keeps in 8 bits.
        {"name": "linear-4b-silu-e4m3", "family": "linear", "rows": 8192, "inp": 2560, "out": 9728, "act": "silu",
         "bias": True, "residual": "none", "held": "e4m3", "grad": True},
        # The 4B shape's narrowing product over a validation batch.
        {"name": "linear-4b-down-eval", "family": "linear", "rows": 8192, "inp": 9728, "out": 2560, "act": "none",
         "bias": False, "residual": "bf16", "held": "bf16", "grad": False},
        # A short sequence's hidden states put into 8 bits and read back: launches.
        {"name": "held-short", "family": "held", "rows": 128, "inp": 1024, "dtype": "bf16"},
        # A whole batch's gate products at the 4B shape.
        {"name": "held-4b", "family": "held", "rows": 16384, "inp": 9728, "dtype": "bf16"},
        # fp32 hidden states (a norm's output), rows and columns off every block.
        {"name": "held-odd-fp32", "family": "held", "rows": 6001, "inp": 1237, "dtype": "fp32"},
        # One token through the 0.6B shape's feed-forward.
        {"name": "mlp-token", "family": "mlp", "rows": 1, "dim": 1024, "ffn": 2816, "residual": "bf16",
         "held": "bf16", "grad": False},
        # The 0.6B shape's feed-forward, training step of 8192 tokens.
        {"name": "mlp-0.6b", "family": "mlp", "rows": 8192, "dim": 1024, "ffn": 2816, "residual": "bf16",
         "held": "bf16", "grad": True},
        # A packed batch without padding, sizes off every tile, kept in 8 bits.
        {"name": "mlp-odd-e4m3", "family": "mlp", "rows": 1999, "dim": 1000, "ffn": 2730, "residual": "none",
         "held": "e4m3", "grad": True},
        # The 4B shape's feed-forward, kept in 8 bits: the largest.
        {"name": "mlp-4b-e4m3", "family": "mlp", "rows": 8192, "dim": 2560, "ffn": 9728, "residual": "bf16",
         "held": "e4m3", "grad": True},
    ]


def _log_uniform(rng: random.Random, lo: float, hi: float) -> int:
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def _width(rng, lo, hi):
    """A layer's width: mostly whole tiles, some only whole vectors, some anything."""
    n, kind = _log_uniform(rng, lo, hi), rng.random()
    return n if kind < 0.15 else -(-n // 8) * 8 if kind < 0.35 else max(64, n // 64 * 64)


def draw(rng: random.Random):
    family = rng.choice(["linear", "linear", "linear", "mlp", "mlp", "held"])
    if family == "held":
        return {"family": family, "rows": _log_uniform(rng, 1, 16384), "inp": _log_uniform(rng, 32, 9728),
                "dtype": rng.choice(["bf16", "bf16", "fp32"])}
    grad = rng.random() < 0.7
    rows = _log_uniform(rng, 64 if grad else 1, 12000)
    if rows > 64 and rng.random() < 0.4:  # batches padded to a round number of tokens
        rows = -(-rows // 128) * 128
    case = {"family": family, "rows": rows}
    if family == "linear":
        case.update(inp=_width(rng, 128, 9728), out=_width(rng, 128, 9728), act=rng.choice(ACTS),
                    bias=rng.random() < 0.5, residual=rng.choice(["none", "bf16", "fp32"]))
        each = 2 * case["inp"] * case["out"]
    else:
        case.update(dim=_width(rng, 128, 2560), ffn=_width(rng, 256, 9728), residual=rng.choice(["none", "bf16"]))
        each = 6 * case["dim"] * case["ffn"]
    case.update(held=rng.choice(["bf16", "e4m3"]), grad=grad)
    case["rows"] = max(1, min(rows, int(3.6e12 / ((3 if grad else 1) * each))))
    return case


# ---------------------------------------------------------------------------- inputs


def _inputs(case, seed):
    """Hidden states of about unit size whose channels differ in spread and of which a few rows are
    large, weights at their initial spread, the gradient of a mean loss's size."""
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return torch.empty(shape, device=dev).normal_(0.0, std, generator=g)

    n = case["rows"]
    d = case["dim"] if case["family"] == "mlp" else case["inp"]
    x = normal(n, d) * normal(d, std=0.5).exp_()
    x[torch.randint(0, n, (max(1, n // 1000),), device=dev, generator=g)] *= 30.0
    if case["family"] == "held":
        x[torch.randint(0, n, (max(1, n // 100),), device=dev, generator=g)] = 0.0  # padding
        return {"x": x if case["dtype"] == "fp32" else x.bfloat16()}
    t = {"x": x.bfloat16()}
    if case["family"] == "linear":
        out = case["out"]
        t["weight"] = normal(out, d, std=d ** -0.5).bfloat16()
        t["bias"] = normal(out, std=0.1).bfloat16() if case["bias"] else None
    else:
        out = d
        t["w_gate"] = normal(case["ffn"], d, std=d ** -0.5).bfloat16()
        t["w_up"] = normal(case["ffn"], d, std=d ** -0.5).bfloat16()
        t["w_down"] = normal(d, case["ffn"], std=case["ffn"] ** -0.5).bfloat16()
    res = {"none": None, "bf16": torch.bfloat16, "fp32": torch.float32}[case["residual"]]
    t["residual"] = None if res is None else normal(n, out).to(res)
    if case["grad"]:
        t["dy"] = normal(n, out, std=1e-3).to(res or torch.bfloat16)
    return t


def prepare(case, seed):
    t = _inputs(case, seed)
    state = {"case": case, "dy": t.pop("dy", None), "t": t, "wanted": []}
    if state["dy"] is not None:
        state["wanted"] = [k for k, v in t.items() if v is not None]
        for k in state["wanted"]:
            t[k].requires_grad_()
    return state


# ---------------------------------------------------------------------------- one pass


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(state):
    import torchure_amd as ta

    case, t = state["case"], state["t"]
    if case["family"] == "held":
        return {"x": ta.dequantize_activation(ta.quantize_activation(t["x"]))}
    checkpoint = None if case["held"] == "bf16" else case["held"]
    with torch.set_grad_enabled(case["grad"]):
        if case["family"] == "linear":
            y = ta.fused_linear(t["x"], t["weight"], t["bias"], residual=t["residual"], activation=case["act"],
                                checkpoint=checkpoint)
        else:
            y = ta.swiglu_mlp(t["x"], t["w_gate"], t["w_up"], t["w_down"], residual=t["residual"],
                              checkpoint=checkpoint)
    if not case["grad"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [t[k] for k in state["wanted"]], state["dy"])
    return {"y": y.detach(), **{"d_" + k: v for k, v in zip(state["wanted"], grads)}}


def _act(name, z):
    if name == "none":
        return z
    if name == "relu":
        return torch.clamp_min(z, 0.0)
    if name == "silu":
        return z / (1.0 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    u = math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)
    return 0.5 * z * (1.0 + torch.tanh(u))


def _act_grad(name, z):
    if name == "none":
        return torch.ones_like(z)
    if name == "relu":
        return (z > 0).to(z.dtype)
    if name == "silu":
        s = 1.0 / (1.0 + torch.exp(-z))
        return s * (1.0 + z * (1.0 - s))
    if name == "gelu":
        return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    u = torch.tanh(c * (z + 0.044715 * z * z * z))
    return 0.5 * (1.0 + u) + 0.5 * z * (1.0 - u * u) * c * (1.0 + 3 * 0.044715 * z * z)


def _blocks(x):
    """(padded copy as row block x 32 x column block x 32, rows, columns)."""
    n, d = x.shape
    np_, dp = -(-n // 32) * 32, -(-d // 32) * 32
    padded = torch.zeros(np_, dp, dtype=x.dtype, device=x.device)
    padded[:n, :d] = x
    return padded.view(np_ // 32, 32, dp // 32, 32)


def _e4m3(x):
    """What 8 bits hold of the fp32 matrix ``x``."""
    b = _blocks(x)
    size = b.abs()
    most = torch.where(torch.isfinite(size), size, 0.0).amax(dim=(1, 3), keepdim=True)
    frac, ex = torch.frexp(most)  # most = frac 2^ex, frac in [0.5, 1): 448 = 0.875 2^9
    e = (ex - 9 + (frac > 0.875)).clamp(-117, 119).int()
    up, down = (((127 + s * e) << 23).view(torch.float32) for s in (1, -1))  # 2^e, 2^-e, to the bit
    values = (b * down).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float() * up
    return values.reshape(values.shape[0] * 32, -1)[: x.shape[0], : x.shape[1]]


def _held(kind, x):
    return x.bfloat16().float() if kind == "bf16" else _e4m3(x)


def _run_plain(state):
    with torch.no_grad():
        case, t, dy = state["case"], state["t"], state["dy"]
        if case["family"] == "held":
            return {"x": _e4m3(t["x"].float()).to(t["x"].dtype)}
        x = t["x"].float()
        res, res_type = 0.0, torch.bfloat16
        if t["residual"] is not None:
            res, res_type = t["residual"].float(), t["residual"].dtype
        if case["family"] == "linear":
            w = t["weight"].float()
            z = x @ w.t()
            if t["bias"] is not None:
                z = z + t["bias"].float()
            out = {"y": (_act(case["act"], z) + res).to(res_type)}
            if not case["grad"]:
                return out
            dz = dy.float() * _act_grad(case["act"], _held(case["held"], z))
            out["d_x"] = (dz @ w).bfloat16()
            out["d_weight"] = (dz.t() @ _held(case["held"], x)).bfloat16()
            if t["bias"] is not None:
                out["d_bias"] = dz.sum(0).bfloat16()
        else:
            wg, wu, wd = (t[k].float() for k in ("w_gate", "w_up", "w_down"))
            gate, up = x @ wg.t(), x @ wu.t()
            h = (_act("silu", gate) * up).bfloat16().float()
            out = {"y": (h @ wd.t() + res).to(res_type)}
            if not case["grad"]:
                return out
            gate, up = _held(case["held"], gate), _held(case["held"], up)
            a = _act("silu", gate)
            dyf = dy.float()
            dh = dyf @ wd
            d_gate, d_up = dh * up * _act_grad("silu", gate), dh * a
            xh = _held(case["held"], x)
            out["d_x"] = (d_gate @ wg + d_up @ wu).bfloat16()
            out["d_w_gate"] = (d_gate.t() @ xh).bfloat16()
            out["d_w_up"] = (d_up.t() @ xh).bfloat16()
            out["d_w_down"] = (dyf.t() @ (a * up).bfloat16().float()).bfloat16()
        if t["residual"] is not None:
            out["d_residual"] = dy
        return out


# ---------------------------------------------------------------------------- in 64 bits


def _two_to(e):
    """2^e in 64 bits to the bit (a power function may be off in its last place)."""
    return ((e.long() + 1023) * (1 << 52)).view(torch.float64)


def _exact_e4m3(x):
    """The 8-bit format of a matrix in 64 bits by its definition: the block's exponent from
    logarithms, rounding to a whole number of the last place's steps."""
    b = _blocks(x)
    most = torch.where(torch.isfinite(b), b, torch.zeros_like(b)).abs().amax(dim=(1, 3), keepdim=True)
    e = torch.ceil(torch.log2(torch.clamp_min(most, 1e-300) / 448.0))
    e = e.clamp(-500, 500)
    e = torch.where(_two_to(e - 1) * 448.0 >= most, e - 1, e)  # a logarithm next to a whole number
    e = torch.where(_two_to(e) * 448.0 < most, e + 1, e)
    scale = _two_to(e.clamp(-117, 119))
    v = (b / scale).clamp(-448.0, 448.0)
    _, ex = torch.frexp(v.abs())
    step = _two_to(torch.clamp_min(ex - 1, -6) - 3)
    v = torch.round(v / step) * step * scale
    return v.reshape(v.shape[0] * 32, -1)[: x.shape[0], : x.shape[1]]


def _exact_held(case, x):
    return x.bfloat16().double() if case["held"] == "bf16" else _exact_e4m3(x)


def _phi(z):
    return torch.special.erfc(z * -(0.5 ** 0.5)) * 0.5


def _exact_act(name, z):
    """(value, derivative) in 64 bits."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, 0.0 * z), torch.where(z > 0, 1.0, 0.0).double()
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    if name == "gelu":
        return z * _phi(z), _phi(z) + z * torch.exp(z * z * -0.5) / math.sqrt(2.0 * math.pi)
    k = 2.0 * math.sqrt(2.0 / math.pi)  # (1 + tanh(u)) / 2 = sigmoid(2 u)
    s = torch.sigmoid(k * (z + 0.044715 * z ** 3))
    return z * s, s + z * s * (1.0 - s) * k * (1.0 + 0.134145 * z ** 2)


def exact(case, seed):
    t = {k: v if v is None else v.double() for k, v in _inputs(case, seed).items()}
    if case["family"] == "held":
        return {"x": _exact_e4m3(t["x"])}
    x, dy, res = t["x"], t.get("dy"), t["residual"]
    if case["family"] == "linear":
        z = torch.mm(x, t["weight"].t())
        if t["bias"] is not None:
            z += t["bias"]
        y = _exact_act(case["act"], z)[0]
        grads = {}
        if dy is not None:
            dz = _exact_act(case["act"], _exact_held(case, z))[1] * dy
            grads = {"d_x": torch.mm(dz, t["weight"]), "d_weight": torch.mm(dz.t(), _exact_held(case, x))}
            if t["bias"] is not None:
                grads["d_bias"] = torch.mv(dz.t(), torch.ones_like(dz[:, 0]))
    else:
        gate, up = torch.mm(x, t["w_gate"].t()), torch.mm(x, t["w_up"].t())
        h = (_exact_act("silu", gate)[0] * up).bfloat16().double()
        y = torch.mm(h, t["w_down"].t())
        grads = {}
        if dy is not None:
            gate, up = _exact_held(case, gate), _exact_held(case, up)
            a, slope = _exact_act("silu", gate)
            dh = torch.mm(dy, t["w_down"])
            grads = {"d_w_down": torch.mm(dy.t(), (a * up).bfloat16().double())}
            d_gate, d_up = dh * slope * up, dh * a
            grads["d_x"] = torch.mm(d_gate, t["w_gate"]).addmm_(d_up, t["w_up"])
            xh = _exact_held(case, x)
            grads["d_w_gate"], grads["d_w_up"] = torch.mm(d_gate.t(), xh), torch.mm(d_up.t(), xh)
    out = {"y": y if res is None else y + res, **grads}
    if dy is not None and res is not None:
        out["d_residual"] = dy
    return out


# ---------------------------------------------------------------------------- what a pass cannot do without


def work(case):
    n = case["rows"]
    if case["family"] == "held":  # in, the 8-bit values out and in, the values out
        size = n * case["inp"]
        return {"bytes": size * (2 * (2 if case["dtype"] == "bf16" else 4) + 2), "flops": 4 * size}
    res = {"none": 0, "bf16": 2, "fp32": 4}[case["residual"]]
    if case["family"] == "linear":
        d, out = case["inp"], case["out"]
        weights, bias, products = d * out, out if case["bias"] else 0, 2 * n * d * out
    else:
        d = out = case["dim"]
        weights, bias, products = 3 * d * case["ffn"], 0, 6 * n * d * case["ffn"]
    moved = 2 * (n * d + weights + bias) + n * out * (res + (res or 2))
    if case["grad"]:  # the output's gradient in, the others out; the residual's is the output's
        moved += 2 * (n * d + weights + bias) + n * out * (res or 2)
    return {"bytes": moved, "flops": products * (3 if case["grad"] else 1)}
