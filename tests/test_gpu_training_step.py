"""The operators of a training step as a model runs them together: a table that is the head's weight too, two blocks of norms, heads'
norms, products and a gated feed-forward on an fp32 residual stream, the fused loss, the clip and AdamW on 8-bit moments with
bf16 working copies. What each norm and the embedding made there, and their gradients there, are held against 64 bits
from what they were given there; the step against the same step in 64 bits."""

from __future__ import annotations

import pytest
import torch

import torchure_amd as ta
from tests.test_gpu_adamw8 import BETAS, LR, SEED, check_step, f64, moments
from tests.test_gpu_norm import BF16, DEV, F32, HALF, U, close, want
from torchure_amd.loss.fused_linear_ce import fused_linear_cross_entropy

pytestmark = pytest.mark.gpu

VOCAB, DIM, HEADS, FFN, PAD, SCALE, WD = 501, 136, 4, 200, 7, 11.6619, 0.1


class Model:
    def __init__(self, layer_norm, seed=0):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.nn.Parameter((torch.randn(*s, generator=g) * 0.05).to(DEV))  # noqa: E731
        one = lambda *s: torch.nn.Parameter((1 + 0.1 * torch.randn(*s, generator=g)).to(DEV))  # noqa: E731
        self.layer_norm, self.blocks, self.seen = layer_norm, 2, []
        self.p = {"table": r(VOCAB, DIM), "last": one(DIM)}
        for i in range(self.blocks):
            self.p |= {f"{i}.first": one(DIM), f"{i}.head": one(DIM // HEADS), f"{i}.second": one(DIM), f"{i}.in": r(DIM, DIM),
                       f"{i}.out": r(DIM, DIM), f"{i}.gate": r(FFN, DIM), f"{i}.up": r(FFN, DIM), f"{i}.down": r(DIM, FFN)}
            if layer_norm:
                self.p |= {f"{i}.bias": r(DIM)}
        self.params = list(self.p.values())
        self.works = ta.attach_bf16_working_params(self.params)
        self.w = dict(zip(self.p, self.works))

    def norm(self, x, name, bias=None, dtype=BF16):
        """The norm of aliases of its own, whose gradients are then this call's alone."""
        t = {"x": x.view_as(x), "weight": self.w[name].view_as(self.w[name]), "bias": None}
        if bias is not None:
            t["bias"] = self.w[bias].view_as(self.w[bias])
            y = ta.layer_norm(t["x"], t["weight"], t["bias"], 1e-5, dtype)
        else:
            y = ta.rms_norm(t["x"], t["weight"], 1e-6, dtype)
        self.seen.append((name, t, y))
        return y

    def loss(self, ids, labels, tied):
        """Of a table's gradient by autograd, or (``tied``) left for embedding_grad_."""
        self.seen = []
        table = self.w["table"].detach() if tied else self.w["table"].view_as(self.w["table"])
        h = ta.embedding(ids, table, SCALE, PAD, F32)
        if tied:
            h.requires_grad_()
        self.embedded = table, h
        for i in range(self.blocks):
            n = self.norm(h, f"{i}.first")
            q = ta.fused_linear(n, self.w[f"{i}.in"])
            q = self.norm(q.unflatten(-1, (HEADS, DIM // HEADS)), f"{i}.head").flatten(-2)
            h = ta.fused_linear(q, self.w[f"{i}.out"], residual=h)
            n = self.norm(h, f"{i}.second", f"{i}.bias" if self.layer_norm else None)
            h = ta.swiglu_mlp(n, self.w[f"{i}.gate"], self.w[f"{i}.up"], self.w[f"{i}.down"], residual=h)
        return fused_linear_cross_entropy(self.norm(h, "last"), self.w["table"], labels)

    def keep_grads(self):
        for _, t, y in self.seen:
            for v in (*t.values(), y):
                if v is not None:
                    v.retain_grad()
        for v in self.embedded:
            if v.requires_grad and not v.is_leaf:
                v.retain_grad()

    def optimizer(self):
        groups = [{"params": [p for p in self.params if p.dim() >= 2], "weight_decay": WD},
                  {"params": [p for p in self.params if p.dim() < 2], "weight_decay": 0.0}]
        return ta.AdamW(groups, lr=LR, betas=BETAS, eps=1e-8, state_bits=8, seed=SEED)

    def zero_grad(self, opt):
        opt.zero_grad()
        for w in self.works:
            w.grad = None


def batch(seed, rows=3, length=47):
    """A padded batch: one row whole, one of which a third is there, one of padding alone."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(8, VOCAB, (rows, length), generator=g)
    ids[1, length // 3:] = PAD
    ids[2] = PAD
    labels = torch.where(ids == PAD, -100, ids).roll(-1, 1)
    return ids.to(DEV), labels.to(DEV)


def table_sums(ids, dy):
    """(what the tokens add to the table, the bound of its fp32 sums): a sum as deep as there are tokens."""
    flat, rows = ids.reshape(-1), dy.reshape(-1, DIM).double()
    rows = rows * (flat != PAD).double()[:, None]
    zero = torch.zeros(VOCAB, DIM, dtype=torch.float64, device=DEV)
    return SCALE * zero.index_add(0, flat, rows), (len(flat) + 2) * U * SCALE * zero.index_add(0, flat, rows.abs())


@pytest.mark.parametrize("layer_norm", [False, True])
@pytest.mark.parametrize("tied", [False, True])
def test_steps(layer_norm, tied):
    model = Model(layer_norm)
    opt = model.optimizer()
    for step in (1, 2, 3):
        ids, labels = batch(step)
        loss = model.loss(ids, labels, tied)
        assert torch.isfinite(loss)
        model.keep_grads()
        loss.backward()
        for name, t, y in model.seen:
            layer = t["bias"] is not None
            found = want(t, y.grad, layer, 1e-5 if layer else 1e-6, y.dtype)
            close(y, *found["y"], name)
            for k, v in t.items():
                if v is not None:
                    close(v.grad, *found[k], f"{name}: gradient of {k}")
        table, h = model.embedded
        y = SCALE * table.double()[ids]
        close(h, y, 2 * U * y.abs(), "lookup")  # the scale's rounding and the product's
        sums, err = table_sums(ids, h.grad)
        if tied:
            head = model.w["table"].grad.clone()
            ta.embedding_grad_(model.w["table"].grad, ids, h.grad, SCALE, PAD)
            sums = sums + head.double()
            close(model.w["table"].grad, sums, err + HALF[BF16] * (sums.abs() + err) + U * sums.abs(), "table")
            rest = torch.ones(VOCAB, dtype=torch.bool, device=DEV)
            rest[ids[ids != PAD]] = False
            assert torch.equal(model.w["table"].grad[rest], head[rest])
        else:
            close(table.grad, sums, err + HALF[BF16] * (sums.abs() + err), "table")
        grads = [f64(w.grad) for w in model.works]
        before = [f64(p) for p in model.params]
        was = [moments(opt, p) if step > 1 else (torch.zeros(p.numel()).double(),) * 2 for p in model.params]
        norm = ta.clip_grad_norm(model.params, None, 0.5)
        coef = torch.clamp(0.5 / (norm + 1e-6), max=1.0).double().cpu()
        opt.step()
        for i, p in enumerate(model.params):
            check_step(f64(p), before[i], was[i], moments(opt, p), grads[i] * coef, step, p.dim() >= 2, wd=WD,
                       copy_=model.works[i].detach().cpu().reshape(-1))
        model.zero_grad(opt)


def test_the_same_bits_twice():
    """Two runs of three steps end in the same masters and moments: no operator's sums change their order."""
    ends = []
    for _ in range(2):
        model = Model(True, seed=5)
        opt = model.optimizer()
        for step in (1, 2, 3):
            ids, labels = batch(step)
            loss = model.loss(ids, labels, False)
            loss.backward()
            ta.clip_grad_norm(model.params, None, 0.5)
            opt.step()
            model.zero_grad(opt)
        ends.append([p.detach().clone() for p in model.params] + list(opt.flat_moments()))
    for a, b in zip(*ends):
        assert torch.equal(a, b)


def test_captured():
    """Lookup, norms and their gradients, and the step, in one graph: every replay is what eager calls give."""
    def passes(model, ids, dy):
        h = ta.embedding(ids, model.w["table"], SCALE, PAD, F32)
        n = ta.layer_norm(ta.rms_norm(h, model.w["0.first"], dtype=F32), model.w["0.second"], model.w["0.bias"], dtype=BF16)
        leaves = [model.w[k] for k in ("table", "0.first", "0.second", "0.bias")]
        return n, torch.autograd.grad(n, leaves, dy)

    model, twin = Model(True, seed=2), Model(True, seed=2)
    ids, _ = batch(9)
    dy = torch.randn(*ids.shape, DIM, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV).to(BF16)
    names = ("table", "0.first", "0.second", "0.bias")

    def prepared(m):
        opt = ta.AdamW([m.p[k] for k in names], lr=LR, betas=BETAS, state_bits=8, seed=SEED)
        for k in names:
            m.w[k].grad = torch.zeros_like(m.w[k])
        opt.init_state()
        launch, = opt.plan_step()
        return launch

    launches = [prepared(m) for m in (model, twin)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        passes(model, ids, dy)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        n, grads = passes(model, ids, dy)
        for k, g in zip(names, grads):
            model.w[k].grad.copy_(g)
        launches[0]()
    for k in range(3):
        ids.copy_(batch(20 + k)[0])
        graph.replay()
        torch.cuda.synchronize()
        m, eager = passes(twin, ids, dy)
        assert torch.equal(n, m), k
        for name, a, b in zip(names, grads, eager):
            assert torch.equal(a, b), (k, name)
            twin.w[name].grad.copy_(b)
        launches[1]()
        for name in names:
            assert torch.equal(model.p[name], twin.p[name]) and torch.equal(model.w[name], twin.w[name]), (k, name)
