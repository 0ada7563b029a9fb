"""The linear layers and the gated feed-forward among a program's other tensors: results that are changed in
place afterwards, operands that are negated views, kept tensors that hooks move, and parts of the
gradients. Bit for bit against the same calls without that."""

from __future__ import annotations

import pytest
import torch

import test_gpu_linear as T
import torchure_amd as ta
from test_gpu_linear_calls import BF16, DEV, F32, on_device, same

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("lead", [(), (5,), (2, 3), (2, 1, 3)])
def test_results_changed_in_place(lead, checkpoint):
    """y.mul_(2).add_(r) gives y's gradients twice, for any number of dimensions."""
    rows = torch.Size(lead).numel()
    t, dy = T.linear_case(rows, 40, 48, "silu", BF16, F32, checkpoint, seed=30)
    m, mdy = T.mlp_case(rows, 40, 56, 48, None, seed=30)
    for call, args, dy in ((lambda x, w, b, r: ta.fused_linear(x, w, b, r, "silu", checkpoint), on_device(t), dy),
                           (lambda x, *w: ta.swiglu_mlp(x, *w[:3], None, checkpoint), on_device(m), mdy)):
        args = {k: v if v is None or k not in ("x", "residual") else v.detach().view(*lead, v.shape[-1]).requires_grad_()
                for k, v in args.items()}
        wanted = [v for v in args.values() if v is not None]
        dy = dy.to(DEV).view(*lead, 48)
        y = call(*args.values())
        want = torch.autograd.grad(y, wanted, 2 * dy)
        z = call(*args.values())
        assert not z._is_view()
        z.mul_(2).add_(dy)
        same(z, (y.detach() * 2).add_(dy))
        for a, b in zip(torch.autograd.grad(z, wanted, dy), want):
            same(a, b)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
@pytest.mark.parametrize("rows,dim,ffn,out", [(1, 8, 1, 8), (33, 24, 7, 16), (70, 40, 77, 24), (300, 64, 640, 40), (1001, 72, 1237, 33)])
def test_the_down_projections_gradient_alone(rows, dim, ffn, out, checkpoint):
    """The gated product made again from what is held: the bits of the call with all gradients."""
    t, dy = T.mlp_case(rows, dim, ffn, out, None, seed=31)
    d, dy = on_device(t), dy.to(DEV)
    args = [d[k] for k in ("x", "w_gate", "w_up", "w_down")]
    y = ta.swiglu_mlp(*args, None, checkpoint)
    want = torch.autograd.grad(y, args, dy)[3]
    z = ta.swiglu_mlp(*(v.detach() for v in args[:3]), args[3], None, checkpoint)
    same(z, y)
    got, = torch.autograd.grad(z, args[3], dy)
    same(got, want)


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_the_down_projections_gradient_alone_keeps_and_makes_nothing_else(checkpoint):
    """Kept: gate and up. In the backward pass: their product and the gradient. (No operand of an fp32
    w_down, no gradients of gate and up, which are three times as many bytes as that product.)"""
    n, dim, ffn = 2048, 256, 1024
    g = torch.Generator(device=DEV).manual_seed(32)
    x, wg, wu = (torch.randn(s, device=DEV, generator=g).to(BF16) for s in ((n, dim), (ffn, dim), (ffn, dim)))
    wd = torch.randn(dim, ffn, device=DEV, generator=g).requires_grad_()
    dy = torch.ones(n, dim, dtype=BF16, device=DEV)

    def step():
        before = torch.cuda.memory_allocated()
        y = ta.swiglu_mlp(x, wg, wu, wd, None, checkpoint)
        kept = torch.cuda.memory_allocated() - before - y.numel() * 2
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        torch.autograd.grad(y, wd, dy)
        return kept, torch.cuda.max_memory_allocated() - held

    step()
    torch.cuda.synchronize()
    kept, more = step()
    slack = 1 << 17
    assert kept <= (2 * n * ffn * 2 if checkpoint is None else 2 * (n * ffn + n * ffn // 1024)) + slack
    from torchure_amd import _native
    split = _native.lib().tm_lin_workspace_bytes(_native.TM_LIN_GRAD_W, n, ffn, dim, 0)
    assert more <= n * ffn * 2 + wd.numel() * 4 + split + slack


@pytest.mark.parametrize("held", [1, 2])
@pytest.mark.parametrize("rows,cols", [(1, 1), (37, 29), (64, 64), (65, 300)])
def test_the_gated_product_writes_its_rows_only(rows, cols, held):
    from torchure_amd import _native

    g = torch.Generator().manual_seed(33)
    z = [T.grid_values(g, (rows, cols), 0.25, 12) for _ in range(2)]
    if held == 1:
        kept = [torch.zeros(rows, -(-cols // 8) * 8, dtype=BF16, device=DEV) for _ in z]
        for k, v in zip(kept, z):
            k[:, :cols] = v.to(DEV)
        exps = [None, None]
    else:
        q = [ta.quantize_activation(v.to(DEV)) for v in z]
        kept, exps = [v.values for v in q], [v.exponents for v in q]
    width = -(-cols // 8) * 8
    room = torch.full((rows + 4, width + 16), 7.0, dtype=BF16, device=DEV)
    _native.check(_native.lib().tm_held_gate(
        room[2:, 8:].data_ptr(), width + 16, kept[0].data_ptr(), kept[1].data_ptr(), *(None if e is None else e.data_ptr() for e in exps),
        kept[0].shape[1], held, rows, cols, _native.stream_handle(torch.device(DEV, 0))), "tm_held_gate")
    inside = torch.zeros(room.shape, dtype=torch.bool, device=DEV)
    inside[2: 2 + rows, 8: 8 + width] = True
    assert bool((room[~inside] == 7.0).all()) and not room[2: 2 + rows, 8 + cols: 8 + width].any()
    gate, up = (T.held64("e4m3" if held == 2 else None, v.double()) for v in z)
    want = T.act64("silu", gate) * up
    T.close(room[2: 2 + rows, 8: 8 + cols], want, want.abs() * 2.0 ** -8 + up.abs() * gate.abs().clamp_min(1) * T.ACT_ERR, "silu(g) u")


@pytest.mark.parametrize("out", [1, 48])
def test_operands_that_are_negated_views(out):
    """z.conj().imag is a view of z's memory with a flag for the sign."""
    g = torch.Generator().manual_seed(34)

    def negated(*shape):
        v = torch.complex(torch.zeros(shape), torch.randn(shape, generator=g)).to(DEV).conj().imag
        assert v.is_neg()
        return v

    x, w, m = (torch.randn(s, generator=g).to(BF16).to(DEV) for s in ((20, 40), (out, 40), (40, 40)))
    b, r, n, h = negated(out), negated(20, out), torch._neg_view(w), torch._neg_view(x)
    clones = [v.clone().resolve_neg() for v in (b, r, n, h)]
    for act in (None, "silu"):
        same(ta.fused_linear(h, n, b, r, act), ta.fused_linear(clones[3], clones[2], clones[0], clones[1], act))
    same(ta.swiglu_mlp(h, m, m, n, r), ta.swiglu_mlp(clones[3], m, m, clones[2], clones[1]))
    a, c = ta.quantize_activation(r), ta.quantize_activation(clones[1])
    assert torch.equal(a.values, c.values) and torch.equal(a.exponents, c.exponents)
    w = w.requires_grad_()
    y = ta.fused_linear(x, w, None, clones[1])
    same(torch.autograd.grad(y, w, r, retain_graph=True)[0], torch.autograd.grad(y, w, clones[1])[0])


@pytest.mark.parametrize("checkpoint", [None, "e4m3"])
def test_kept_tensors_that_come_back_in_other_strides(checkpoint):
    """Hooks that give some of what is kept back in rows of their own, wider ones or columns."""
    t, dy = T.linear_case(40, 64, 48, "silu", BF16, None, checkpoint, seed=35)
    m, mdy = T.mlp_case(40, 64, 96, 48, None, seed=35)
    d, dy, m, mdy = on_device(t), dy.to(DEV), on_device(m), mdy.to(DEV)
    for name in ("w_gate", "w_up"):  # equal strides
        room = torch.zeros(96, 192, dtype=BF16, device=DEV)
        room[:, 64:128] = m[name].detach()
        m[name] = room[:, 64:128].requires_grad_()

    def wider(v):
        return torch.empty(v.shape[0], v.shape[1] + 32, dtype=v.dtype, device=DEV)[:, : v.shape[1]].copy_(v)

    ways = (torch.Tensor.contiguous, wider, lambda v: v.t().contiguous().t())
    calls = ((lambda a: ta.fused_linear(*a, None, "silu", checkpoint), [d[k] for k in ("x", "weight", "bias")], dy),
             (lambda a: ta.swiglu_mlp(*a, None, checkpoint), [m[k] for k in ("x", "w_gate", "w_up", "w_down")], mdy))
    for call, args, g in calls:
        want = torch.autograd.grad(call(args), args, g)
        for way in ways:
            for part in range(2):
                count = [0]

                def unpack(v):
                    count[0] += 1
                    return way(v.clone()) if count[0] % 2 == part else v

                with torch.autograd.graph.saved_tensors_hooks(lambda v: v, unpack):
                    y = call(args)
                for a, b in zip(torch.autograd.grad(y, args, g), want):
                    same(a, b)
                assert count[0] > 1


def test_large_matrices_that_a_product_reads_next():
    """On either side of the size from which bf16 matrices may go past the caches: the same bits."""
    from torchure_amd import _native

    g = torch.Generator(device=DEV).manual_seed(36)
    for rows in (10_000, 10_300):
        x, w = torch.randn(rows, 8192, generator=g, device=DEV).to(BF16), torch.randn(40, 8192, generator=g, device=DEV).to(BF16)
        dy = torch.randn(rows, 40, generator=g, device=DEV).to(BF16)
        w.requires_grad_()
        q = ta.quantize_activation(x)
        y = ta.fused_linear(x, w, checkpoint="e4m3")
        same(y, ta.fused_linear(x, w))
        held = ta.dequantize_activation(q)
        same(torch.autograd.grad(y, w, dy)[0], torch.autograd.grad(ta.fused_linear(held, w), w, dy)[0])
        lib, stream = _native.lib(), _native.stream_handle(torch.device(DEV, 0))
        values, exps, back = torch.empty_like(q.values), torch.empty_like(q.exponents), torch.empty_like(x)
        _native.check(lib.tm_quantize_e4m3(values.data_ptr(), exps.data_ptr(), 8192, x.data_ptr(), _native.TM_READ_NEXT, 8192, rows,
                                           8192, None, 0, stream), "tm_quantize_e4m3")
        _native.check(lib.tm_dequantize_e4m3(back.data_ptr(), _native.TM_READ_NEXT, 8192, values.data_ptr(), exps.data_ptr(), 8192,
                                             rows, 8192, stream), "tm_dequantize_e4m3")
        assert torch.equal(values, q.values) and torch.equal(exps, q.exponents)
        same(back, held)
