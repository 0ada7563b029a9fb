"""The token embedding and its gradient against the same sums in 64 bits, and as programs call them.

A gradient's row is a sum of c rows in fp32, times the scale: at most c + 1 roundings of 2^-24 of the sum of magnitudes, then
the result's own."""

from __future__ import annotations

import math

import pytest
import torch

import torchure_amd as ta

pytestmark = pytest.mark.gpu

DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}
U = 2.0 ** -24


def same(a, b, what=""):
    assert a.dtype == b.dtype and a.shape == b.shape, what
    kind = torch.int16 if a.dtype == BF16 else torch.int32
    assert torch.equal(a.detach().contiguous().view(kind), b.detach().contiguous().view(kind)), what


def close(got, value, bound, what):
    got = got.detach().double()
    assert got.shape == value.shape, what
    bad = ~((got - value).abs() <= bound)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((got - value).abs().max()):.3g}"


def ids_of(kind, n, vocab, g):
    if kind == "same":
        return torch.full((n,), vocab // 2, device=DEV)
    if kind == "text":
        return (torch.rand(n, generator=g, device=DEV).pow(4) * vocab).long().clamp_(max=vocab - 1)
    if kind == "runs":
        return (torch.arange(n, device=DEV) // 45) % vocab
    if kind == "apart":
        return torch.arange(n, device=DEV) % vocab
    return torch.randint(0, vocab, (n,), generator=g, device=DEV)


def grads64(ids, dy, vocab, scale, padding=None):
    """(sums, bound without the result's rounding) of valid ids."""
    ids, dy = ids.reshape(-1), dy.reshape(-1, dy.shape[-1]).double()
    ok = (ids >= 0) & (ids < vocab)
    if padding is not None:
        ok &= ids != padding
    where = ids[ok].long()
    s = torch.zeros(vocab, dy.shape[1], dtype=torch.float64, device=DEV).index_add_(0, where, dy[ok]) * scale
    size = torch.zeros_like(s).index_add_(0, where, dy[ok].abs()) * abs(scale)
    count = torch.zeros(vocab, device=DEV, dtype=torch.float64).index_add_(0, where, torch.ones(len(where), device=DEV, dtype=torch.float64))
    return s, (count[:, None] + 2) * U * size


def check(ids, vocab, dim, w=F32, out=None, scale=1.0, padding=None, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    weight = torch.randn(vocab, dim, generator=g, device=DEV).to(w).requires_grad_()
    y = ta.embedding(ids, weight, scale, padding, out)
    out = out or w
    assert y.dtype == out and y.shape == (*ids.shape, dim)
    flat = ids.reshape(-1).long()
    ok = (flat >= 0) & (flat < vocab)
    value = weight.detach()[torch.where(ok, flat, 0)].double() * scale
    rows = y.reshape(-1, dim)
    close(rows[ok], value[ok], (HALF[out] + U) * value[ok].abs(), "y")
    assert torch.isnan(rows[~ok]).all()
    with torch.no_grad():
        same(ta.embedding(ids, weight, scale, padding, out), y)
    dy = torch.randn(y.shape, generator=g, device=DEV).to(out)
    dw, = torch.autograd.grad(y, weight, dy)
    assert dw.dtype == w and dw.is_contiguous()
    s, e = grads64(ids, dy, vocab, scale, padding)
    close(dw, s, e + HALF[w] * (s.abs() + e), "gradient")
    # the same sums, added to a table that is there
    there = torch.randn(vocab, dim, generator=g, device=DEV).to(w)
    table, version = there.clone(), 0
    version = table._version
    assert ta.embedding_grad_(table, ids, dy, scale, padding) is table and table._version > version
    total = there.double() + s
    close(table, total, e + U * s.abs() + HALF[w] * (total.abs() + e), "added gradient")
    rest = ~torch.isin(torch.arange(vocab, device=DEV), flat if padding is None else flat[flat != padding])
    same(table[rest], there[rest], "rows without tokens")
    assert not dw[rest].any()
    again, = torch.autograd.grad(ta.embedding(ids, weight, scale, padding, out), weight, dy)
    same(again, dw, "two runs")
    return weight, dy, y, dw


@pytest.mark.parametrize("n", [1, 2, 31, 32, 33, 63, 64, 65, 200, 1023, 1024, 1025, 2500, 9001])
@pytest.mark.parametrize("kind", ["text", "same", "runs", "apart", "any"])
def test_tokens(kind, n):
    g = torch.Generator(device=DEV).manual_seed(n)
    check(ids_of(kind, n, 1000, g), 1000, 72, seed=n)


@pytest.mark.parametrize("dim", [1, 3, 4, 7, 8, 9, 31, 64, 100, 255, 256, 257, 512, 777, 1000, 1024, 1237, 2560, 5000])
@pytest.mark.parametrize("w,out", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
def test_widths_and_types(dim, w, out):
    g = torch.Generator(device=DEV).manual_seed(dim)
    check(ids_of("text", 500, 300, g), 300, dim, w, out, scale=27.875, padding=3, seed=dim)


@pytest.mark.parametrize("vocab", [1, 2, 5, 255, 256, 257, 511, 513, 8192, 50257, 151936, (1 << 21) + 5, (1 << 22) + 77])
@pytest.mark.parametrize("kind", ["text", "any", "same"])
def test_vocabularies(kind, vocab):
    g = torch.Generator(device=DEV).manual_seed(vocab)
    check(ids_of(kind, 3000, vocab, g), vocab, 16 if vocab > 1 << 20 else 40, BF16, seed=1)


@pytest.mark.parametrize("kind", ["text", "same", "any"])
def test_many_tokens(kind):
    g = torch.Generator(device=DEV).manual_seed(5)
    check(ids_of(kind, 150_001, 4096, g), 4096, 64, scale=0.5)


@pytest.mark.parametrize("n", [2047, 2049, 4097, 8191, 8193, 20000])
@pytest.mark.parametrize("vocab", [1, 2, 300])
def test_more_of_an_id_than_wait_at_once(vocab, n):
    g = torch.Generator(device=DEV).manual_seed(n)
    check(ids_of("text", n, vocab, g), vocab, 40, BF16, padding=vocab - 1 if vocab > 2 else None, seed=n)


@pytest.mark.parametrize("scale", [0.0, -1.0, 1e-3, 32.0, 27.875])
def test_scales(scale):
    g = torch.Generator(device=DEV).manual_seed(6)
    check(ids_of("text", 700, 500, g), 500, 48, BF16, scale=scale)


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_ids_of_every_shape(dtype):
    g = torch.Generator(device=DEV).manual_seed(7)
    ids = ids_of("text", 480, 200, g).to(dtype)
    weight, dy, y, dw = check(ids, 200, 40)
    for shape in ((4, 120), (2, 3, 80), (480, 1)):
        z = ta.embedding(ids.view(shape), weight)
        same(z, y.view(*shape, 40))
        got, = torch.autograd.grad(z, weight, dy.view(*shape, 40))
        same(got, dw)
    strided = torch.zeros(960, dtype=dtype, device=DEV)[::2].copy_(ids)
    same(ta.embedding(strided, weight), y)
    turned = ids.view(4, 120).t()
    same(ta.embedding(turned, weight), y.view(4, 120, 40).transpose(0, 1))
    got, = torch.autograd.grad(ta.embedding(turned, weight), weight, dy.view(4, 120, 40).transpose(0, 1))
    s, e = grads64(turned, dy.view(4, 120, 40).transpose(0, 1), 200, 1.0)
    close(got, s, e + U * s.abs(), "turned ids")
    one = ta.embedding(ids[5], weight)
    assert one.shape == (40,)
    same(one, y[5])


@pytest.mark.parametrize("padding", [0, 3, 199, -1, -200])
def test_padding(padding):
    g = torch.Generator(device=DEV).manual_seed(8)
    ids = ids_of("text", 600, 200, g)
    ids[400:] = padding % 200
    weight = torch.randn(200, 40, device=DEV).requires_grad_()
    y = ta.embedding(ids, weight, padding_idx=padding)
    same(y, ta.embedding(ids, weight))
    dy = torch.randn_like(y)
    dw, = torch.autograd.grad(y, weight, dy)
    s, e = grads64(ids, dy, 200, 1.0, padding % 200)
    close(dw, s, e + U * s.abs(), "gradient")
    assert not dw[padding].any()
    full = torch.autograd.grad(ta.embedding(ids, weight), weight, dy)[0]
    keep = torch.arange(200, device=DEV) != padding % 200
    # (fewer tokens on the list are summed in other pieces: either side is within the bound)
    close(full[keep], dw.double()[keep], 2 * (e + U * s.abs())[keep], "the other rows")
    alone = torch.full((70,), padding % 200, device=DEV)
    assert not torch.autograd.grad(ta.embedding(alone, weight, padding_idx=padding).sum(), weight)[0].any()


@pytest.mark.parametrize("dtype", [torch.int64, torch.int32])
def test_ids_outside_the_table(dtype):
    g = torch.Generator(device=DEV).manual_seed(9)
    ids = ids_of("text", 500, 300, g).to(dtype)
    for i, bad in enumerate((-1, 300, 301, -2 ** 31, 2 ** 31 - 1) + ((2 ** 32 + 5, -2 ** 63, 2 ** 63 - 1, 2 ** 40) if dtype == torch.int64 else ())):
        ids[7 * i + 3] = bad
    check(ids, 300, 33, BF16)
    check(ids[3:4], 300, 33)


# ---------------------------------------------------------------------------- layouts


def test_layouts():
    g = torch.Generator(device=DEV).manual_seed(10)
    ids = ids_of("text", 400, 100, g)
    for w in (BF16, F32):
        weight, dy, y, dw = check(ids, 100, 72, w)
        room = torch.full((104, 100), float("nan"), dtype=w, device=DEV)
        for v in (room[2:102, 3:75], torch.empty(72, 100, dtype=w, device=DEV).t(), torch.empty(200, 72, dtype=w, device=DEV)[::2],
                  torch.empty(100 * 72 + 1, dtype=w, device=DEV)[1:].view(100, 72)):
            with torch.no_grad():
                v.copy_(weight)
            u = v.detach().requires_grad_()
            z = ta.embedding(ids, u)
            same(z, y)
            back = torch.empty(72, 400, dtype=w, device=DEV).t().copy_(dy)
            same(torch.autograd.grad(z, u, back)[0], dw)
        a = torch.autograd.grad(ta.embedding(ids, weight).sum(), weight)[0]
        same(a, torch.autograd.grad(ta.embedding(ids, weight), weight, torch.ones_like(dy))[0])
        # a table within another, its rows apart: what lies between stays
        wide = torch.randn(100, 90, device=DEV).to(w)
        before = wide.clone()
        ta.embedding_grad_(wide[:, 5:77], ids, dy)
        plain = ta.embedding_grad_(before[:, 5:77].clone(), ids, dy)
        same(wide[:, 5:77], plain)
        same(wide[:, :5], before[:, :5])
        same(wide[:, 77:], before[:, 77:])


def test_special_values():
    g = torch.Generator(device=DEV).manual_seed(11)
    ids = ids_of("text", 400, 100, g)
    weight = torch.randn(100, 40, device=DEV).requires_grad_()
    y = ta.embedding(ids, weight)
    dy = torch.randn_like(y)
    dw, = torch.autograd.grad(y, weight, dy)
    bad = dy.clone()
    at = int(ids[17])
    bad[17] = math.nan
    got, = torch.autograd.grad(ta.embedding(ids, weight), weight, bad)
    keep = torch.arange(100, device=DEV) != at
    assert torch.isnan(got[at]).all()
    same(got[keep], dw[keep])
    table = torch.full((100, 40), math.nan, device=DEV)
    ta.embedding_grad_(table, ids[:0], dy[:0])
    assert torch.isnan(table).all()


def test_no_tokens():
    weight = torch.randn(100, 40, device=DEV).requires_grad_()
    y = ta.embedding(torch.empty(2, 0, dtype=torch.int64, device=DEV), weight, dtype=BF16)
    assert y.shape == (2, 0, 40) and y.dtype == BF16
    g, = torch.autograd.grad(y.sum(), weight)
    assert g.shape == weight.shape and not g.any()


# ---------------------------------------------------------------------------- as programs call it


def test_more_elements_than_32_bits():
    g = torch.Generator(device=DEV).manual_seed(12)
    table = torch.zeros(1_100_000, 2048, dtype=BF16, device=DEV)
    table[-50:] = torch.randn(50, 2048, generator=g, device=DEV).to(BF16)
    ids = torch.randint(1_099_950, 1_100_000, (300,), generator=g, device=DEV)
    small = table[-50:].clone().requires_grad_()
    y = ta.embedding(ids, table)
    same(y, ta.embedding(ids - 1_099_950, small.detach()))
    dy = torch.randn(300, 2048, generator=g, device=DEV).to(BF16)
    want, = torch.autograd.grad(ta.embedding(ids - 1_099_950, small), small, dy)
    dw, = torch.autograd.grad(ta.embedding(ids, table.requires_grad_()), table, dy)
    same(dw[-50:], want)
    assert not dw[:-50].any()
    del dw, table
    many = torch.randint(0, 50, (1_100_000,), generator=g, device=DEV)
    many[:-300] = 49
    z = ta.embedding(many, small)
    same(z[-300:], ta.embedding(many[-300:], small))
    del z
    dy = torch.zeros(1_100_000, 2048, dtype=BF16, device=DEV)
    dy[-300:] = torch.randn(300, 2048, generator=g, device=DEV).to(BF16)
    got = ta.embedding_grad_(torch.zeros(50, 2048, device=DEV), many, dy)
    s, e = grads64(many[-300:], dy[-300:], 50, 1.0)
    close(got, s, e + U * s.abs(), "long gradient")


def test_autocast_forward_mode_and_twice():
    g = torch.Generator(device=DEV).manual_seed(13)
    ids = ids_of("text", 100, 50, g)
    weight, dy, y, _ = check(ids, 50, 24)
    with torch.autocast("cuda", dtype=BF16):
        same(ta.embedding(ids, weight), y)
    d, = torch.autograd.grad(ta.embedding(ids, weight), weight, dy.clone().requires_grad_(), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiat"):
        torch.autograd.grad(d.sum(), weight)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError):
            ta.embedding(ids, torch.autograd.forward_ad.make_dual(weight.detach(), torch.ones_like(weight)))


def test_another_stream():
    g = torch.Generator(device=DEV).manual_seed(14)
    ids = ids_of("text", 3000, 5000, g)
    weight, dy, y, dw = check(ids, 5000, 256)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s):
            z = ta.embedding(ids, weight)
            got, = torch.autograd.grad(z, weight, dy)
            table = ta.embedding_grad_(torch.zeros_like(weight).detach(), ids, dy)
        s.synchronize()
        same(z, y)
        same(got, dw)
        same(table, dw)


def test_graphs():
    """Two captured passes with workspaces of their own, replayed in turn on new ids, eager calls between."""
    g = torch.Generator(device=DEV).manual_seed(15)
    cases = []
    for n, vocab, dim in ((2000, 3000, 128), (77, 500, 1000)):
        weight = torch.randn(vocab, dim, device=DEV).requires_grad_()
        cases.append((ids_of("text", n, vocab, g), weight, torch.randn(n, dim, device=DEV), torch.zeros(vocab, dim, device=DEV)))
    side, graphs, outs = torch.cuda.Stream(), [], []
    for ids, weight, dy, table in cases:
        with torch.cuda.stream(side):
            torch.autograd.grad(ta.embedding(ids, weight), weight, dy)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ta.embedding(ids, weight)
            dw, = torch.autograd.grad(y, weight, dy)
            ta.embedding_grad_(table, ids, dy)
        graphs.append(graph)
        outs.append((y.detach(), dw))
        del y
    sums = [torch.zeros_like(c[3]) for c in cases]
    for k in range(3):
        for ids, weight, _, _ in cases:
            ids.copy_(ids_of("text" if k else "runs", len(ids), len(weight), g))
        for graph in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for (ids, weight, dy, table), (y, dw), total in zip(cases, outs, sums):
            z = ta.embedding(ids, weight)
            same(z, y)
            same(torch.autograd.grad(z, weight, dy)[0], dw, f"replay {k}")
            same(ta.embedding_grad_(total, ids, dy), table, f"replay {k}")
            del z


def test_kept_ids_are_guarded():
    weight = torch.randn(50, 24, device=DEV).requires_grad_()
    ids = torch.arange(30, device=DEV)
    y = ta.embedding(ids, weight)
    ids += 1
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    y = ta.embedding(ids, weight)
    y += 1


def test_refused_on_the_device():
    weight, ids = torch.randn(50, 24, device=DEV), torch.arange(30, device=DEV)
    dy = torch.randn(30, 24, device=DEV)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ta.embedding(ids.cpu(), weight)
    with pytest.raises(RuntimeError, match="share memory"):
        ta.embedding_grad_(weight, ids, weight[:30])
    with pytest.raises(RuntimeError, match="strides"):
        ta.embedding_grad_(weight[:1].expand(50, 24), ids, dy)
    with pytest.raises(RuntimeError, match="strides"):
        ta.embedding_grad_(torch.zeros(24, 50, device=DEV).t(), ids, dy)
    with pytest.raises(RuntimeError, match="requires a gradient"):
        ta.embedding_grad_(weight.clone().requires_grad_(), ids, dy)
