"""The embedding's gradient by sums that are exact, so that every token counts once, and on the stream that it is called on."""

from __future__ import annotations

import pytest
import torch

import torchure_amd as ta

pytestmark = pytest.mark.gpu

DEV, BF16, F32 = "cuda", torch.bfloat16, torch.float32


def ids_of(kind, n, vocab, g):
    if kind == "same":
        return torch.full((n,), vocab // 2, device=DEV)
    if kind == "text":
        return (torch.rand(n, generator=g, device=DEV).pow(4) * vocab).long().clamp_(max=vocab - 1)
    return torch.randint(0, vocab, (n,), generator=g, device=DEV)


def check(kind, n, vocab, cols, w, out, scale=0.5, padding=None, id_type=torch.int64):
    """Whole numbers from 1 to 7: their sums are below 2^24, and a token that is lost, doubled or in another's row shows."""
    g = torch.Generator(device=DEV).manual_seed(n + cols)
    ids = ids_of(kind, n, vocab, g)
    if padding is not None:
        ids[n - n // 3:] = padding
    dy = torch.randint(1, 8, (n, cols), generator=g, device=DEV).to(out)
    takes_part = ids != (-1 if padding is None else padding)
    sums = torch.zeros(vocab, cols, dtype=torch.float64, device=DEV).index_add_(0, ids[takes_part], dy[takes_part].double())
    weight = torch.zeros(vocab, cols, device=DEV, dtype=w, requires_grad=True)
    y = ta.embedding(ids.to(id_type), weight, scale, padding, out)
    dw, = torch.autograd.grad(y, weight, dy)
    assert torch.equal(dw, (sums * scale).float().to(w))
    table = torch.randint(0, 9, (vocab, cols), generator=g, device=DEV).to(w)
    want = (table.double() + sums * scale).float().to(w)
    assert torch.equal(ta.embedding_grad_(table, ids.to(id_type), dy, scale, padding), want)


@pytest.mark.parametrize("w,out", [(F32, F32), (BF16, BF16), (F32, BF16)])
@pytest.mark.parametrize("n", [1, 33, 2049, 8193, 20_000, 50_001, 150_001])
@pytest.mark.parametrize("kind,vocab", [("same", 4096), ("text", 4096), ("text", 1), ("any", 2), ("any", 300)])
def test_every_token_counts_once(kind, vocab, n, w, out):
    check(kind, n, vocab, 64, w, out)


@pytest.mark.parametrize("w,out", [(BF16, BF16), (F32, BF16), (F32, F32)])
@pytest.mark.parametrize("cols", [777, 520, 1237])
@pytest.mark.parametrize("n,vocab", [(8192, 151_936), (50_001, 4096), (50_001, 300)])
def test_padded_batches_of_odd_widths(n, vocab, cols, w, out):
    check("text", n, vocab, cols, w, out, padding=3, id_type=torch.int32 if cols == 520 else torch.int64)


def beside():
    """A stream whose work runs beside the current one's (streams share the few hardware queues)."""
    for _ in range(8):
        s, done = torch.cuda.Stream(), torch.cuda.Event()
        torch.cuda._sleep(20_000_000)  # a bounded spin
        done.record()
        with torch.cuda.stream(s):
            torch.ones(1, device=DEV)
        s.synchronize()
        free = not done.query()
        torch.cuda.synchronize()
        if free:
            return s
    pytest.skip("no stream runs beside the current one")


def test_node_called_on_another_stream():
    """A node that is called directly runs where it is called, not where its forward pass ran."""
    g = torch.Generator(device=DEV).manual_seed(2)
    ids = ids_of("text", 3000, 500, g)
    weight = torch.randn(500, 256, generator=g, device=DEV).requires_grad_()
    dy = torch.randn(3000, 256, generator=g, device=DEV)
    want, = torch.autograd.grad(ta.embedding(ids, weight), weight, dy)
    y = ta.embedding(ids, weight)
    torch.cuda.synchronize()
    s = beside()
    with torch.cuda.stream(s):
        spoilt = torch.full_like(want, float("nan"))
    s.synchronize()
    del spoilt  # (its block is the result's)
    torch.cuda._sleep(100_000_000)  # the forward pass's stream is busy
    with torch.no_grad(), torch.cuda.stream(s):
        got = next(v for v in y.grad_fn(dy) if v is not None).clone()
    s.synchronize()
    assert torch.equal(got, want)
    torch.cuda.synchronize()
