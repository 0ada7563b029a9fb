"""What the norms and the embedding refuse, without a GPU: the Python checks (the one of the device left out to reach the
others) and the C ABI's, which all come before any HIP call."""

from __future__ import annotations

import pytest
import torch

import torchure_amd as ta
from torchure_amd import _native, embed, norm

BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16
FAKE = 0x1000


def ones(*shape, dtype=BF16):
    return torch.ones(shape, dtype=dtype)


@pytest.fixture
def no_device(monkeypatch):
    monkeypatch.setattr(norm, "_on_gpu", lambda t, who, what: None)
    monkeypatch.setattr(embed, "_on_gpu", lambda t, who, what: None)


def test_cpu_tensors():
    for call in (lambda: ta.rms_norm(ones(3, 4)), lambda: ta.layer_norm(ones(3, 4), ones(4), ones(4)),
                 lambda: ta.embedding(torch.arange(3), ones(4, 5)),
                 lambda: ta.embedding_grad_(ones(4, 5), torch.arange(3), ones(3, 5))):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


@pytest.mark.parametrize("args,error,match", [
    (dict(x=ones(3, 4, dtype=F16)), NotImplementedError, "x must be"),
    (dict(x=ones()), ValueError, "dimension"),
    (dict(x=ones(3, 0), weight=None, bias=None), RuntimeError, "0 features"),
    (dict(x=ones(2, 16385), weight=None, bias=None), RuntimeError, "16385 features"),
    (dict(weight=ones(4, dtype=F16)), NotImplementedError, "weight must be"),
    (dict(bias=ones(4, dtype=torch.float64)), NotImplementedError, "bias must be"),
    (dict(weight=ones(3)), RuntimeError, "weight of shape"),
    (dict(weight=ones(1, 4)), RuntimeError, "weight of shape"),
    (dict(bias=ones(5)), RuntimeError, "bias of shape"),
    (dict(dtype=F16), NotImplementedError, "dtype"),
    (dict(dtype=torch.int32), NotImplementedError, "dtype"),
    (dict(eps=-1e-6), ValueError, "eps"),
    (dict(eps=float("nan")), ValueError, "eps"),
    (dict(x=torch.eye(4).to_sparse()), NotImplementedError, "dense"),
])
def test_layer_norm(no_device, args, error, match):
    with pytest.raises(error, match=match):
        ta.layer_norm(**{"x": ones(3, 4), "weight": ones(4), "bias": ones(4), **args})


def test_rms_norm(no_device):
    with pytest.raises(RuntimeError, match="weight of shape"):
        ta.rms_norm(ones(3, 4), ones(5))
    with pytest.raises(TypeError):
        ta.rms_norm(ones(3, 4), ones(4), bias=ones(4))


def test_no_rows(no_device):
    y = ta.layer_norm(ones(0, 4).requires_grad_(), ones(4), dtype=F32)
    assert y.shape == (0, 4) and y.dtype == F32 and y.grad_fn is not None


def test_norm_checks_without_gpu():
    lib = _native.lib()
    #       y     f  rstd  mean  x     f  ldx w     f  b     f  layer eps   rows cols
    good = [FAKE, 0, FAKE, FAKE, FAKE, 0, 40, FAKE, 0, FAKE, 0, 1, 1e-5, 33, 40, None]
    for at, bad in ((0, None), (0, 0x1001), (2, 0x1002), (3, None), (3, 0x1002), (4, None), (4, 0x1001), (6, 39), (7, 0x1001),
                    (9, 0x1001), (13, -1), (13, (1 << 40) + 1), (14, 0), (14, -1), (14, 16385)):
        args = list(good)
        args[at] = bad
        assert lib.tm_norm_forward(*args) < 0 and b"tm_norm_forward" in lib.tm_last_error(), (at, bad)
        assert b"launch" not in lib.tm_last_error(), (at, bad)
    assert lib.tm_norm_forward(*good[:13], 0, 40, None) == 0  # nothing to do
    args = list(good)
    args[1], args[0] = 1, 0x1002
    assert lib.tm_norm_forward(*args) < 0
    need = lib.tm_norm_workspace_bytes(33, 40, 0, 0, 1)
    assert need > 0 and need % 320 == 0 and lib.tm_norm_workspace_bytes(33, 40, 0, 0, 0) == need // 2
    assert lib.tm_norm_workspace_bytes(0, 40, 0, 0, 1) == 0 and lib.tm_norm_workspace_bytes(1, 16385, 0, 0, 1) == 0
    #       dx    dw    db    bf dy    yf lddy x    xf ldx rstd  mean  w     wf dwf layer rows cols ws
    good = [FAKE, FAKE, FAKE, 0, FAKE, 0, 40, FAKE, 0, 40, FAKE, FAKE, FAKE, 0, 0, 1, 33, 40, FAKE, need, None]
    for at, bad in ((0, 0x1001), (1, 0x1001), (2, 0x1001), (4, None), (4, 0x1001), (6, 39), (7, None), (7, 0x1001), (9, 39), (10, None),
                    (11, None), (12, 0x1001), (15, 0), (16, 0), (16, -1), (17, 0), (17, 16385), (18, None), (18, 0x1002),
                    (19, need - 1)):
        args = list(good)
        args[at] = bad
        assert lib.tm_norm_backward(*args) < 0 and b"tm_norm_backward" in lib.tm_last_error(), (at, bad)
        assert b"launch" not in lib.tm_last_error(), (at, bad)
    assert lib.tm_norm_backward(None, None, None, *good[3:18], None, 0, None) == 0  # nothing wanted


IDS = torch.arange(3)


@pytest.mark.parametrize("args,error,match", [
    (dict(ids=IDS.float()), NotImplementedError, "ids must be"),
    (dict(ids=IDS.to(torch.int16)), NotImplementedError, "ids must be"),
    (dict(weight=ones(4, 5, dtype=F16)), NotImplementedError, "weight must be"),
    (dict(weight=ones(4)), RuntimeError, "weight of shape"),
    (dict(weight=ones(2, 4, 5)), RuntimeError, "weight of shape"),
    (dict(weight=ones(0, 5)), RuntimeError, "weight of shape"),
    (dict(weight=ones(4, 0)), RuntimeError, "weight of shape"),
    (dict(weight=torch.eye(4).to_sparse()), NotImplementedError, "dense"),
    (dict(padding_idx=4), ValueError, "padding_idx"),
    (dict(padding_idx=-5), ValueError, "padding_idx"),
    (dict(dtype=F16), NotImplementedError, "dtype"),
])
def test_embedding(no_device, args, error, match):
    with pytest.raises(error, match=match):
        ta.embedding(**{"ids": IDS, "weight": ones(4, 5), **args})


@pytest.mark.parametrize("args,error,match", [
    (dict(grad=ones(4, 5, dtype=F16)), NotImplementedError, "grad must be"),
    (dict(dy=ones(3, 5, dtype=F16)), NotImplementedError, "dy must be"),
    (dict(dy=ones(3, 4)), RuntimeError, "dy of shape"),
    (dict(dy=ones(5)), RuntimeError, "dy of shape"),
    (dict(dy=ones(1, 3, 5)), RuntimeError, "dy of shape"),
    (dict(grad=ones(5, 4).t()), RuntimeError, "strides"),
    (dict(grad=ones(1, 5).expand(4, 5)), RuntimeError, "strides"),
    (dict(grad=ones(4, 10)[:, ::2]), RuntimeError, "strides"),
    (dict(grad=ones(4, 5).requires_grad_()), RuntimeError, "requires a gradient"),
    (dict(padding_idx=7), ValueError, "padding_idx"),
])
def test_embedding_grad(no_device, args, error, match):
    with pytest.raises(error, match=match):
        ta.embedding_grad_(**{"grad": ones(4, 5), "ids": IDS, "dy": ones(3, 5), **args})


def test_embedding_grad_into_its_own_input(no_device):
    table = ones(8, 5)
    with pytest.raises(RuntimeError, match="share memory"):
        ta.embedding_grad_(table, IDS, table[5:])
    with pytest.raises(RuntimeError, match="share memory"):
        ta.embedding_grad_(table[:6], IDS, table[5:])


def test_no_tokens(no_device):
    y = ta.embedding(IDS[:0].view(0, 1), ones(4, 5).requires_grad_(), dtype=F32)
    assert y.shape == (0, 1, 5) and y.dtype == F32 and y.grad_fn is not None
    table = ones(4, 5)
    assert ta.embedding_grad_(table, IDS[:0], ones(0, 5)) is table


def test_embedding_checks_without_gpu():
    lib = _native.lib()
    #       y     f  w     f  ldw ids   64 tokens vocab cols scale
    good = [FAKE, 0, FAKE, 0, 40, FAKE, 1, 33, 100, 40, 1.0, None]
    for at, bad in ((0, None), (0, 0x1001), (2, None), (2, 0x1001), (4, 39), (5, None), (5, 0x1004), (7, -1), (7, (1 << 30) + 1), (8, 0),
                    (8, (1 << 30) + 1), (9, 0), (9, (1 << 20) + 1)):
        args = list(good)
        args[at] = bad
        assert lib.tm_embed_lookup(*args) < 0 and b"tm_embed_lookup" in lib.tm_last_error(), (at, bad)
        assert b"launch" not in lib.tm_last_error(), (at, bad)
    assert lib.tm_embed_lookup(*good[:7], 0, 100, 40, 1.0, None) == 0  # nothing to do
    need = lib.tm_embed_grad_workspace_bytes(33, 100, 40)
    assert need == 16 + 2 * 144 + 8 * 256 + 8 * 2 * 40
    for bad in ((0, 100, 40), (33, 0, 40), (33, 100, 0), ((1 << 30) + 1, 100, 40)):
        assert lib.tm_embed_grad_workspace_bytes(*bad) == 0
    #       dw    f  ldw dy    f  lddy ids  64 tokens vocab cols scale pad add ws
    good = [FAKE, 0, 40, FAKE, 0, 40, FAKE, 1, 33, 100, 40, 1.0, -1, 0, FAKE, need, None]
    for at, bad in ((0, None), (0, 0x1001), (2, 39), (3, None), (3, 0x1001), (5, 39), (6, None), (6, 0x1004), (8, 0), (8, -1), (9, 0), (10, 0),
                    (14, None), (14, 0x1008), (15, need - 1)):
        args = list(good)
        args[at] = bad
        assert lib.tm_embed_grad(*args) < 0 and b"tm_embed_grad" in lib.tm_last_error(), (at, bad)
        assert b"launch" not in lib.tm_last_error(), (at, bad)
    big = (1 << 30, 100, 1 << 12)
    args = [FAKE, 0, 1 << 12, FAKE, 0, 1 << 12, FAKE, 1, *big, 1.0, -1, 0, FAKE, lib.tm_embed_grad_workspace_bytes(*big), None]
    assert lib.tm_embed_grad(*args) < 0 and b"too large" in lib.tm_last_error()


def test_adamw_state_bits():
    p = torch.nn.Parameter(torch.zeros(4))
    for bits in (16, 4, 0, "8", None, 8.5):
        with pytest.raises(ValueError, match="state_bits"):
            ta.AdamW([p], state_bits=bits)
    for seed in (-1, 1 << 64):
        with pytest.raises(ValueError, match="seed"):
            ta.AdamW([p], state_bits=8, seed=seed)
    for seed in (1.5, "1", None):
        with pytest.raises(TypeError):
            ta.AdamW([p], state_bits=8, seed=seed)
    opt = ta.AdamW([p], state_bits=8, seed=(1 << 64) - 1)
    with pytest.raises(RuntimeError, match="no param has state"):
        opt.flat_moments()
    with pytest.raises(RuntimeError, match="state_bits=32"):
        ta.AdamW([p]).flat_moments()


def test_8_bit_moments_checks_without_gpu():
    lib = _native.lib()
    for n, size in ((-1, 0), (0, 0), (1, 260), (256, 260), (257, 520), (1 << 33, (1 << 33) * 65 // 64)):
        assert lib.tm_moments8_bytes(n) == size
    groups = (_native.TmHyper * 2)()
    #       tensors n  chunks n  elems
    table = [FAKE, 3, FAKE, 5, 65536]
    wrong = ((0, None), (1, -1), (1, 1 << 32), (2, None), (3, -1), (3, 1 << 32), (4, 0), (4, -256), (4, 65537), (4, 1 << 31))
    for name, rest in (("tm_adamw8_step", [groups, 2, None, 7, FAKE, None]), ("tm_moments8_read", [None]), ("tm_moments8_write", [None])):
        for at, bad in wrong:
            args = table + rest
            args[at] = bad
            assert getattr(lib, name)(*args) < 0 and name.encode() in lib.tm_last_error(), (name, at, bad)
            assert b"launch" not in lib.tm_last_error(), (name, at, bad)
    for at, bad in ((5, None), (6, 0), (6, -1), (6, _native.TM_MAX_GROUPS + 1), (9, None)):
        args = table + [groups, 2, None, 7, FAKE, None]
        args[at] = bad
        assert lib.tm_adamw8_step(*args) < 0 and b"tm_adamw8_step" in lib.tm_last_error(), (at, bad)
