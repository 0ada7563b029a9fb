"""What the linear layers, the gated feed-forward and the 8-bit activations refuse, without a GPU: the
Python checks (the one of the device left out to reach the others) and the C ABI's, which all come
before any HIP call."""

from __future__ import annotations

import ctypes
import re

import pytest
import torch

import torchure_amd as ta
from torchure_amd import _native, linear

BF16, F32, F16 = torch.bfloat16, torch.float32, torch.float16


def ones(*shape, dtype=BF16):
    return torch.ones(shape, dtype=dtype)


def test_cpu_tensors():
    x, w = ones(3, 4), ones(5, 4)
    q = ta.QuantizedActivation(torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8), x.shape, BF16)
    for call in (lambda: ta.fused_linear(x, w), lambda: ta.swiglu_mlp(x, w, w, ones(4, 5)),
                 lambda: ta.quantize_activation(x), lambda: ta.dequantize_activation(q)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            call()


@pytest.fixture
def no_device(monkeypatch):
    monkeypatch.setattr(linear, "_on_gpu", lambda t, who, what: None)


@pytest.mark.parametrize("args,error,match", [
    (dict(activation="tanh"), ValueError, "activation"),
    (dict(activation=""), ValueError, "activation"),
    (dict(checkpoint="int8"), ValueError, "checkpoint"),
    (dict(weight=ones(5, 3)), RuntimeError, "do not match"),
    (dict(weight=ones(4)), RuntimeError, "do not match"),
    (dict(weight=ones(1, 5, 4)), RuntimeError, "do not match"),
    (dict(x=ones()), RuntimeError, "do not match"),
    (dict(weight=ones(0, 4)), RuntimeError, "no elements"),
    (dict(x=ones(3, 0), weight=ones(5, 0)), RuntimeError, "no elements"),
    (dict(x=ones(3, 4, dtype=F32)), NotImplementedError, "autocast off"),
    (dict(x=ones(3, 4, dtype=F16)), NotImplementedError, "x must be bfloat16"),
    (dict(weight=ones(5, 4, dtype=F16)), NotImplementedError, "weight"),
    (dict(bias=ones(5, dtype=F16)), NotImplementedError, "bias"),
    (dict(residual=ones(3, 5, dtype=torch.float64)), NotImplementedError, "residual"),
    (dict(bias=ones(4)), RuntimeError, "bias"),
    (dict(bias=ones(1, 5)), RuntimeError, "bias"),
    (dict(residual=ones(5)), RuntimeError, "residual"),
    (dict(residual=ones(3, 4)), RuntimeError, "residual"),
    (dict(residual=ones(1, 3, 5)), RuntimeError, "residual"),
])
def test_fused_linear(no_device, args, error, match):
    with pytest.raises(error, match=match):
        ta.fused_linear(**{"x": ones(3, 4), "weight": ones(5, 4), **args})


@pytest.mark.parametrize("args,error,match", [
    (dict(checkpoint="bf16"), ValueError, "checkpoint"),
    (dict(w_up=ones(6, 4)), RuntimeError, "do not match"),
    (dict(w_down=ones(4, 6)), RuntimeError, "do not match"),
    (dict(w_gate=ones(5, 3), w_up=ones(5, 3)), RuntimeError, "do not match"),
    (dict(x=ones(3, 4, dtype=F32)), NotImplementedError, "autocast off"),
    (dict(w_down=ones(4, 5, dtype=F16)), NotImplementedError, "w_down"),
    (dict(residual=ones(3, 5)), RuntimeError, "residual"),
    (dict(w_gate=ones(0, 4), w_up=ones(0, 4), w_down=ones(4, 0)), RuntimeError, "no elements"),
])
def test_swiglu_mlp(no_device, args, error, match):
    with pytest.raises(error, match=match):
        ta.swiglu_mlp(**{"x": ones(3, 4), "w_gate": ones(5, 4), "w_up": ones(5, 4), "w_down": ones(4, 5), **args})


def test_quantize(no_device):
    with pytest.raises(NotImplementedError, match="x must be"):
        ta.quantize_activation(ones(3, dtype=F16))
    with pytest.raises(ValueError, match="dimension"):
        ta.quantize_activation(ones())
    values, exps = torch.zeros(3, 32, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8)
    shape = torch.Size((3, 4))
    with pytest.raises(NotImplementedError, match="dtype"):
        ta.dequantize_activation(ta.QuantizedActivation(values, exps, shape, BF16), F16)
    for v, e, s in ((values[:2], exps, shape), (values[:, :16], exps, shape), (values, exps[:0], shape),
                    (values.float(), exps, shape), (values, exps, torch.Size((33, 4))), (values, exps, torch.Size((3, 40))),
                    (torch.zeros(32, 3, dtype=torch.uint8).t(), exps, shape)):
        with pytest.raises(RuntimeError, match="not those"):
            ta.dequantize_activation(ta.QuantizedActivation(v, e, s, BF16))


# ---------------------------------------------------------------------------- the C ABI


def test_lin_record_layout_matches_header():
    with open(_native.HEADER_PATH) as f:
        text = f.read()
    body = re.search(r"typedef struct tm_lin \{(.*?)\} tm_lin_t;", text, re.S).group(1)
    names, size = [], 0
    for kind, star, fields in re.findall(r"(?:const )?(void|uint16_t|uint8_t|int64_t|int32_t)(\*?) ([\w, ]+);", body):
        for name in fields.split(", "):
            names.append(name)
            size += 4 if kind == "int32_t" else 8
            assert star or kind in ("int64_t", "int32_t")
    assert names == [n for n, _ in _native.TmLin._fields_] and ctypes.sizeof(_native.TmLin) == size
    for name in re.findall(r"#define (TM_(?:HELD|LIN)_\w+) ", text):
        assert getattr(_native, name) == int(re.search(rf"#define {name} (\d+)", text).group(1))
    for i, name in enumerate(_native.TM_ACTS):
        assert int(re.search(rf"#define TM_ACT_{name.upper()} +(\d+)", text).group(1)) == i


FAKE = 0x1000
FORWARD, GATE, GRAD_X, GATE_GRAD, GRAD_W = range(5)


def lin(ws=1 << 40, d_ws=FAKE, **fields):
    """tm_lin's answer to 64 rows of 40 features into 48, but for ``fields``."""
    d = _native.TmLin(rows=640, inp=40, out=48, a=FAKE, b0=FAKE, o0=FAKE, lda=64, ldb=64, ldo=128, op=FORWARD)
    for k, v in fields.items():
        setattr(d, k, v)
    rc = _native.lib().tm_lin(ctypes.byref(d), d_ws, ws, None)
    return rc, _native.lib().tm_last_error()


@pytest.mark.parametrize("fields,match", [
    (dict(op=5), b"op"), (dict(op=-1), b"op"), (dict(rows=0), b"rows"), (dict(inp=0), b"rows"), (dict(out=-1), b"rows"),
    (dict(rows=(1 << 30) + 1), b"rows"), (dict(out=(1 << 22) + 1), b"rows"),
    (dict(rows=1 << 30, out=1 << 22, ldo=1 << 23), b"too large"),
    (dict(a=None), b"null"), (dict(b0=None), b"null"), (dict(o0=None), b"null"), (dict(op=GATE, z0=FAKE, z1=FAKE), b"null"),
    (dict(a=0x1008), b"aligned"), (dict(b0=0x1002), b"aligned"), (dict(lda=44), b"multiple of 8"),
    (dict(ldb=52), b"multiple of 8"), (dict(lda=32), b"elements apart"), (dict(ldb=32), b"elements apart"),
    (dict(lda=1 << 23), b"2\\^23"), (dict(op=GRAD_X, lda=40), b"elements apart"),
    (dict(op=GRAD_X, b1=FAKE, lda=64), b"elements apart"), (dict(op=GRAD_W, o1=FAKE, lda=64), b"elements apart"),
    (dict(ldo=47), b"output rows"), (dict(ldo=1 << 24), b"2\\^24"), (dict(res=FAKE, ldr=47), b"2\\^24"),
    (dict(res=FAKE, ldr=1 << 24), b"2\\^24"), (dict(o0=0x1001), b"aligned"), (dict(out_f32=1, o0=0x1002), b"aligned"),
    (dict(res=0x1001, ldr=48), b"aligned"), (dict(res=0x1002, ldr=48, res_f32=1), b"aligned"), (dict(bias=0x1001), b"aligned"),
    (dict(bias=0x1002, bias_f32=1), b"aligned"), (dict(act=5), b"act"), (dict(act=-1), b"act"), (dict(held=3), b"held"),
    (dict(held=1, z0=None, ldz=48), b"null"), (dict(held=1, z0=FAKE, ldz=40), b"held"),
    (dict(held=1, z0=0x1008, ldz=48), b"aligned"), (dict(held=2, z0=FAKE, s0=FAKE, ldz=48), b"held"),
    (dict(held=2, z0=FAKE, s0=None, ldz=64), b"exponents"),
    (dict(op=GATE, b1=FAKE, ldo=40, held=1, z0=FAKE, z1=FAKE, ldz=48), b"gate"),
    (dict(op=GATE_GRAD, lda=48, ldo=64, held=1, z0=FAKE, z1=FAKE, ldz=40), b"gate"),
    (dict(op=GATE_GRAD, lda=48, ldo=128, held=0, z0=FAKE, z1=FAKE, ldz=40), b"held"),
])
def test_lin_argument_checks_without_gpu(fields, match):
    rc, text = lin(**fields)
    assert rc < 0 and re.search(match, text), text


def test_lin_workspace_checks_without_gpu():
    need = _native.lib().tm_lin_workspace_bytes(GRAD_W, 8192, 1024, 256, 0)
    assert need > 0
    case = dict(op=GRAD_W, rows=8192, inp=1024, out=256, lda=256, ldb=1024, ldo=1024)
    for ws, at in ((need - 1, FAKE), (need, None), (need, 0x1008)):
        rc, text = lin(ws, at, **case)
        assert rc < 0 and b"workspace" in text
    assert _native.lib().tm_lin_workspace_bytes(GRAD_W, 0, 1024, 256, 0) == 0
    assert _native.lib().tm_lin_workspace_bytes(7, 64, 64, 64, 0) == 0
    assert _native.lib().tm_lin(None, None, 0, None) < 0


def test_activation_checks_without_gpu():
    lib = _native.lib()
    good = [FAKE, FAKE, 64, FAKE, 0, 40, 33, 40, None, 0, None]
    for at, bad in ((0, None), (0, 0x1008), (1, None), (2, 40), (3, None), (3, 0x1001), (5, 39), (6, -1), (7, -1)):
        args = list(good)
        args[at] = bad
        assert lib.tm_quantize_e4m3(*args) < 0, at
    assert lib.tm_quantize_e4m3(FAKE, FAKE, 64, FAKE, 0, 40, 33, 40, FAKE, 48, None) < 0  # copy rows: 40
    assert lib.tm_quantize_e4m3(FAKE, FAKE, 64, FAKE, 1, 40, 33, 40, 0x1002, 40, None) < 0
    assert lib.tm_quantize_e4m3(None, None, 0, None, 0, 0, 0, 40, None, 0, None) == 0  # nothing to do
    good = [FAKE, 0, 40, FAKE, FAKE, 64, 33, 40, None]
    for at, bad in ((0, None), (0, 0x1001), (2, 39), (3, None), (3, 0x1004), (4, None), (5, 48), (6, -1)):
        args = list(good)
        args[at] = bad
        assert lib.tm_dequantize_e4m3(*args) < 0, at
    need = lib.tm_act_grad_workspace_bytes(70, 40)
    assert need == 2 * 40 * 4 and lib.tm_act_grad_workspace_bytes(0, 40) == 0
    good = [FAKE, 40, FAKE, 0, FAKE, 0, 40, FAKE, FAKE, 64, 2, 2, 70, 40, FAKE, need, None]
    for at, bad in ((0, 0x1008), (1, 44), (1, 32), (4, None), (4, 0x1001), (6, 39), (7, None), (7, 0x1004), (8, None), (9, 40),
                    (10, 0), (10, 3), (11, 5), (11, -1), (12, 0), (12, -1), (13, 0), (14, None), (15, need - 1)):
        args = list(good)
        args[at] = bad
        assert lib.tm_act_grad(*args) < 0, at


@pytest.mark.parametrize("fields", [
    dict(op=GRAD_W, o1=FAKE, lda=128, ldo=40, ldo1=48),  # two outputs, one distance
    dict(op=GRAD_W, o1=FAKE, lda=128, ldo=40),
    dict(op=GATE_GRAD, lda=48, ldo=128, held=1, z0=FAKE, z1=FAKE, ldz=40, o1=FAKE, ldo1=1 << 24),
])
def test_second_output_rows_without_gpu(fields):
    rc, text = lin(**fields)
    assert rc < 0 and b"2^24" in text, text


def test_launches_of_2_to_the_32_work_items_without_gpu():
    lib = _native.lib()
    rows = 1 << 30  # of one column: 2^25 bands of 32 rows
    assert lib.tm_quantize_e4m3(FAKE, FAKE, 32, FAKE, 0, 1, rows, 1, None, 0, None) < 0
    assert b"too large" in lib.tm_last_error()
    assert lib.tm_dequantize_e4m3(FAKE, 0, 1, FAKE, FAKE, 32, rows, 1, None) < 0
    need = lib.tm_act_grad_workspace_bytes(1, 1 << 30)
    assert lib.tm_act_grad(None, 0, FAKE, 0, FAKE, 0, 1 << 30, None, None, 0, 0, 0, 1, 1 << 30, FAKE, need, None) < 0
    assert lib.tm_act_grad(FAKE, 8, None, 0, FAKE, 0, 1, None, None, 0, 0, 0, rows, 1, None, 0, None) < 0


def test_a_quantized_activation_without_dimensions(no_device):
    one = torch.zeros(1, 32, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="not those"):
        ta.dequantize_activation(ta.QuantizedActivation(one, one[:, :1], torch.Size(()), BF16))


@pytest.mark.parametrize("wide", [64, 128, 136])
def test_act_grad_launches_of_2_to_the_31_workgroups_without_gpu(wide):
    """2^25 bands of 32 rows by ``wide`` groups of 256 columns: 2^31 workgroups, 2^32, and more than that."""
    lib = _native.lib()
    rows, cols = 1 << 30, 256 * wide
    assert lib.tm_act_grad(FAKE, cols, None, 0, FAKE, 0, cols, None, None, 0, 0, 0, rows, cols, None, 0, None) < 0
    assert b"too large" in lib.tm_last_error()


def test_held_gate_checks_without_gpu():
    lib = _native.lib()
    good = [FAKE, 40, FAKE, FAKE, FAKE, FAKE, 64, _native.TM_HELD_E4M3, 33, 40, None]
    for at, bad in ((0, None), (0, 0x1008), (1, 44), (1, 32), (2, None), (2, 0x1004), (3, None), (3, 0x1008), (4, None), (5, None),
                    (6, 40), (6, 96), (7, 0), (7, 1), (7, 3), (8, -1), (9, -1), (8, (1 << 30) + 1)):
        args = list(good)
        args[at] = bad
        if (at, bad) == (7, 1):
            args[6] = 36  # bf16 rows: whole groups of 8
        assert lib.tm_held_gate(*args) < 0 and b"tm_held_gate" in lib.tm_last_error(), (at, bad)
        assert b"launch" not in lib.tm_last_error(), (at, bad)
    assert lib.tm_held_gate(None, 0, None, None, None, None, 0, 0, 0, 40, None) == 0  # nothing to do
    assert lib.tm_held_gate(FAKE, 8, FAKE, FAKE, None, None, 8, _native.TM_HELD_BF16, 1 << 30, 1, None) < 0  # 2^25 bands
    assert b"too large" in lib.tm_last_error()


def test_unknown_flags_without_gpu():
    lib = _native.lib()
    for flags in (4, 5, -1, 1 << 30):
        assert lib.tm_quantize_e4m3(FAKE, FAKE, 64, FAKE, flags, 40, 33, 40, None, 0, None) < 0
        assert b"flags" in lib.tm_last_error()
        assert lib.tm_dequantize_e4m3(FAKE, flags, 40, FAKE, FAKE, 64, 33, 40, None) < 0
        assert b"flags" in lib.tm_last_error()
