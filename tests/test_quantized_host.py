"""Refusals of products with 4-bit weights (no GPU), and the sizes of packed weights."""

from __future__ import annotations

import pytest
import torch

from semblend_amd import _lib
from semblend_amd.quantized import QuantizedLinear, quantized_linear

FAKE = 4096  # an address that is never read: the checks come first
BF16 = torch.bfloat16


@pytest.fixture
def on_cpu(monkeypatch):
    """The Python checks behind the device check, with CPU tensors and the library call replaced."""
    calls = []
    cpu = torch.device("cpu")
    monkeypatch.setattr(_lib, "require_device", lambda *t: cpu)
    monkeypatch.setattr(_lib, "launch", lambda dev, name, *a: calls.append((name, a)))
    return calls


def _codes(n=32, k=128):
    return torch.full((n, k), 3, dtype=torch.uint8)


def _scales(n=32, groups=2, dtype=BF16):
    return torch.ones((n, groups), dtype=dtype)


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="device tensors"):
        QuantizedLinear(_codes(), _scales())
    with pytest.raises(RuntimeError, match="device tensors"):
        QuantizedLinear.quantize(torch.zeros((4, 64)), group=32)


def test_weight_refusals(on_cpu):
    zeros = torch.full((32, 2), 8, dtype=torch.uint8)
    bad = [(TypeError, lambda: QuantizedLinear(_codes().int(), _scales())),
           (TypeError, lambda: QuantizedLinear(_codes(), _scales().float())),
           (TypeError, lambda: QuantizedLinear(_codes(), _scales(), zeros.int())),
           (ValueError, lambda: QuantizedLinear(_codes()[0], _scales())),
           (ValueError, lambda: QuantizedLinear(_codes(), _scales()[0])),
           (ValueError, lambda: QuantizedLinear(_codes(), _scales(31))),
           (ValueError, lambda: QuantizedLinear(_codes(), _scales(groups=3))),
           (ValueError, lambda: QuantizedLinear(_codes(), _scales(groups=8))),      # groups of 16
           (ValueError, lambda: QuantizedLinear(_codes()[:0], _scales(0))),
           (ValueError, lambda: QuantizedLinear(_codes(), _scales(), zeros[:, :1])),
           (ValueError, lambda: QuantizedLinear(_codes() + 13, _scales())),
           (ValueError, lambda: QuantizedLinear(_codes(), _scales(), zeros + 8)),
           (ValueError, lambda: QuantizedLinear.quantize(torch.zeros((4, 64)), group=48)),
           (ValueError, lambda: QuantizedLinear.quantize(torch.zeros((4, 64)), group=0)),
           (ValueError, lambda: QuantizedLinear.quantize(torch.zeros(64), group=32)),
           (TypeError, lambda: QuantizedLinear.quantize(torch.zeros((4, 64)), 32,
                                                        scale_dtype=torch.float32))]
    for i, (exc, call) in enumerate(bad):
        with pytest.raises(exc):
            call()
            pytest.fail(f"case {i} was accepted")
    assert not on_cpu
    w = QuantizedLinear(_codes(), _scales(), zeros)
    assert (w.shape, w.group, w.in_features, w.out_features) == ((32, 128), 64, 128, 32)
    assert on_cpu[0][0] == "sb_w4_pack"
    assert QuantizedLinear(_codes(), _scales(groups=1)).group == 128


def test_product_refusals(on_cpu):
    w = QuantizedLinear(_codes(), _scales())
    on_cpu.clear()
    x, b = torch.zeros((3, 128), dtype=BF16), torch.zeros(32, dtype=BF16)
    bad = [(TypeError, lambda: quantized_linear(x, torch.zeros((32, 128)))),
           (TypeError, lambda: quantized_linear(x.float(), w)),
           (ValueError, lambda: quantized_linear(x[:, :64], w)),
           (ValueError, lambda: quantized_linear(x[0, 0], w)),
           (ValueError, lambda: quantized_linear(x, w, bias=b[:31])),
           (ValueError, lambda: quantized_linear(x, w, bias=b.half())),
           (ValueError, lambda: quantized_linear(x, w, out=x)),
           (ValueError, lambda: quantized_linear(x, w, out=torch.zeros((3, 32)))),
           (ValueError, lambda: quantized_linear(x, w, out=torch.zeros((3, 64), dtype=BF16)[:, ::2])),
           (TypeError, lambda: w.dequantize(torch.float64))]
    for i, (exc, call) in enumerate(bad):
        with pytest.raises(exc):
            call()
            pytest.fail(f"case {i} was accepted")
    assert not on_cpu
    assert quantized_linear(x[:0], w).shape == (0, 32)
    assert not on_cpu
    assert quantized_linear(x[None], w, bias=b).shape == (1, 3, 32)
    assert on_cpu[0][0] == "sb_w4_linear"


def _linear(**over):
    a = dict(y=FAKE, x=FAKE, w=FAKE, t=FAKE, b=None, m=3, n=32, k=128, g=64, xs=128, ys=32, ws=None, wsb=0,
             sdt=2, dt=2)
    a.update(over)
    return _lib.lib().sb_w4_linear(*a.values(), None)


def _pack(**over):
    a = dict(w=FAKE, t=FAKE, c=FAKE, s=FAKE, z=None, n=32, k=128, g=64, cs=128, ss=2, zs=0)
    a.update(over)
    return _lib.lib().sb_w4_pack(*a.values(), None)


def _unpack(**over):
    a = dict(o=FAKE, w=FAKE, t=FAKE, n=32, k=128, g=64, os=128, sdt=2, dt=2)
    a.update(over)
    return _lib.lib().sb_w4_dequantize(*a.values(), None)


@pytest.mark.parametrize("call,over,words", [
    (_linear, dict(dt=0), b"bf16 or fp16"), (_linear, dict(sdt=0), b"scales"), (_linear, dict(y=None), b"null"),
    (_linear, dict(t=None), b"null"), (_linear, dict(m=-1), b"positive"), (_linear, dict(n=0), b"positive"),
    (_linear, dict(g=48), b"multiple of 32"), (_linear, dict(k=100), b"multiple of 32"),
    (_linear, dict(x=FAKE + 2), b"aligned"), (_linear, dict(xs=132), b"aligned"),
    (_linear, dict(m=1 << 31), b"limit"), (_linear, dict(n=1 << 31), b"limit"),
    (_linear, dict(k=(1 << 22) + 64), b"limit"), (_linear, dict(xs=(1 << 22) + 8), b"limit"),
    (_linear, dict(m=4096, n=8192, k=1024, xs=1024), b"workspace"),
    (_linear, dict(m=4096, n=8192, k=1024, xs=1024, ws=FAKE, wsb=100), b"workspace"),
    (_linear, dict(w=FAKE + 8), b"aligned"), (_linear, dict(t=FAKE + 4), b"aligned"),
    (_linear, dict(ys=0), b"overlap"), (_linear, dict(ys=31), b"overlap"),
    (_pack, dict(c=None), b"null"), (_pack, dict(g=16), b"multiple of 32"), (_pack, dict(k=0), b"positive"),
    (_pack, dict(w=FAKE + 8), b"aligned"), (_unpack, dict(dt=3), b"invalid dtype"),
    (_unpack, dict(sdt=3), b"scales"), (_unpack, dict(o=None), b"null"),
])
def test_c_refusals(call, over, words):
    assert call(**over) == _lib.SB_ERR_INVALID_ARGUMENT
    assert words in _lib.lib().sb_last_error_string(), _lib.lib().sb_last_error_string()


def test_sizes():
    size = _lib.size_query
    assert size("sb_w4_codes_size", 16, 128) == 1024
    assert size("sb_w4_codes_size", 17, 160) == 4 * 1024
    assert size("sb_w4_table_size", 16, 128, 128) == 64
    assert size("sb_w4_table_size", 17, 160, 32) == 2 * 8 * 64
    assert size("sb_w4_table_size", 16, 192, 96) == 8 * 64
    assert size("sb_w4_linear_workspace_size", 4, 32, 128, 64, 2) == 0
    assert size("sb_w4_linear_workspace_size", 4096, 8192, 1024, 64, 2) > 0
    assert size("sb_w4_linear_workspace_size", 4096, 32, 128, 48, 2) == 0
    # the few-rows kernel's grid ends at 65535 x 64 rows: more take tiles, whose sums lie there
    assert size("sb_w4_linear_workspace_size", 65535 * 64 + 1, 16, 128, 64, 2) > 0
    assert _linear(m=0, x=None) == _lib.SB_OK
