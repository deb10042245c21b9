"""Refusals of the paged-cache operators (no GPU): argument checks of the Python entry points and
of the C ABI, before any launch, and the 64-bit reference's own quantiser."""

from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

from semblend_amd import _lib
from semblend_amd import paged_cache as pc

from . import paged_reference as ref

FAKE = 4096  # an address that is never read: the checks come first


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_cache_shapes():
    codes = torch.zeros((4, 2, 2, 16, 32), dtype=torch.uint8)
    scales = torch.zeros((4, 2, 2, 16, 2), dtype=torch.uint8)
    assert pc.QuantizedKVCache(codes, scales).shape == (4, 2, 2, 16, 64)
    for c, s, exc in ((codes.int(), scales, TypeError), (codes[:, :1], scales, ValueError),
                      (codes[..., :24], scales, ValueError), (codes, scales[:3], ValueError),
                      (codes[..., ::2], scales[..., :1], ValueError)):
        with pytest.raises(exc):
            pc.QuantizedKVCache(c, s)
    with pytest.raises(ValueError):
        pc.QuantizedKVCache.allocate(2, 1, 16, 48, "cpu")


def test_cpu_tensors_are_refused():
    kv = torch.zeros((4, 2, 2, 16, 64))
    x = torch.zeros((3, 2, 64))
    q4 = pc.QuantizedKVCache.allocate(4, 2, 16, 64, "cpu")
    bt = torch.arange(4, dtype=torch.int32)
    for cache in (kv, q4):
        for call in (lambda c: pc.append_kv_paged(c, x, x, bt, [0, 1, 2]),
                     lambda c: pc.gather_kv_paged(c, bt, [0, 1]),
                     lambda c: pc.paged_attention(x, c, bt, [0, 1, 2])):
            with pytest.raises(RuntimeError, match="device tensors"):
                call(cache)


@pytest.fixture
def on_cpu(monkeypatch):
    """The Python checks behind the device check, with CPU tensors and the library call replaced."""
    calls = []
    cpu = torch.device("cpu")
    monkeypatch.setattr(_lib, "require_device", lambda *t: cpu)
    monkeypatch.setattr(_lib, "as_index", lambda t, d: torch.as_tensor(t).to(torch.int32).reshape(-1))
    monkeypatch.setattr(_lib, "launch", lambda dev, name, *a: calls.append((name, a)))
    return calls


def test_python_refusals(on_cpu):
    kv = torch.zeros((4, 2, 2, 16, 64), dtype=torch.bfloat16)
    q4 = pc.QuantizedKVCache.allocate(4, 2, 16, 64, "cpu")
    x = torch.zeros((3, 2, 64), dtype=torch.bfloat16)
    q = torch.zeros((3, 6, 64), dtype=torch.bfloat16)
    bt = torch.zeros((3, 4), dtype=torch.int32)
    pos = [0, 1, 2]
    ap, at, ga = pc.append_kv_paged, pc.paged_attention, pc.gather_kv_paged
    bad = [
        (TypeError, lambda: ap(kv.float(), x, x, bt, pos)),
        (TypeError, lambda: ap(kv, x, x.float(), bt, pos)),
        (TypeError, lambda: ap(kv, x, x, bt, pos, rope_base=1e4, query=q.float())),
        (ValueError, lambda: ap(kv[:, :1], x, x, bt, pos)),
        (ValueError, lambda: ap(kv, x[..., :32], x[..., :32], bt, pos)),
        (ValueError, lambda: ap(kv, x, x[:2], bt, pos)),
        (ValueError, lambda: ap(kv, x[:, :1], x[:, :1], bt, pos)),
        (ValueError, lambda: ap(kv, x, x, bt, [0, 1])),
        (ValueError, lambda: ap(kv, x, x, bt[:2], pos)),                 # 3 rows, 2 requests
        (ValueError, lambda: ap(kv, x, x, bt, pos, row_starts=[0, 3])),  # not R + 1 entries
        (ValueError, lambda: ap(kv, x, x, bt[0], pos, row_starts=[0, 3])),
        (ValueError, lambda: ap(kv, x, x, bt[None], pos)),
        (ValueError, lambda: ap(kv, x, x, bt[:, :0], pos)),
        (ValueError, lambda: ap(kv, x, x, bt, pos, query=q)),            # no rope_base
        (ValueError, lambda: ap(kv, x, x, bt, pos, rotations=pos)),
        (ValueError, lambda: ap(kv, x, x, bt, pos, rope_base=0.5)),
        (ValueError, lambda: ap(kv, x, x, bt, pos, rope_base=math.nan)),
        (ValueError, lambda: ap(kv, x, x, bt, pos, rope_base=1e4, rotations=[1])),
        (ValueError, lambda: ap(kv, x, x, bt, pos, query_out=q)),
        (ValueError, lambda: ap(kv, x, x, bt, pos, rope_base=1e4, query=q, query_out=x)),
        (TypeError, lambda: at(q.float(), kv, bt, pos)),
        (ValueError, lambda: at(q[0], kv, bt, pos)),
        (ValueError, lambda: at(q[..., :32], kv, bt, pos)),
        (ValueError, lambda: at(q[:, :5], kv, bt, pos)),
        (ValueError, lambda: at(q, q4, bt, pos, window=0)),
        (ValueError, lambda: at(q, q4, bt, pos, window=-3)),
        (ValueError, lambda: at(q, q4, bt, pos, sinks=-1)),
        (ValueError, lambda: at(q, q4, bt, pos, out=x)),
        (ValueError, lambda: at(q, q4, bt, pos, out=q.float())),
        (TypeError, lambda: ga(kv, bt[0], pos, dtype=torch.float32)),
        (TypeError, lambda: ga(q4, bt[0], pos, dtype=torch.float64)),
        (ValueError, lambda: ga(q4, bt[0], pos, num_rows=4)),
        (ValueError, lambda: ga(q4, bt[0], num_rows=-1)),
        (ValueError, lambda: ga(q4, bt[0], pos, out=x)),
    ]
    for i, (exc, call) in enumerate(bad):
        with pytest.raises(exc):
            call()
            pytest.fail(f"case {i} was accepted")
    assert not on_cpu
    ap(kv, x[:0], x[:0], bt, [])          # nothing to do: no launch
    at(q[:0], kv, bt, [])
    assert ga(q4, bt[0], []).shape == (2, 2, 0, 64)
    assert not on_cpu


def _append(**over):
    a = dict(cache=FAKE, scales=None, k=FAKE, v=FAKE, q=None, qo=None, bt=FAKE, ts=4, pos=FAKE,
             rot=None, starts=FAKE, inv=None, n=3, r=2, hkv=2, hq=0, d=64, bs=16, nb=8, nbs=4,
             ks=_i64(128, 64, 1), vs=_i64(128, 64, 1), qs=None, qos=None,
             cs=_i64(4096, 2048, 1024, 64, 1), ss=None, dt=2, cdt=2)
    a.update(over)
    return _lib.lib().sb_append_kv_paged(*a.values(), None)


def _gather(**over):
    a = dict(out=FAKE, cache=FAKE, scales=None, bt=FAKE, pos=FAKE, n=3, hkv=2, d=64, bs=16, nb=8,
             nbs=4, os=_i64(384, 192, 64, 1), cs=_i64(4096, 2048, 1024, 64, 1), ss=None, dt=2,
             cdt=2)
    a.update(over)
    return _lib.lib().sb_gather_kv_paged(*a.values(), None)


def _attend(**over):
    a = dict(out=FAKE, q=FAKE, cache=FAKE, scales=None, bt=FAKE, ts=4, pos=FAKE, starts=FAKE,
             ws=None, wsb=0, n=3, r=2, mr=0, hq=4, hkv=2, d=64, bs=16, nb=8, nbs=4, win=0, sinks=0,
             scale=0.125, qs=_i64(256, 64, 1), os=_i64(256, 64, 1),
             cs=_i64(4096, 2048, 1024, 64, 1), ss=None, dt=2, cdt=2)
    a.update(over)
    return _lib.lib().sb_paged_attention(*a.values(), None)


@pytest.mark.parametrize("call,over,words", [
    (_append, dict(dt=7), b"invalid dtype"),
    (_append, dict(cdt=1), b"dtype"),
    (_append, dict(k=None), b"null"),
    (_append, dict(cdt=3), b"null"),                       # no scales
    (_append, dict(q=FAKE, hq=2), b"null"),                # no query_out
    (_append, dict(n=-1), b"positive"),
    (_append, dict(bs=0), b"positive"),
    (_append, dict(d=63), b"even"),
    (_append, dict(d=514), b"512"),
    (_append, dict(d=48, cdt=3, scales=FAKE, ss=_i64(8, 4, 2, 1, 1)), b"multiple of 32"),
    (_append, dict(starts=None), b"one token per request"),
    (_append, dict(ks=_i64(128, 64, 2)), b"contiguous"),
    (_append, dict(n=1 << 32), b"32 bits"),
    (_gather, dict(dt=3), b"invalid dtype"),
    (_gather, dict(cdt=0), b"dtype"),
    (_gather, dict(out=None), b"null"),
    (_gather, dict(nb=0), b"positive"),
    (_gather, dict(os=_i64(1, 1, 1, 2)), b"contiguous"),
    (_gather, dict(d=1024), b"512"),
    (_attend, dict(dt=5), b"invalid dtype"),
    (_attend, dict(cdt=0), b"dtype"),
    (_attend, dict(pos=None), b"null"),
    (_attend, dict(hq=5), b"multiple"),
    (_attend, dict(d=1024), b"512"),
    (_attend, dict(win=-1), b"negative"),
    (_attend, dict(sinks=-1), b"negative"),
    (_attend, dict(starts=None), b"one row per request"),
    (_attend, dict(qs=_i64(256, 64, 2)), b"contiguous"),
    (_attend, dict(n=1 << 30), b"32 bits"),
    (_attend, dict(cs=_i64(1 << 33, 2048, 1024, 64, 1)), b"4 GiB"),
    (_attend, dict(n=1, r=1, starts=None, nbs=4096), b"workspace"),   # split, no workspace
])
def test_c_refusals(call, over, words):
    assert call(**over) == _lib.SB_ERR_INVALID_ARGUMENT
    assert words in _lib.lib().sb_last_error_string(), _lib.lib().sb_last_error_string()


def test_empty_calls():
    assert _append(n=0, k=None) == _lib.SB_OK
    assert _gather(n=0, out=None) == _lib.SB_OK
    assert _attend(n=0, q=None) == _lib.SB_OK


def test_workspace_query():
    size = lambda *a: _lib.size_query("sb_paged_attention_workspace_size", *a)
    # one row over a long context is split; 512 of them over short ones are not
    assert size(1, 1, 0, 1, 28, 4, 128, 16, 1000, 0, 0, 2, 2) > 0
    assert size(512, 512, 0, 1, 32, 8, 128, 16, 100, 0, 0, 2, 2) == 0
    assert size(1, 1, 0, 1, 28, 4, 96, 16, 1000, 0, 0, 2, 2) == 0      # not on the matrix cores
    assert size(0, 1, 0, 1, 28, 4, 128, 16, 1000, 0, 0, 2, 3) == 0
    assert size(4, 1, 0, 1, 28, 3, 128, 16, 1000, 0, 0, 2, 2) == 0


def test_reference_quantiser():
    """The reference's own codes at hand-made values."""
    x = torch.zeros(32, dtype=torch.float64)
    x[:10] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.0, -0.26])
    code, scale = ref.quantize(x[None])
    assert scale.tolist() == [[127]]
    assert code[0, :10].tolist() == [0, 2, 2, 4, 4, 6, 6, 7, 7, 9]
    code, scale = ref.quantize((x * 1.0001)[None])   # above 7: the next power of two
    assert scale.tolist() == [[128]] and code[0, 8].item() == 6
    packed = torch.tensor([[0x21] * 16], dtype=torch.uint8)
    assert ref.dequantize(packed, torch.tensor([[128]], dtype=torch.uint8))[0, :2].tolist() == [1.0, 2.0]


@pytest.mark.parametrize("host", [True, False])
def test_entries_called_with_python_values(host, monkeypatch):
    """Both forms of a call with Python values (through the host library, or ctypes without it)
    reach the entry point with the same arguments: its refusals say which one was wrong."""
    if not host:
        monkeypatch.setattr(_lib, "_host", False)
    strides = dict(ks=(128, 64, 1), vs=(128, 64, 1), cs=(4096, 2048, 1024, 64, 1))
    refusals = [(_append, strides | dict(cdt=1), "dtype"),
                (_append, strides | dict(k=None), "null"),
                (_append, strides | dict(ks=(128, 64, 2)), "contiguous"),
                (_append, strides | dict(n=1 << 32), "32 bits"),
                (_append, strides | dict(d=48, cdt=3, scales=FAKE, ss=(8, 4, 2, 1, 1)), "of 32"),
                (_gather, dict(os=(1, 1, 1, 2), cs=strides["cs"]), "contiguous"),
                (_gather, dict(os=(384, 192, 64, 1), cs=strides["cs"], nb=0), "positive"),
                (_attend, dict(qs=(256, 64, 1), os=(256, 64, 1), cs=(1 << 33, 2048, 1024, 64, 1)),
                 "4 GiB"),
                (_attend, dict(qs=(256, 64, 2), os=(256, 64, 1), cs=strides["cs"]), "contiguous"),
                (_attend, dict(qs=(256, 64, 1), os=(256, 64, 1), cs=strides["cs"], win=-1),
                 "negative")]
    names = {_append: "sb_append_kv_paged", _gather: "sb_gather_kv_paged",
             _attend: "sb_paged_attention"}
    for call, over, words in refusals:
        entry = _lib._entry(names[call])
        assert (type(entry).__name__ == "builtin_function_or_method") == host
        with monkeypatch.context() as m:  # (the same argument list, given to the callable)
            m.setattr(_lib, "lib", lambda entry=entry, name=names[call]:
                      type("entries", (), {name: staticmethod(entry)}))
            assert call(**over) == _lib.SB_ERR_INVALID_ARGUMENT
        assert words in _lib.lib().sb_last_error_string().decode()
    # nothing to do: every argument is accepted
    with monkeypatch.context() as m:
        m.setattr(_lib, "lib", lambda entry=entry: type("entries", (), {
            "sb_paged_attention": staticmethod(entry)}))
        assert _attend(n=0, qs=(256, 64, 1), os=(256, 64, 1), cs=strides["cs"]) == _lib.SB_OK


def test_entries_refuse_other_values():
    entry = _lib._entry("sb_gather_kv_paged")
    good = [FAKE, FAKE, None, FAKE, None, 0, 2, 64, 16, 8, 4, (1, 1, 1, 1), (1, 1, 1, 1, 1), None,
            2, 2, None]
    assert entry(*good) == _lib.SB_OK                     # no rows: nothing is read
    for i, bad in ((0, "x"), (0, 1.5), (5, 2.5), (5, None), (5, 1 << 64), (11, [1, 1, 1, 1]),
                   (11, (1,) * 6), (11, (1, 1, 1, "1")), (14, 1 << 40), (14, None)):
        args = list(good)
        args[i] = bad
        with pytest.raises((TypeError, OverflowError)):
            entry(*args)
    with pytest.raises(TypeError):
        entry(*good[:-1])
    assert _lib.host_lib().sb_host_entry(b"sb_version", FAKE) is None


def test_workspace_of_many_requests():
    """A chunk or several among many requests: the partials of split key ranges go by what a round or
    two of workgroups can hold, not by the row tiles that such a batch might have."""
    size = lambda *a: _lib.size_query("sb_paged_attention_workspace_size", *a)
    # (rows, requests, query and KV heads, pages of a table)
    for rows, requests, hq, hkv, width in ((767, 256, 32, 8, 512), (300, 128, 32, 8, 512),
                                           (575, 64, 32, 8, 512), (127, 64, 28, 4, 512),
                                           (511, 256, 28, 4, 2048), (4000, 1000, 32, 8, 2048)):
        for dt, cdt in ((2, 2), (1, 1), (2, 3)):
            got = size(rows, requests, 1, rows, hq, hkv, 128, 16, width, 0, 0, dt, cdt)
            assert got <= 100e6, (rows, requests, got)
    # (a launch of n items is split while (n - 1) of them are below two rounds of 256)
    rng = random.Random(1)
    for _ in range(2000):
        hkv = rng.choice((1, 2, 4, 8, 16, 32))
        requests, d = int(2 ** rng.uniform(0, 11)), rng.choice((64, 128))
        rows = requests + int(2 ** rng.uniform(0, 12))
        got = size(rows, requests, 1, rng.choice((0, rows)), hkv * rng.choice((1, 4, 7)), hkv, d, 16,
                   int(2 ** rng.uniform(0, 14)), rng.choice((0, 1, 700, 40000)), rng.choice((0, 4)),
                   rng.choice((1, 2)), rng.choice((1, 2, 3)))
        assert got <= 4 * (d + 2) * 1024 * (256 + 16), (rows, requests, hkv, got)


def test_gradients_are_refused_not_lost(on_cpu):
    """A result whose gradient torch would ask for raises there; others carry no record."""
    kv = torch.zeros((4, 2, 2, 16, 64))
    q4 = pc.QuantizedKVCache.allocate(4, 2, 16, 64, "cpu")
    bt = torch.zeros((3, 4), dtype=torch.int32)
    pos = [0, 1, 2]
    x = torch.zeros((3, 2, 64))
    w = torch.ones(64, requires_grad=True)
    calls = {
        "paged_attention": lambda q, out=None, c=kv: pc.paged_attention(q, c, bt, pos, out=out),
        "append_kv_paged": lambda q, out=None, c=kv: pc.append_kv_paged(
            c, x, x, bt, pos, rope_base=1e4, query=q, query_out=out),
    }
    for name, call in calls.items():
        for cache in (kv, q4):
            for q in (torch.zeros((3, 6, 64), requires_grad=True), torch.ones((3, 6, 64)) * w,
                      (torch.ones((3, 64, 6)) * w[None, :, None]).transpose(1, 2)):
                got = call(q, c=cache)
                assert got.requires_grad and got.shape == q.shape
                with pytest.raises(RuntimeError, match=f"{name} has no backward"):
                    (got * 2).sum().backward()
                with torch.no_grad():
                    assert not call(q, c=cache).requires_grad
                assert not call(q.detach(), c=cache).requires_grad
                out = torch.zeros(q.shape)
                assert call(q, out, cache) is out and not out.requires_grad
    got = pc.paged_attention(x, kv.clone().requires_grad_(), bt, pos)
    with pytest.raises(RuntimeError, match="no backward"):
        got.sum().backward()
