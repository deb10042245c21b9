"""Rotary embeddings without a GPU: frequencies of every scaling against 64-bit formulas, refusals of
the Python entry points and of the C ABI before any launch."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from semblend_amd import _lib
from semblend_amd import paged_cache as pc
from semblend_amd import rope_correction as rc
from semblend_amd.rotary import RotaryEmbedding, apply_rotary

FAKE = 4096  # an address that is never read: the checks come first


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def _plain(base, n):
    return [base ** (-2 * i / n) for i in range(n // 2)]


def test_plain_frequencies_are_the_paths_own():
    for base, d in ((1e4, 128), (1e6, 64), (5e5, 80)):
        got = RotaryEmbedding.from_config(d, base)
        assert torch.equal(got.inv_freq, rc.inv_freq_table(base, d, torch.device("cpu")))
        assert (got.rotary_dim, got.head_dim, got.layout, got.factor) == (d, d, "half", 1.0)
    part = RotaryEmbedding.from_config(128, 1e4, rotary_dim=32, layout="interleaved")
    assert part.rotary_dim == 32
    assert torch.equal(part.inv_freq, rc.inv_freq_table(1e4, 32, torch.device("cpu")))


def _close(got, want):
    # fp32 evaluation: base^x (two ulps), its reciprocal, and up to six operations more
    torch.testing.assert_close(got.double(), torch.tensor(want, dtype=torch.float64),
                               rtol=12 * 2.0 ** -24, atol=0)


def test_linear_scaling():
    got = RotaryEmbedding.from_config(64, 1e4, scaling={"type": "linear", "factor": 4.0})
    _close(got.inv_freq, [f / 4 for f in _plain(1e4, 64)])


def test_scaling_by_wavelength():
    cfg = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}
    got = RotaryEmbedding.from_config(128, 5e5, scaling=cfg)
    want, kinds = [], set()
    for f in _plain(5e5, 128):
        wave = 2 * math.pi / f
        t = (8192 / wave - 1) / 3
        kinds.add("long" if t < 0 else "short" if t > 1 else "between")
        want.append(f / 8 if t < 0 else f if t > 1 else (1 - t) * f / 8 + t * f)
    assert kinds == {"long", "short", "between"}
    # (the blend's t is off by a few 2^-24 of 8192 / wave < 4, of a result of at least f / 8)
    torch.testing.assert_close(got.inv_freq.double(), torch.tensor(want, dtype=torch.float64),
                               rtol=64 * 2.0 ** -24, atol=0)
    assert got.factor == 1.0


@pytest.mark.parametrize("more,factor", [
    ({}, 0.1 * math.log(4.0) + 1), ({"attention_factor": 1.5}, 1.5),
    ({"mscale": 0.7, "mscale_all_dim": 1.0}, (0.07 * math.log(4) + 1) / (0.1 * math.log(4) + 1))])
def test_yarn(more, factor):
    cfg = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768, **more}
    got = RotaryEmbedding.from_config(128, 1e6, scaling=cfg)
    assert abs(got.factor - factor) < 1e-12
    at = lambda turns: 128 * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(1e6))
    low, high = math.floor(at(32)), math.ceil(at(1))
    want = []
    for i, f in enumerate(_plain(1e6, 128)):
        r = min(max((i - low) / (high - low), 0.0), 1.0)
        want.append(f / 4 * r + f * (1 - r))
    torch.testing.assert_close(got.inv_freq.double(), torch.tensor(want, dtype=torch.float64),
                               rtol=64 * 2.0 ** -24, atol=0)


def test_embedding_refusals():
    one = [1.0, 0.5]
    for bad in (lambda: RotaryEmbedding([], 64), lambda: RotaryEmbedding([[1.0, .5]], 64),
                lambda: RotaryEmbedding([1.5, 0.1], 64), lambda: RotaryEmbedding([-.1, 0.1], 64),
                lambda: RotaryEmbedding([math.nan, 0.1], 64), lambda: RotaryEmbedding(one, 63),
                lambda: RotaryEmbedding(one, 514), lambda: RotaryEmbedding(one, 2),
                lambda: RotaryEmbedding([0.5], 64), lambda: RotaryEmbedding(one, 64, "neox"),
                lambda: RotaryEmbedding(one, 64, factor=0.0),
                lambda: RotaryEmbedding(one, 64, factor=math.nan),
                lambda: RotaryEmbedding.from_config(64, 0.5),
                lambda: RotaryEmbedding.from_config(64, rotary_dim=66),
                lambda: RotaryEmbedding.from_config(64, rotary_dim=3),
                lambda: RotaryEmbedding.from_config(64, scaling={"type": "dynamic", "factor": 2.0}),
                lambda: RotaryEmbedding.from_config(64, scaling={"factor": 2.0}),
                lambda: RotaryEmbedding.from_config(64, scaling={"type": "linear"}),
                lambda: RotaryEmbedding.from_config(64, scaling={"type": "linear", "factor": .5}),
                lambda: RotaryEmbedding.from_config(64, scaling={"type": "yarn", "factor": 2.0})):
        with pytest.raises(ValueError):
            bad()
            pytest.fail("accepted")
    kept = RotaryEmbedding(one, 64)
    kept.inv_freq.zero_()  # (a copy)
    assert kept.inv_freq.tolist() == one
    assert RotaryEmbedding([0.5], 64, "interleaved").rotary_dim == 2


@pytest.fixture
def on_cpu(monkeypatch):
    """The Python checks behind the device check, with CPU tensors and the library call replaced."""
    calls = []
    cpu = torch.device("cpu")
    monkeypatch.setattr(_lib, "require_device", lambda *t: cpu)
    monkeypatch.setattr(_lib, "as_index", lambda t, d: torch.as_tensor(t).to(torch.int32).reshape(-1))
    monkeypatch.setattr(_lib, "launch", lambda dev, name, *a: calls.append((name, a)))
    return calls


def test_cpu_tensors_are_refused():
    rot = RotaryEmbedding.from_config(64)
    x = torch.zeros((3, 2, 64))
    with pytest.raises(RuntimeError, match="device tensors"):
        apply_rotary(x, [0, 1, 2], rot)
    with pytest.raises(RuntimeError, match="device tensors"):
        pc.append_kv_paged(torch.zeros((4, 2, 2, 16, 64)), x, x, [0], [0, 1, 2], rotary=rot)


def test_python_refusals(on_cpu):
    rot = RotaryEmbedding.from_config(64)
    more = RotaryEmbedding.from_config(64, scaling={"type": "yarn", "factor": 2.0,
                                                    "original_max_position_embeddings": 4096})
    x, k = torch.zeros((3, 6, 64)), torch.zeros((3, 2, 64))
    pos = [0, 1, 2]
    kv, bt = torch.zeros((4, 2, 2, 16, 64)), torch.zeros((3, 4), dtype=torch.int32)
    ap = pc.append_kv_paged
    bad = [(ValueError, lambda: apply_rotary(x[0], pos, rot)),
           (TypeError, lambda: apply_rotary(x, pos, 1e4)),
           (TypeError, lambda: apply_rotary(x.double(), pos, rot)),
           (TypeError, lambda: apply_rotary(x, pos, rot, key=k.half())),
           (ValueError, lambda: apply_rotary(x[..., :32], pos, rot)),
           (ValueError, lambda: apply_rotary(x, pos[:2], rot)),
           (ValueError, lambda: apply_rotary(x, pos, rot, key=k[:2])),
           (ValueError, lambda: apply_rotary(x, pos, rot, key=k[..., :32])),
           (ValueError, lambda: apply_rotary(x, pos, rot, query_out=k)),
           (ValueError, lambda: apply_rotary(x, pos, rot, query_out=x.half())),
           (ValueError, lambda: apply_rotary(x, pos, rot, key=k, key_out=x)),
           (ValueError, lambda: apply_rotary(x, pos, rot, key_out=k)),
           (ValueError, lambda: ap(kv, k, k, bt, pos, rope_base=1e4, rotary=rot)),
           (ValueError, lambda: ap(kv[..., :32], k[..., :32], k[..., :32], bt, pos, rotary=rot)),
           (ValueError, lambda: ap(kv, k, k, bt, pos, rotary=more, rotations=pos, query=x))]
    for i, (exc, call) in enumerate(bad):
        with pytest.raises(exc):
            call()
            pytest.fail(f"case {i} was accepted")
    assert not on_cpu
    assert apply_rotary(x[:0], [], rot).shape == (0, 6, 64)
    assert not on_cpu
    apply_rotary(x, pos, rot, key=k)
    ap(kv, k, k, bt, pos, rotary=more, rotations=pos)
    assert [c[0] for c in on_cpu] == ["sb_apply_rotary", "sb_append_kv_rotary_paged"]
    assert on_cpu[1][1][-5:] == (32, 1, 1.0, 0, 0)  # rotations: the factor is in the donor's K


def _apply(**over):
    a = dict(qo=FAKE, q=FAKE, ko=None, k=None, pos=FAKE, inv=FAKE, n=3, hq=4, hk=0, d=64,
             qs=_i64(256, 64, 1), qos=_i64(256, 64, 1), ks=None, kos=None, pairs=32, layout=1,
             factor=1.0, dt=2)
    a.update(over)
    return _lib.lib().sb_apply_rotary(*a.values(), None)


def _append(**over):
    a = dict(cache=FAKE, scales=None, k=FAKE, v=FAKE, q=None, qo=None, bt=FAKE, ts=4, pos=FAKE,
             rot=None, starts=FAKE, inv=FAKE, n=3, r=2, hkv=2, hq=0, d=128, bs=16, nb=8, nbs=4,
             ks=_i64(256, 128, 1), vs=_i64(256, 128, 1), qs=None, qos=None,
             cs=_i64(8192, 4096, 2048, 128, 1), ss=None, pairs=64, layout=1, factor=1.0, dt=2, cdt=2)
    a.update(over)
    return _lib.lib().sb_append_kv_rotary_paged(*a.values(), None)


def _scatter(**over):
    a = dict(kv=FAKE, dn=FAKE, layers=2, bt=FAKE, dp=FAKE, tp=FAKE, inv=FAKE, n=3, h=2, bs=16, d=64,
             sd=32, nb=8, nbs=4, cs=_i64(4096, 2048, 1024, 64, 1), ds=_i64(4096, 2048, 64, 1),
             pairs=32, layout=1, dt=2, flags=0)
    a.update(over)
    return _lib.lib().sb_rotary_scatter_paged_layers(*a.values(), None)


def _shift(entry="sb_rotary_shift_paged_layers", **over):
    a = dict(kv=FAKE, layers=2, bt=FAKE, pos=FAKE, dl=FAKE, n=3, inv=FAKE, h=2, bs=16, d=64, nb=8,
             nbs=4, cs=_i64(4096, 1024, 64, 1), pairs=32, layout=1, dt=2)
    a.update(over)
    return getattr(_lib.lib(), entry)(*a.values(), None)


def _shift_host(**over):
    from ctypes import POINTER, c_int32, cast
    addr = over.pop("pos", FAKE)
    over["pos"] = over["dl"] = None if addr is None else cast(addr, POINTER(c_int32))
    return _shift("sb_rotary_shift_paged_layers_host", **over)


Q4 = dict(cdt=3, scales=FAKE, ss=_i64(1, 1, 1, 1, 1))


@pytest.mark.parametrize("call,over,words", [
    (_apply, dict(dt=4), b"invalid dtype"), (_apply, dict(q=None), b"null"),
    (_apply, dict(inv=None), b"null"), (_apply, dict(k=FAKE), b"null"), (_apply, dict(n=-1), b"positive"),
    (_apply, dict(hq=0), b"positive"), (_apply, dict(d=62, pairs=32), b"head_dim / 2"),
    (_apply, dict(d=63), b"even"), (_apply, dict(d=514), b"512"), (_apply, dict(pairs=0), b"pair"),
    (_apply, dict(pairs=31), b"even number"), (_apply, dict(layout=2), b"layout"),
    (_apply, dict(factor=0.0), b"factor"), (_apply, dict(factor=math.nan), b"factor"),
    (_apply, dict(qs=_i64(256, 64, 2)), b"contiguous"),
    (_apply, dict(qos=_i64(0, 64, 1)), b"overlap"), (_apply, dict(qos=_i64(256, 0, 1)), b"overlap"), (_apply, dict(n=1 << 31), b"limit"),
    (_append, dict(inv=None), b"null"), (_append, dict(pairs=65), b"head_dim / 2"),
    (_append, dict(layout=-1), b"layout"), (_append, dict(Q4, pairs=16), b"whole blocks"),
    (_append, dict(Q4, pairs=48), b"whole blocks"), (_append, dict(Q4, pairs=8, layout=0), b"whole blocks"),
    (_append, dict(factor=-1.0), b"factor"),
    (_scatter, dict(dn=None), b"null"), (_scatter, dict(sd=0), b"positive"), (_scatter, dict(flags=2), b"flags"),
    (_scatter, dict(layers=0), b"positive"), (_scatter, dict(layers=5000), b"limit"),
    (_scatter, dict(pairs=33), b"head_dim / 2"), (_scatter, dict(ds=_i64(1, 1, 1, 2)), b"contiguous"),
    (_shift, dict(pos=None), b"null"), (_shift, dict(dt=3), b"invalid dtype"),
    (_shift, dict(cs=_i64(1, 1, 1, 2)), b"contiguous"), (_shift, dict(nbs=0), b"positive"),
    (_shift_host, dict(n=257), b"256"), (_shift_host, dict(pos=None), b"null"),
])
def test_c_refusals(call, over, words):
    assert call(**over) == _lib.SB_ERR_INVALID_ARGUMENT
    assert words in _lib.lib().sb_last_error_string(), _lib.lib().sb_last_error_string()


def test_empty_calls():
    assert _apply(n=0, q=None) == _lib.SB_OK
    assert _append(n=0, inv=None) == _lib.SB_OK
    assert _scatter(n=0, kv=None) == _lib.SB_OK
    assert _shift(n=0, kv=None) == _lib.SB_OK
    assert _shift_host(n=0, pos=None) == _lib.SB_OK
