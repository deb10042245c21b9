"""Rotary embeddings and 4-bit weights without a GPU: threads, configurations, outputs whose rows overlap."""

from __future__ import annotations

import ctypes
import shutil
import subprocess
import threading
from pathlib import Path

import pytest
import torch

from semblend_amd import _lib
from semblend_amd.rotary import RotaryEmbedding


def test_first_calls_of_two_threads_share_one_table():
    """A table that a call or a captured graph reads lives as long as the embedding: a second thread's copy,
    made at the same time, does not take its place."""
    rot = RotaryEmbedding.from_config(64)
    both, got, cpu = threading.Barrier(2, timeout=10), [None, None], torch.device("cpu")

    class Frequencies:
        kept = rot._inv_freq

        def to(self, dev):
            both.wait()  # (each thread has seen that there is no table)
            return self.kept.clone()

    rot._inv_freq = Frequencies()

    def first(i):
        got[i] = rot._table(cpu, 64)

    threads = [threading.Thread(target=first, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    assert got[0] is not None and got[0] is got[1]
    assert rot._table(cpu, 64) is got[0]


HERE = Path(__file__).resolve().parent
FAKE = 4096  # an address that is never read: the checks come first


def _i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_rows_overlap_is_that_of_all_pairs(tmp_path):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "overlap_check"
    subprocess.run([gxx, "-O2", "-std=c++17", "-o", str(exe), str(HERE / "overlap_check.cpp")], check=True,
                   capture_output=True, text=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and " 0 wrong" in r.stdout, r.stdout


@pytest.mark.parametrize("strides", [(64, 64), (64, 128), (200, 32), (0, 64), (256, 0), (-64, 64), (128, 96)])
@pytest.mark.parametrize("out", ["query", "key", "append"])
def test_outputs_whose_rows_overlap_are_refused(out, strides):
    """Three tokens of four heads of 64."""
    plain, bad = _i64(256, 64, 1), _i64(*strides, 1)
    if out == "append":
        cache = _i64(8192, 4096, 1024, 64, 1)
        rc = _lib.lib().sb_append_kv_rotary_paged(
            FAKE, None, FAKE, FAKE, FAKE, FAKE, FAKE, 4, FAKE, None, None, FAKE, 3, 1, 4, 4, 64, 16, 8, 4, plain,
            plain, plain, bad, cache, None, 32, 1, 1.0, 2, 2, None)
    else:
        key = out == "key"
        rc = _lib.lib().sb_apply_rotary(
            FAKE, FAKE, FAKE if key else None, FAKE if key else None, FAKE, FAKE, 3, 4, 4 if key else 0, 64, plain,
            plain if key else bad, plain if key else None, bad if key else None, 32, 1, 1.0, 2, None)
    assert rc == _lib.SB_ERR_INVALID_ARGUMENT
    assert b"overlap" in _lib.lib().sb_last_error_string()


@pytest.mark.parametrize("scaling", [
    {"rope_type": "default"}, {"type": "linear", "factor": 4.0},
    {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
     "original_max_position_embeddings": 8192},
    {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}])
def test_base_and_part_of_the_dictionary(scaling):
    """A dictionary that holds the base and the turned share of the head gives what the arguments give."""
    want = RotaryEmbedding.from_config(128, 5e5, rotary_dim=64, scaling=scaling)
    both = {**scaling, "rope_theta": 500000, "partial_rotary_factor": 0.5}
    for got in (RotaryEmbedding.from_config(128, scaling=both),
                RotaryEmbedding.from_config(128, 5e5, 64, scaling=both),
                RotaryEmbedding.from_config(128, rotary_dim=64, scaling={**scaling, "rope_theta": 5e5}),
                RotaryEmbedding.from_config(128, 5e5, scaling={**scaling, "partial_rotary_factor": 0.5})):
        assert torch.equal(got.inv_freq, want.inv_freq)
        assert (got.rotary_dim, got.factor) == (64, want.factor)
    for bad in (dict(rope_base=1e4), dict(rotary_dim=128), dict(rotary_dim=32)):
        with pytest.raises(ValueError, match="holds"):
            RotaryEmbedding.from_config(128, scaling=both, **bad)
    for part in (0.0, 1.5, 0.01):
        with pytest.raises(ValueError, match="rotary_dim"):
            RotaryEmbedding.from_config(128, scaling={**scaling, "partial_rotary_factor": part})
    plain = RotaryEmbedding.from_config(128)
    assert torch.equal(plain.inv_freq, RotaryEmbedding.from_config(128, 1e4).inv_freq)


def test_null_is_what_is_not_set():
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    unset = dict.fromkeys(("beta_fast", "beta_slow", "attention_factor", "mscale", "mscale_all_dim", "truncate",
                           "rope_theta", "partial_rotary_factor", "type"))
    want = RotaryEmbedding.from_config(128, 1e6, scaling=yarn)
    got = RotaryEmbedding.from_config(128, 1e6, scaling={**unset, **yarn})
    assert torch.equal(got.inv_freq, want.inv_freq) and got.factor == want.factor
    older = {"rope_type": None, "type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}
    assert torch.equal(RotaryEmbedding.from_config(128, 1e6, scaling=older).inv_freq, want.inv_freq)
    whole = RotaryEmbedding.from_config(128, 1e6, scaling={**yarn, "truncate": False})
    assert not torch.equal(whole.inv_freq, want.inv_freq)
    with pytest.raises(ValueError, match="factor"):
        RotaryEmbedding.from_config(128, 1e6, scaling={**yarn, "factor": None})


@pytest.mark.parametrize("over,words", [(dict(stride=127), b"overlap"), (dict(stride=0), b"overlap"),
                                        (dict(packed=FAKE + 8), b"aligned"), (dict(table=FAKE + 4), b"aligned")])
def test_dequantize_refusals(over, words):
    a = dict(packed=FAKE, table=FAKE, stride=128)
    a.update(over)
    rc = _lib.lib().sb_w4_dequantize(FAKE, a["packed"], a["table"], 32, 128, 64, a["stride"], 2, 2, None)
    assert rc == _lib.SB_ERR_INVALID_ARGUMENT
    assert words in _lib.lib().sb_last_error_string()
