"""Rotary embeddings and 4-bit weights without a GPU: threads, configurations, outputs whose rows overlap."""

from __future__ import annotations

import threading

import torch

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
