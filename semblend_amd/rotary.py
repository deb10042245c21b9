"""A model's own rotary positions: interleaved or half pairs, part of the head, frequencies scaled
for long contexts.

The reference rotates interleaved pairs (2i, 2i + 1) of whole heads by the plain frequencies
1 / base^(2i / head_dim) (semblend_core/rope_correction.py:163-178, :317-326). Published models
mostly pair element i with element i + n / 2 of the n that they rotate, some rotate the first part of
a head only, and many scale the frequencies. A :class:`RotaryEmbedding` says which; with it

* :func:`apply_rotary` turns the Q and K rows of new tokens (no reference counterpart);
* ``paged_cache.append_kv_paged(..., rotary=)`` does so on the way into the pages;
* ``rope_correction.rope_correct_scatter_paged_layers``, ``prepare_scatter_paged_layers`` and
  ``apply_rope_deltas_inplace_layers`` (``rotary=``) correct a donor's K by the way it has moved;
* ``triton_kernels.qkv_projection_paged`` and ``partial_prefill_layer_paged`` (``rotary=``) run a
  layer of such a model.

Angles, sines and cosines are taken in 64 bits from the embedding's fp32 frequencies; rows are turned
in fp32 (fp32 rows: in 64 bits) and rounded once.
"""

from __future__ import annotations

import math

import torch

from . import _lib
from .paged_cache import _device, _index, _like, _recorded, _rows

__all__ = ["RotaryEmbedding", "apply_rotary"]


def _base_frequencies(rope_base: float, rotary_dim: int) -> torch.Tensor:
    # (the expression of rope_correction.inv_freq_table: the same bits)
    return 1.0 / (rope_base ** (torch.arange(0, rotary_dim, 2, dtype=torch.float32) / rotary_dim))


def _number(scaling: dict, key: str, default=None) -> float:
    value = scaling.get(key)
    if value is None:  # (configurations write null for what is not set)
        value = default
    if value is None:
        raise ValueError(f"scaling needs {key!r}")
    return float(value)


def _by_wavelength(f: torch.Tensor, scaling: dict) -> torch.Tensor:
    """Frequencies of long waves divided by the factor, of short ones kept, blended between: the
    scaling that the Llama 3.1 models were published with (2024), "llama3" in configurations."""
    factor = _number(scaling, "factor")
    lo, hi = _number(scaling, "low_freq_factor"), _number(scaling, "high_freq_factor")
    length = _number(scaling, "original_max_position_embeddings")
    if not (factor >= 1 and 0 < lo < hi and length > 0):
        raise ValueError("scaling by wavelength needs factor >= 1, 0 < low_freq_factor < "
                         "high_freq_factor and a positive length")
    wave = 2 * math.pi / f
    t = (length / wave - lo) / (hi - lo)
    between = (1 - t) * f / factor + t * f
    return torch.where(wave > length / lo, f / factor, torch.where(wave < length / hi, f, between))


def _by_rotations(f: torch.Tensor, rope_base: float, scaling: dict) -> tuple[torch.Tensor, float]:
    """(frequencies, factor of cosine and sine) of the YaRN method (B. Peng et al., "YaRN: Efficient
    Context Window Extension of Large Language Models", 2023): pairs that turn less than beta_slow
    times over the trained length are divided by the factor, those of more than beta_fast kept, a
    linear ramp over the pairs between. Two keys are not the paper's but later configurations', with
    the meaning that the transformers library documents: "truncate" (by default the ramp's ends are
    whole pairs) and "mscale" with "mscale_all_dim" (the factor is a quotient of two)."""
    factor = _number(scaling, "factor")
    length = _number(scaling, "original_max_position_embeddings")
    fast, slow = _number(scaling, "beta_fast", 32.0), _number(scaling, "beta_slow", 1.0)
    if not (factor >= 1 and length > 0 and fast > slow > 0 and rope_base > 1):
        raise ValueError("yarn scaling needs factor >= 1, a positive length, beta_fast > beta_slow > "
                         "0 and a rope_base above 1")
    dim = 2 * f.shape[0]

    def pair_of(turns: float) -> float:
        return dim * math.log(length / (turns * 2 * math.pi)) / (2 * math.log(rope_base))

    low, high = pair_of(fast), pair_of(slow)
    truncate = scaling.get("truncate")
    if truncate is None or truncate:
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, dim - 1)
    if low == high:
        high += 0.001
    ramp = ((torch.arange(dim // 2, dtype=torch.float32) - low) / (high - low)).clamp(0, 1)
    given = scaling.get("attention_factor")
    if given is None:
        def grown(m: float) -> float:
            return 0.1 * m * math.log(factor) + 1.0 if factor > 1 else 1.0
        m, m_all = scaling.get("mscale"), scaling.get("mscale_all_dim")
        given = grown(float(m)) / grown(float(m_all)) if m and m_all else grown(1.0)
    return f / factor * ramp + f * (1 - ramp), float(given)


class RotaryEmbedding:
    """How a model turns its Q and K rows: ``inv_freq`` (n / 2 frequencies of 0 to 1, kept in fp32 as
    models keep them) turn the first n elements of a head of ``head_dim``; ``layout`` "half" pairs
    element i with i + n / 2 (n a multiple of 4), "interleaved" 2i with 2i + 1; cosine and sine are
    multiplied by ``factor`` where rows are first turned (a cached K that moves holds it already).
    Immutable; a device's copy of the frequencies is made at the first call there, which cannot be
    inside a graph capture, and lives as long as the embedding: a captured graph's calls read it."""

    def __init__(self, inv_freq, head_dim: int, layout: str = "half", factor: float = 1.0):
        f = torch.as_tensor(inv_freq).detach().to(device="cpu", dtype=torch.float32).clone()
        if f.dim() != 1 or f.shape[0] == 0:
            raise ValueError("inv_freq must be a list of frequencies")
        if not bool(((f >= 0) & (f <= 1)).all()):
            raise ValueError("frequencies must lie in 0 .. 1")
        if layout not in _lib.SB_ROTARY:
            raise ValueError(f"layout must be one of {sorted(_lib.SB_ROTARY)}, got {layout!r}")
        head_dim = int(head_dim)
        if head_dim < 2 or head_dim % 2 or head_dim > 512:
            raise ValueError("head_dim must be even and at most 512")
        if 2 * f.shape[0] > head_dim:
            raise ValueError(f"{f.shape[0]} frequencies turn more than head_dim = {head_dim}")
        if layout == "half" and f.shape[0] % 2:
            raise ValueError("the half layout needs an even number of frequencies")
        factor = float(factor)
        if not 0 < factor <= 1e4:
            raise ValueError("factor must be positive and at most 1e4")
        self._inv_freq, self._head_dim, self._layout, self._factor = f, head_dim, layout, factor
        self._code = _lib.SB_ROTARY[layout]
        self._tables: dict = {}

    @classmethod
    def from_config(cls, head_dim: int, rope_base: float | None = None,
                    rotary_dim: int | None = None, layout: str = "half",
                    scaling: dict | None = None) -> "RotaryEmbedding":
        """From a model's configuration: ``rotary_dim`` elements of a head are turned (all by default)
        by 1 / rope_base^(2i / rotary_dim) (10000 by default), changed by ``scaling``, a dictionary as
        configurations hold it ("rope_type" or "type" and its numbers): "default", "linear", "llama3"
        (by wavelength) and "yarn". Others are refused: give their frequencies to the constructor. (A
        scaling that changes with the length of the context turns cached K of other lengths by
        other frequencies, which no shift corrects.) Where the dictionary holds "rope_theta" or
        "partial_rotary_factor", these are the rope_base and the share of the head that is turned; an
        argument that says otherwise is refused."""
        theta, part = ((scaling or {}).get(k) for k in ("rope_theta", "partial_rotary_factor"))
        if theta is not None:
            if rope_base is not None and float(rope_base) != float(theta):
                raise ValueError(f"rope_base is {rope_base}, scaling holds a rope_theta of {theta}")
            rope_base = float(theta)
        if part is not None:
            turned = int(head_dim * float(part))
            if rotary_dim is not None and int(rotary_dim) != turned:
                raise ValueError(f"rotary_dim is {rotary_dim}, scaling holds a partial_rotary_factor "
                                 f"of {part}")
            rotary_dim = turned
        rope_base = 10000.0 if rope_base is None else rope_base
        n = head_dim if rotary_dim is None else int(rotary_dim)
        if n < 2 or n % 2 or n > head_dim:
            raise ValueError("rotary_dim must be even, between 2 and head_dim")
        if not rope_base >= 1.0:
            raise ValueError("rope_base must be at least 1")
        f, factor = _base_frequencies(rope_base, n), 1.0
        kind = "default"
        if scaling:
            kind = scaling.get("rope_type")
            kind = scaling.get("type") if kind is None else kind
        if kind == "linear":
            by = _number(scaling, "factor")
            if not by >= 1:
                raise ValueError("linear scaling needs factor >= 1")
            f = f / by
        elif kind == "llama3":
            f = _by_wavelength(f, scaling)
        elif kind == "yarn":
            f, factor = _by_rotations(f, float(rope_base), scaling)
        elif kind != "default":
            raise ValueError(f"unknown rope scaling {kind!r}; the frequencies can be given directly")
        return cls(f, head_dim, layout, factor)

    @property
    def inv_freq(self) -> torch.Tensor:
        """A copy of the frequencies (fp32, on the host)."""
        return self._inv_freq.clone()

    @property
    def head_dim(self) -> int:
        return self._head_dim

    @property
    def rotary_dim(self) -> int:
        return 2 * self._inv_freq.shape[0]

    @property
    def layout(self) -> str:
        return self._layout

    @property
    def factor(self) -> float:
        return self._factor

    def _table(self, dev: torch.device, head_dim: int) -> torch.Tensor:
        """The frequencies on a device, for rows of head_dim."""
        if head_dim != self._head_dim:
            raise ValueError(f"the rotary embedding is for head_dim {self._head_dim}, not {head_dim}")
        table = self._tables.get(dev)
        if table is None:
            if dev.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("a rotary embedding's first call on a device cannot be captured "
                                   "into a graph: make one call before")
            # (waits: any stream may use it; of two threads' first calls one's copy is kept, for both)
            table = self._tables.setdefault(dev, self._inv_freq.to(dev))
        return table


def apply_rotary(
    query: torch.Tensor,
    positions: torch.Tensor,
    rotary: RotaryEmbedding,
    key: torch.Tensor | None = None,
    query_out: torch.Tensor | None = None,
    key_out: torch.Tensor | None = None,
):
    """Q (and K) rows of new tokens turned by their positions, in one launch.

    query: [T, num_q_heads, head_dim]; key: [T, num_kv_heads, head_dim] of the same type (bf16, fp16
    or fp32), any strides (views of a fused projection's output, for instance); positions: [T]
    int32, any sign. Results go to ``query_out`` / ``key_out`` (new tensors by default), which may be
    the inputs themselves and must not overlap them otherwise; rows of an output that share elements
    are refused. Returns query_out, or (query_out,
    key_out) with a key. No backward pass: as in :mod:`semblend_amd.paged_cache`, a new result of an
    input that requires a gradient raises when its gradient is asked for.
    8192 tokens of 32 / 8 heads x 128 in bf16: 168 MB in 27 us; 32 tokens of 28 / 4 heads
    7.5. Extension with no reference counterpart.
    """
    dev = _device(query, (key, query_out, key_out))
    shape, dtype = query.shape, query.dtype
    if len(shape) != 3:
        raise ValueError("query must be [tokens, num_q_heads, head_dim]")
    if not isinstance(rotary, RotaryEmbedding):
        raise TypeError("rotary must be a RotaryEmbedding")
    num, heads, d = shape
    table = rotary._table(dev, d)
    dt = _lib.dtype_code(query)
    q, qst = _rows(query)
    new_q, new_k = query_out is None, key is not None and key_out is None
    if new_q:
        query_out, qost = _like(q, qst)
    else:
        qost = query_out.stride()
        if query_out.shape != shape or query_out.dtype != dtype or qost[2] != 1:
            raise ValueError("query_out must be like query, with a unit last stride")
    k = kst = kost = None
    kv = 0
    if key is not None:
        kshape = key.shape
        if len(kshape) != 3 or kshape[0] != num or kshape[2] != d:
            raise ValueError("key must be [tokens, num_kv_heads, head_dim]")
        if key.dtype != dtype:
            raise TypeError("query and key must share a dtype")
        kv = kshape[1]
        k, kst = _rows(key)
        if key_out is None:
            key_out, kost = _like(k, kst)
        else:
            kost = key_out.stride()
            if key_out.shape != kshape or key_out.dtype != dtype or kost[2] != 1:
                raise ValueError("key_out must be like key, with a unit last stride")
    elif key_out is not None:
        raise ValueError("key_out goes with key")
    pos = _index(positions, dev)
    if pos.shape[0] != num:
        raise ValueError("positions must have one entry per token")
    if num:
        _lib.launch(dev, "sb_apply_rotary", query_out.data_ptr(), q.data_ptr(),
                    None if k is None else key_out.data_ptr(), _lib.ptr(k), pos.data_ptr(),
                    table.data_ptr(), num, heads, kv, d, qst, qost, kst, kost,
                    rotary._inv_freq.shape[0], rotary._code, rotary._factor, dt)
    if new_q and query.requires_grad:
        query_out = _recorded("apply_rotary", query_out, query)
    if key is None:
        return query_out
    if new_k and key.requires_grad:
        key_out = _recorded("apply_rotary", key_out, key)
    return query_out, key_out
