"""A serving batch's operators over the paged K/V caches of this path: new tokens appended, their
attention (single tokens, prompt chunks, sliding window with first tokens that stay visible), and
4-bit pages.

The reference reuses donor K/V for a prefill and leaves the decode steps behind it to its host
engine (synapse_kv_connector/model_runner_hook.py:519-585 walks one request's layers); these are
extensions with no reference counterpart, on the same caches, block tables and positions as
``triton_kernels`` and ``rope_correction``:

* :func:`append_kv_paged` — K and V of new tokens into their slots, K (and Q) rotated on the way;
* :func:`paged_attention` — attention of a batch's rows over their pages;
* :class:`QuantizedKVCache` — pages of MXFP4 (blocks of 32 4-bit values that share a power of
  two), a cache of either function at 0.27 of the bytes of a 16-bit one;
* :func:`gather_kv_paged` — a request's rows read back as a donor buffer
  (``scatter_donor_kv_paged`` and ``rope_correct_scatter_paged`` take it; ``append_kv_paged`` with
  ``rotations`` appends it to 4-bit pages).

Batches: ``row_starts`` [num_requests + 1] (int32, on the device) says where each request's rows
begin; without it row i is request i's only one, as in a decode step, or, with one request, all
rows are that one's. Rows of no request and rows with a negative position are padding and left as
they are. A decode step of one row per request is best given without ``row_starts``: attention
then deals the keys of all requests out evenly (64 rows, one over 32768 keys and the others over
300, 32 / 8 heads x 128: 48 us, with ``row_starts`` 453). All metadata is read on the device, so a
step can be captured into a HIP graph once and replayed with new positions.

These are a server's calls and have no backward pass: a result that torch would differentiate
through (an input requires a gradient, in grad mode) raises when its gradient is asked for. Rows
written into a cache, ``out`` or ``query_out`` leave no record there.
"""

from __future__ import annotations

import functools
import math

import torch

from . import _lib
from .rope_correction import inv_freq_table

__all__ = ["QuantizedKVCache", "append_kv_paged", "gather_kv_paged", "paged_attention"]


@functools.lru_cache(maxsize=1024)
def _workspace_bytes(*sizes: int) -> int:
    return _lib.size_query("sb_paged_attention_workspace_size", *sizes)


class QuantizedKVCache:
    """Paged K/V in MXFP4: ``codes`` [num_blocks, 2, num_kv_heads, block_size, head_dim / 2] uint8
    (value 2i in the low half of byte i: sign, two exponent bits, one mantissa bit) and ``scales``
    [num_blocks, 2, num_kv_heads, block_size, head_dim / 32] uint8 (e + 127: the 32 values are 2^e
    times the 4-bit ones; 255: NaN). Any strides with unit last ones."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
            raise TypeError("codes and scales must be uint8")
        if codes.dim() != 5 or codes.shape[1] != 2 or codes.shape[4] % 16:
            raise ValueError("codes must be [num_blocks, 2, num_kv_heads, block_size, head_dim / 2] "
                             "with a head_dim that is a multiple of 32")
        if scales.shape != (*codes.shape[:4], codes.shape[4] // 16):
            raise ValueError("scales must be [num_blocks, 2, num_kv_heads, block_size, "
                             "head_dim / 32]")
        if codes.stride(4) != 1 or scales.stride(4) != 1:
            raise ValueError("codes and scales need unit last strides")
        if codes.device != scales.device:
            raise RuntimeError("codes and scales on different devices")
        self._codes, self._scales = codes, scales
        nb, _, heads, bs, half = codes.shape
        self.shape = (nb, 2, heads, bs, 2 * half)
        self.device = codes.device

    @property
    def codes(self) -> torch.Tensor:
        return self._codes

    @property
    def scales(self) -> torch.Tensor:
        return self._scales

    @classmethod
    def allocate(cls, num_blocks: int, num_kv_heads: int, block_size: int, head_dim: int,
                 device) -> "QuantizedKVCache":
        """An empty cache (every value 0)."""
        if head_dim % 32:
            raise ValueError("head_dim must be a multiple of 32")
        shape = (num_blocks, 2, num_kv_heads, block_size)
        return cls(torch.zeros((*shape, head_dim // 2), dtype=torch.uint8, device=device),
                   torch.zeros((*shape, head_dim // 32), dtype=torch.uint8, device=device))


# A call's checks cost as much host time as its launch, so the usual cases come first below and a
# tensor's shape and strides are read once.
def _device(first: torch.Tensor, rest) -> torch.device:
    """``_lib.require_device`` of all of them, by their device numbers."""
    index = first.get_device()
    if index < 0:
        return _lib.require_device(first, *rest)
    for t in rest:
        if t is not None and t.get_device() != index:
            return _lib.require_device(first, *rest)
    return first.device


def _cache_args(kv_cache, dtype: torch.dtype, *rows):
    """(device, shape, base, scale base, strides, scale strides, dtype code) of either cache; the
    ``rows`` tensors must be on its device."""
    if isinstance(kv_cache, QuantizedKVCache):
        codes, scales = kv_cache._codes, kv_cache._scales
        return (_device(codes, rows), kv_cache.shape, codes.data_ptr(),
                scales.data_ptr(), codes.stride(), scales.stride(),
                _lib.SB_DTYPE_MXFP4)
    dev = _device(kv_cache, rows)
    shape, strides = kv_cache.shape, kv_cache.stride()
    if len(shape) != 5 or shape[1] != 2:
        raise ValueError("kv_cache must be [num_blocks, 2, num_kv_heads, block_size, head_dim]")
    if kv_cache.dtype != dtype:
        raise TypeError("the rows and kv_cache must share a dtype (or kv_cache be a "
                        "QuantizedKVCache)")
    if strides[4] != 1:
        raise ValueError("kv_cache needs a unit last stride")
    return (dev, shape, kv_cache.data_ptr(), None, strides, None,
            _lib.dtype_code(kv_cache))


def _index(t, dev) -> torch.Tensor:
    """``_lib.as_index`` with the usual case (already a device index array) first."""
    if type(t) is torch.Tensor and t.dtype is torch.int32 and t.get_device() == dev.index \
            and t.dim() == 1 and t.is_contiguous():
        return t
    return _lib.as_index(t, dev)


def _batch_args(dev, num_rows: int, block_tables, positions, row_starts):
    """(tables, positions, row_starts, number of requests, entries of a table) checked and on the
    device. A 1-D table is one request's, and all rows are that request's."""
    bt = block_tables
    if not isinstance(bt, torch.Tensor):
        bt = torch.as_tensor(bt, dtype=torch.int32)
    if bt.dim() == 1:
        if row_starts is not None:
            raise ValueError("row_starts goes with block_tables [num_requests, max_blocks]")
        bt = _index(bt, dev).unsqueeze(0)
    elif bt.dim() != 2:
        raise ValueError("block_tables must be [num_requests, max_blocks], or [max_blocks] for "
                         "one request")
    elif bt.dtype is not torch.int32 or bt.get_device() != dev.index or (
            bt.stride(1) != 1 and bt.shape[1] > 1):
        shape = bt.shape
        bt = _index(bt.reshape(-1), dev).view(shape)
    pos = _index(positions, dev)
    if pos.shape[0] != num_rows:
        raise ValueError("positions must have one entry per row")
    requests, width = bt.shape
    if row_starts is not None:
        row_starts = _index(row_starts, dev)
        if row_starts.shape[0] != requests + 1:
            raise ValueError("row_starts must have num_requests + 1 entries")
    elif num_rows > requests != 1:
        raise ValueError("without row_starts there is one row per request: "
                         f"{num_rows} rows, {requests} block tables")
    if width == 0 or requests == 0:
        raise ValueError("block_tables is empty")
    return bt, pos, row_starts, requests, width


def _rows(t: torch.Tensor):
    """(t, its strides), copied where its last dimension is not contiguous."""
    st = t.stride()
    if st[2] != 1:
        t = t.contiguous()
        st = t.stride()
    return t, st


def _like(t: torch.Tensor, strides):
    """(a new dense tensor of t's shape and dtype, its strides)."""
    if t.is_contiguous():
        return torch.empty_like(t), strides
    new = torch.empty(t.shape, dtype=t.dtype, device=t.device)
    return new, new.stride()


class _NoBackward(torch.autograd.Function):
    """``out`` as a function of ``inputs`` that cannot be differentiated."""

    @staticmethod
    def forward(ctx, name, out, *inputs):
        ctx.name = name
        ctx.mark_dirty(out)
        return out

    @staticmethod
    def backward(ctx, *grads):
        raise RuntimeError(f"{ctx.name} has no backward pass; call it under torch.no_grad(), or on "
                           "detached tensors")


def _recorded(name: str, out: torch.Tensor, *inputs: torch.Tensor) -> torch.Tensor:
    """A new result, so that a gradient of it raises instead of missing these inputs."""
    return _NoBackward.apply(name, out, *inputs) if torch.is_grad_enabled() else out


def append_kv_paged(
    kv_cache,
    key: torch.Tensor,
    value: torch.Tensor,
    block_tables: torch.Tensor,
    positions: torch.Tensor,
    row_starts: torch.Tensor | None = None,
    rope_base: float | None = None,
    rotations: torch.Tensor | None = None,
    query: torch.Tensor | None = None,
    query_out: torch.Tensor | None = None,
    rotary=None,
) -> torch.Tensor | None:
    """K and V of new tokens into the cache slots of their positions, in one launch.

    kv_cache: [num_blocks, 2, num_kv_heads, block_size, head_dim] of the keys' dtype, or a
    :class:`QuantizedKVCache`; key / value: [T, num_kv_heads, head_dim] (bf16, fp16 or fp32, any
    strides); block_tables: [num_requests, max_blocks], or [max_blocks] for one request;
    positions: [T], each token's position in its request; row_starts: see the module.
    With ``rope_base`` (at least 1), K is rotated by its position with the interleaved RoPE of
    this path before its one rounding, and so is ``query`` [T, num_q_heads, head_dim], which goes
    to ``query_out`` (a new tensor by default; returned; rows that share elements are refused). The
    angle is position * inv_freq with the path's fp32 frequencies, the product and its sine and
    cosine in 64 bits.
    ``rotations``: [T], the positions to rotate by instead (a donor's K, rotated already at d and
    appended at t: t - d).
    ``rotary``: a :class:`semblend_amd.rotary.RotaryEmbedding` instead of ``rope_base``: half pairs,
    part of the head, scaled frequencies, its factor on cosine and sine (not with ``rotations``: that
    K holds it already; a query then needs a factor of 1). 4-bit pages take embeddings whose turned
    elements (half layout: either half of them, and of the others) are whole blocks of 32.
    Tokens whose position has no page are not appended (their query is rotated still); padding
    rows are left out altogether. Two tokens with one slot race: slots must be distinct.
    Extension with no reference counterpart (``partial_prefill`` writes its new K/V into
    contiguous caches, semblend_core/triton_kernels.py:904-909).
    """
    dtype = key.dtype
    dev, shape, base, sbase, st, sst, code = _cache_args(kv_cache, dtype, key, value, query,
                                                         query_out)
    _, _, heads, bs, d = shape
    if value.dtype != dtype or (query is not None and query.dtype != dtype):
        raise TypeError("key, value and query must share a dtype")
    kshape = key.shape
    if len(kshape) != 3 or kshape[1] != heads or kshape[2] != d or value.shape != kshape:
        raise ValueError("key and value must be [tokens, num_kv_heads, head_dim] with the "
                         "cache's heads and head_dim")
    num = kshape[0]
    k, kst = _rows(key)
    v, vst = _rows(value)
    dt = _lib.dtype_code(key)
    if rotary is not None:
        if rope_base is not None:
            raise ValueError("rope_base and rotary are alternatives")
        if rotations is not None and query is not None and rotary.factor != 1.0:
            raise ValueError("with rotations the factor of rotary applies to no row: a query needs "
                             "a factor of 1")
    elif rope_base is None and (rotations is not None or query is not None):
        raise ValueError("rotations and query go with rope_base or rotary")
    if rope_base is not None and not rope_base >= 1.0:
        raise ValueError("rope_base must be at least 1")
    if d % 2:
        raise ValueError("head_dim must be even")
    q, qst, ost, hq = None, None, None, 0
    new = query is not None and query_out is None
    if query is not None:
        qshape = query.shape
        if len(qshape) != 3 or qshape[0] != num or qshape[2] != d:
            raise ValueError("query must be [tokens, num_q_heads, head_dim]")
        hq = qshape[1]
        q, qst = _rows(query)
        if query_out is None:
            query_out, ost = _like(q, qst)
        else:
            ost = query_out.stride()
            if query_out.shape != qshape or query_out.dtype != dtype or ost[2] != 1:
                raise ValueError("query_out must be like query, with a unit last stride")
    elif query_out is not None:
        raise ValueError("query_out goes with query")
    if num == 0:
        return query_out
    bt, pos, starts, requests, width = _batch_args(dev, num, block_tables, positions, row_starts)
    rot = None
    if rotations is not None:
        rot = _index(rotations, dev)
        if rot.shape[0] != num:
            raise ValueError("rotations must have one entry per token")
    qp, qop = (None, None) if q is None else (q.data_ptr(), query_out.data_ptr())
    if rotary is None:
        inv = inv_freq_table(rope_base, d, dev) if rope_base is not None else None
        _lib.launch(
            dev, "sb_append_kv_paged",
            base, sbase, k.data_ptr(), v.data_ptr(), qp, qop, bt.data_ptr(), bt.stride(0),
            pos.data_ptr(), _lib.ptr(rot), _lib.ptr(starts), _lib.ptr(inv), num, requests, heads, hq, d,
            bs, shape[0], width, kst, vst, qst, ost, st, sst, dt, code)
    else:
        inv = rotary._table(dev, d)
        _lib.launch(
            dev, "sb_append_kv_rotary_paged",
            base, sbase, k.data_ptr(), v.data_ptr(), qp, qop, bt.data_ptr(), bt.stride(0),
            pos.data_ptr(), _lib.ptr(rot), _lib.ptr(starts), inv.data_ptr(), num, requests, heads, hq, d,
            bs, shape[0], width, kst, vst, qst, ost, st, sst, inv.shape[0], rotary._code,
            1.0 if rot is not None else rotary._factor, dt, code)
    if new and query.requires_grad:
        return _recorded("append_kv_paged", query_out, query)
    return query_out


def gather_kv_paged(
    kv_cache,
    block_table: torch.Tensor,
    positions: torch.Tensor | None = None,
    num_rows: int | None = None,
    dtype: torch.dtype | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """A request's cache rows as a contiguous donor buffer [2, num_kv_heads, N, head_dim].

    Row i is position ``positions[i]``, or position i of the first ``num_rows`` (default: all the
    table names). dtype: the cache's own; for a :class:`QuantizedKVCache` bf16 (the default) and
    fp32, which hold its values exactly, or fp16, rounded once. Positions without a page give
    zeros. Extension with no reference counterpart (the reference's connectors copy donor rows
    out of the cache with torch indexing, synapse_kv_connector/model_runner_hook.py:215-276).
    """
    quant = isinstance(kv_cache, QuantizedKVCache)
    if dtype is None:
        dtype = torch.bfloat16 if quant else kv_cache.dtype
    dev, shape, base, sbase, st, sst, code = _cache_args(kv_cache, dtype)
    _, _, heads, bs, d = shape
    bt = _index(block_table, dev)
    pos = None
    if positions is not None:
        pos = _index(positions, dev)
        if num_rows is not None and num_rows != pos.shape[0]:
            raise ValueError("num_rows and positions differ")
        num_rows = pos.shape[0]
    elif num_rows is None:
        num_rows = bt.shape[0] * bs
    if num_rows < 0:
        raise ValueError("num_rows must not be negative")
    if out is None:
        out = torch.empty((2, heads, num_rows, d), dtype=dtype, device=dev)
    elif (out.shape != (2, heads, num_rows, d) or out.dtype != dtype or out.device != dev
          or out.stride(3) != 1):
        raise ValueError("out must be [2, num_kv_heads, rows, head_dim] of dtype on the cache's "
                         "device, with a unit last stride")
    dt = _lib.dtype_code(out)
    if num_rows == 0:
        return out
    if bt.shape[0] == 0:
        return out.zero_()
    _lib.launch(dev, "sb_gather_kv_paged", out.data_ptr(), base, sbase, bt.data_ptr(),
                _lib.ptr(pos), num_rows, heads, d, bs, shape[0], bt.shape[0],
                out.stride(), st, sst, dt, code)
    return out


def paged_attention(
    query: torch.Tensor,
    kv_cache,
    block_tables: torch.Tensor,
    positions: torch.Tensor,
    row_starts: torch.Tensor | None = None,
    max_rows: int | None = None,
    window: int | None = None,
    sinks: int = 0,
    scale: float | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """GQA attention of a batch's rows over their paged caches.

    query: [R, num_q_heads, head_dim] (bf16, fp16 or fp32), row r the token at ``positions[r]`` of
    its request; kv_cache: [num_blocks, 2, num_kv_heads, block_size, head_dim] of the query's
    dtype (any strides), or a :class:`QuantizedKVCache`; block_tables: [num_requests,
    max_blocks], or [max_blocks] for one request; row_starts: see the module. Query head h reads
    KV head ``h // (num_q_heads // num_kv_heads)``; ``scale`` is 1 / sqrt(head_dim) by default.
    Row r sees the keys j <= positions[r]; with ``window``, only those with
    ``j > positions[r] - window`` or ``j < sinks``. Keys behind the block table, or in a page that
    is none of the pool's (-1 for instance), are not seen; pages between the sinks and the window
    are not read, and their entries may hold anything. What lies in keys that a row does not see
    (NaN included) does not reach it. A row that sees no key gets zeros.
    ``max_rows``: no request has more rows than this; it only helps to choose kernels (a decode
    step of several rows a request runs as one launch fewer, and a few dozen rows over at most a
    thousand keys are faster on the single-token kernel, which 1 asks for). Scores, sums and
    outputs are fp32, rounded once; 16-bit calls round the weights to their dtype for the product
    with V (fp16: a weight below 2^-25 of the row's largest may be zero there). fp16 queries take
    4-bit values below 2^18, as pages of fp16 tokens hold them: a page written from wider tokens may
    hold larger ones, which are infinite to such a query.
    Returns [R, num_q_heads, head_dim] (``out`` if given; padding rows of it are left as they
    are). Over one request's 16-bit or fp32 pages without a window
    ``triton_kernels.partial_prefill_attention_paged`` computes the same; this call takes ragged
    batches described on the device, that one splits a chunk over a few thousand keys better (28 / 4
    heads x 128, this call against that one: 1 row of 4096 keys 14 and 18 us, 40 of 4096 32 and 27,
    614 of 4096 52 and 41, 2458 of 16384 317 and 312; fp32, 32 / 8 heads, 500 of 4096 187 and 245).
    Extension with no reference counterpart: the reference's attention is MHA over contiguous K/V
    (semblend_core/triton_kernels.py:655-734), without window.
    """
    qshape, dtype = query.shape, query.dtype
    if len(qshape) != 3:
        raise ValueError("query must be [rows, num_q_heads, head_dim]")
    dev, shape, base, sbase, st, sst, code = _cache_args(kv_cache, dtype, query, out)
    num, hq, d = qshape
    nb, _, heads, bs, hd = shape
    if hd != d:
        raise ValueError("query and kv_cache head_dim differ")
    if hq % heads:
        raise ValueError("num_q_heads must be a multiple of num_kv_heads")
    if window is not None and window < 1:
        raise ValueError("window must be at least 1 (None: no window)")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    q, qst = _rows(query)
    if scale is None:
        scale = 1.0 / math.sqrt(d)
    new = out is None
    if new:
        out, ost = _like(q, qst)
    else:
        ost = out.stride()
        if out.shape != qshape or out.dtype != dtype or ost[2] != 1:
            raise ValueError("out must be like query, with a unit last stride")
    dt = _lib.dtype_code(q)
    if num == 0:
        return out
    bt, pos, starts, requests, width = _batch_args(dev, num, block_tables, positions, row_starts)
    most = num if max_rows is None else min(max(1, int(max_rows)), num)
    win = 0 if window is None or window > 0x7fffffff else int(window)
    sinks = min(int(sinks), 0x7fffffff)
    ws_bytes = _workspace_bytes(num, requests, int(starts is not None), most, hq, heads, d, bs,
                                width, win, sinks, dt, code)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
    _lib.launch(
        dev, "sb_paged_attention",
        out.data_ptr(), q.data_ptr(), base, sbase, bt.data_ptr(), bt.stride(0), pos.data_ptr(),
        _lib.ptr(starts), _lib.ptr(ws), ws_bytes, num, requests, most, hq, heads, d, bs, nb,
        width, win, sinks, float(scale), qst, ost, st, sst, dt, code)
    if new and (query.requires_grad or sbase is None and kv_cache.requires_grad):
        return _recorded("paged_attention", out, query, *(() if sbase else (kv_cache,)))
    return out
