"""A model as it is published, over this path: 4-bit weights, half pairs, scaled frequencies. Its layers'
steps run together as a server runs them (a partial prefill over a donor's corrected K/V, then decode
steps), each stage against 64 bits of the stage's own inputs."""

from __future__ import annotations

import pytest
import torch

from semblend_amd import paged_cache as pc
from semblend_amd import rope_correction as rc
from semblend_amd import triton_kernels as tk
from semblend_amd.batch import KVReuseBatch, ReuseRequest
from semblend_amd.quantized import QuantizedLinear, quantized_linear
from semblend_amd.rotary import RotaryEmbedding, apply_rotary

from . import paged_reference as pref
from . import quantized_reference as qref
from . import rotary_reference as rref
from .helpers import assert_bit_exact, gen, randn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SCALED = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}


def _weight(n, k, group, dtype, seed, zeros=True):
    codes, scales, z = qref.make(n, k, group, dtype, seed, zeros)
    scales = (scales.float() / k ** 0.5 * 4).to(dtype)
    return (codes, scales, z), QuantizedLinear(codes.cuda(), scales.cuda(), None if z is None else z.cuda())


def _table(n, bs, seed, spare=4):
    need = -(-n // bs)
    return torch.randperm(need + spare, generator=gen(seed))[:need].to(torch.int32), need + spare


def _check_layer(x, pos, wq, wo, bias, rot, rope_base, res, cache, before, table, hq, hkv, d):
    """Every stage of a layer's result against 64 bits of what went into it."""
    bs = cache.shape[3]
    inside = (pos >= 0) & (pos < x.shape[0])
    rows = x[pos.long().clamp(0, x.shape[0] - 1)]
    y, bound = qref.linear(rows, *wq, bias)
    y = y.view(-1, hq + 2 * hkv, d)
    bound = bound.view_as(y)
    freq, layout = (rot.inv_freq, rot.layout) if rot else (
        rc.inv_freq_table(rope_base, d, torch.device("cpu")), "interleaved")
    factor = rot.factor if rot else 1.0
    want, norm = rref.turn(y, pos, freq, layout, factor)
    spread, _ = rref.turn(bound, pos * 0, freq, layout)          # (norm of the pair's two bounds)
    a, b = rref.pairs_of(2 * freq.shape[0], layout)
    both = torch.sqrt(spread[..., a] ** 2 + spread[..., b] ** 2) * factor
    spread[..., a] = spread[..., b] = both
    u = pref.half_step(x.dtype)
    tol = spread * (1 + u) + u * want.abs() + 2.0 ** -22 * norm * (1 + u) + 1e-30
    q = res.query.cpu().double()
    assert ((q - want[:, :hq]).abs() <= tol[:, :hq])[inside].all()
    assert (q[~inside] == 0).all()
    got = cache.cpu()
    left = torch.ones(got.shape[0], got.shape[3], dtype=torch.bool)
    for i in range(len(pos)):
        p = int(pos[i])
        if not inside[i]:
            continue
        page, slot = int(table[p // bs]), p % bs
        left[page, slot] = False
        k, v = got[page, 0, :, slot].double(), got[page, 1, :, slot].double()
        assert ((k - want[i, hq:hq + hkv]).abs() <= tol[i, hq:hq + hkv]).all()
        assert ((v - y[i, hq + hkv:]).abs() <= bound[i, hq + hkv:]).all()
    left = left[:, None, None, :].expand(got.shape[:4])
    assert_bit_exact(got[left], before[left])
    at = inside.nonzero().flatten()
    out, mass, serr = pref.attention(res.query.cpu()[at], got.double(), table[None], pos[at], [0, len(at)],
                                     None, 0, d ** -0.5)
    err = (res.attention.cpu()[at].double() - out).abs()
    assert (err <= pref.attention_bound(out, mass, serr, x.dtype, int(pos.max()) + 1)).all()
    if wo is not None:
        qref.check(res.output.cpu(), *qref.linear(res.attention.cpu().flatten(1), *wo))


@pytest.mark.parametrize("dtype,layout,scaling,rope_base", [
    (BF16, "half", SCALED, None), (FP16, "half", None, None), (BF16, "interleaved", None, None),
    (BF16, None, None, 1e6)])
@pytest.mark.parametrize("rows", [1, 40, 300])
def test_layer_of_partial_prefill(dev, dtype, layout, scaling, rope_base, rows):
    """A donor's rows scattered into the layer's pages, the others recomputed by the layer with 4-bit
    projections; rows outside the hidden states give zero queries and write nothing."""
    hq, hkv, d, hidden, bs, seq = 6, 2, 64, 384, 16, 700
    wq, qw = _weight((hq + 2 * hkv) * d, hidden, 64, dtype, 1)
    wo, ow = _weight(hidden, hq * d, 128, dtype, 2, zeros=False)
    bias = randn(((hq + 2 * hkv) * d,), dtype, 3)
    rot = layout and RotaryEmbedding.from_config(d, 5e5, layout=layout, scaling=scaling)
    x = randn((seq, hidden), dtype, 4)
    table, nb = _table(seq + 64, bs, 5)
    cache = randn((nb, 2, hkv, bs, d), dtype, 6).cuda()
    pos = torch.randperm(seq, generator=gen(7))[:rows].sort().values.to(torch.int32)
    if rows > 1:
        pos[-1] = seq + 30                        # in the table, not among the hidden states
    if rot:
        donor = randn((2, hkv, 800, d), dtype, 8).cuda()
        reused = torch.ones(seq, dtype=torch.bool)
        reused[pos[pos < seq].long()] = False
        t = reused.nonzero().flatten().to(torch.int32).cuda()
        rc.rope_correct_scatter_paged_layers([cache], [donor], table.cuda(), t + 37, t, rotary=rot)
    before = cache.cpu().clone()
    res = tk.partial_prefill_layer_paged(x.cuda(), qw, ow, pos.cuda(), cache, table.cuda(), hq, hkv, d,
                                         qkv_bias=bias.cuda(), rope_base=rope_base, rotary=rot)
    if rows > 1:  # (the row outside attends with a zero query; what it gives is not looked at)
        keep = torch.arange(rows) < rows - 1
        qref.check(res.output.cpu()[keep], *(v[keep] for v in qref.linear(
            res.attention.cpu().flatten(1), *wo)))
        _check_layer(x, pos, wq, None, bias, rot, rope_base, res, cache, before, table, hq, hkv, d)
    else:
        _check_layer(x, pos, wq, wo, bias, rot, rope_base, res, cache, before, table, hq, hkv, d)


def test_projection_without_rotation_and_of_plain_weights(dev):
    """A quantized projection without rotation, and a 16-bit one with half pairs: the same K/V and Q as
    the product (the library's) and the append give."""
    hq, hkv, d, hidden, bs, seq = 4, 2, 64, 256, 16, 100
    _, qw = _weight((hq + 2 * hkv) * d, hidden, 32, BF16, 1)
    x = randn((seq, hidden), BF16, 2).cuda()
    table, nb = _table(seq, bs, 3)
    pos = torch.arange(0, seq, 3, dtype=torch.int32).cuda()
    a, b = (torch.zeros((nb, 2, hkv, bs, d), dtype=BF16, device="cuda") for _ in range(2))
    out = torch.full((pos.shape[0], hq, d), 7.0, dtype=BF16, device="cuda")
    q = tk.qkv_projection_paged(x, qw, pos, a, table.cuda(), hq, hkv, d, out=out)
    assert q is out
    y = quantized_linear(x[pos.long()], qw).view(-1, hq + 2 * hkv, d)
    pc.append_kv_paged(b, y[:, hq:hq + hkv], y[:, hq + hkv:], table.cuda(), pos)
    assert_bit_exact(q.cpu(), y[:, :hq].contiguous().cpu())
    assert_bit_exact(a.cpu(), b.cpu())
    rot = RotaryEmbedding.from_config(d, 1e4, rotary_dim=32)
    w = qw.dequantize(BF16)
    a.zero_(), b.zero_()
    q = tk.qkv_projection_paged(x, w, pos, a, table.cuda(), hq, hkv, d, rotary=rot)
    y = torch.nn.functional.linear(x[pos.long()], w).view(-1, hq + 2 * hkv, d)
    got = pc.append_kv_paged(b, y[:, hq:hq + hkv], y[:, hq + hkv:], table.cuda(), pos, rotary=rot,
                             query=y[:, :hq])
    assert_bit_exact(q.cpu(), got.cpu())
    assert_bit_exact(a.cpu(), b.cpu())
    with pytest.raises(ValueError, match="auto"):
        tk.qkv_projection_paged(x, qw, pos, a, table.cuda(), hq, hkv, d, backend="fused")
    with pytest.raises(ValueError, match="alternatives"):
        tk.qkv_projection_paged(x, qw, pos, a, table.cuda(), hq, hkv, d, rotary=rot, rope_base=1e4)
    with pytest.raises(ValueError, match="qkv_weight"):
        tk.qkv_projection_paged(x, qw, pos, a, table.cuda(), hq, hkv + 1, d)
    empty = tk.qkv_projection_paged(x, qw, pos[:0], a, table.cuda(), hq, hkv, d, rotary=rot)
    assert empty.shape == (0, hq, d)


@pytest.mark.parametrize("quant", [False, True])
def test_decode_steps_captured(dev, quant):
    """Decode steps of a ragged batch captured once and replayed token after token: projection, append
    with rotation, attention over 16-bit or 4-bit pages, output projection. Every replay equals the
    eager step, and its stages are within their bounds of 64 bits."""
    hq, hkv, d, hidden, bs, requests = 6, 2, 64, 384, 16, 5
    lens = [3, 200, 64, 17, 90]
    wq, qw = _weight((hq + 2 * hkv) * d, hidden, 128, BF16, 1)
    wo, ow = _weight(hidden, hq * d, 64, BF16, 2)
    bias = randn(((hq + 2 * hkv) * d,), BF16, 3)
    bias_d = bias.cuda()
    rot = RotaryEmbedding.from_config(d, 1e6, scaling=SCALED)
    width = -(-(max(lens) + 8) // bs)
    pages = torch.randperm(requests * width, generator=gen(4)).to(torch.int32).view(requests, width)
    tables = pages.cuda()

    def fresh():
        if quant:
            c = pc.QuantizedKVCache.allocate(requests * width, hkv, bs, d, "cuda")
        else:
            c = torch.zeros((requests * width, 2, hkv, bs, d), dtype=BF16, device="cuda")
        starts = torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()
        at = torch.cat([torch.arange(n) for n in lens]).to(torch.int32).cuda()
        kv = randn((sum(lens), 2 * hkv, d), BF16, 5).cuda()
        pc.append_kv_paged(c, kv[:, :hkv], kv[:, hkv:], tables, at, starts, rotary=rot)
        return c

    x = torch.zeros((requests, hidden), dtype=BF16, device="cuda")
    pos = torch.tensor(lens, dtype=torch.int32).cuda()
    cache, eager = fresh(), fresh()

    def step(c):
        y = quantized_linear(x, qw, bias=bias_d).view(requests, hq + 2 * hkv, d)
        q = pc.append_kv_paged(c, y[:, hq:hq + hkv], y[:, hq + hkv:], tables, pos, rotary=rot,
                               query=y[:, :hq])
        o = pc.paged_attention(q, c, tables, pos)
        return y, q, o, quantized_linear(o.flatten(1), ow)

    step(fresh())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(cache)
    for token in range(4):
        x.copy_(randn((requests, hidden), BF16, 100 + token))
        want = step(eager)
        for t in outs:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert_bit_exact(a.cpu(), b.cpu())
        y, q, o, out = (t.cpu() for t in outs)
        qref.check(y.flatten(1), *qref.linear(x.cpu(), *wq, bias))
        rref.check(q, *rref.turn(y[:, :hq], pos.cpu(), rot.inv_freq, rot.layout))
        c64 = pref.dequantize(cache.codes.cpu(), cache.scales.cpu()) if quant else cache.cpu().double()
        k, norm = rref.turn(y[:, hq:hq + hkv], pos.cpu(), rot.inv_freq, rot.layout)
        for i in range(requests):
            p = int(pos[i])
            row = c64[int(pages[i, p // bs]), :, :, p % bs]
            if quant:
                assert torch.equal(row[0], pref.dequantize(*_packed(k[i])))
                assert torch.equal(row[1], pref.dequantize(*_packed(y[i, hq + hkv:].double())))
            else:
                rref.check(row[0][None].to(BF16), k[i:i + 1], norm[i:i + 1])
                assert_bit_exact(row[1].to(BF16), y[i, hq + hkv:])
        ref, mass, serr = pref.attention(q, c64, pages, pos.cpu(), None, None, 0, d ** -0.5)
        assert ((o.double() - ref).abs() <= pref.attention_bound(ref, mass, serr, BF16, 300)).all()
        qref.check(out, *qref.linear(o.flatten(1), *wo))
        pos += 1


def test_projection_captured(dev):
    """The projection in parts captured with positions and hidden states that change from replay to
    replay, rows outside the hidden states among them."""
    hq, hkv, d, hidden, bs, seq, rows = 4, 2, 64, 256, 16, 90, 37
    _, qw = _weight((hq + 2 * hkv) * d, hidden, 64, BF16, 1)
    rot = RotaryEmbedding.from_config(d, 1e4)
    table, nb = _table(seq + 40, bs, 2)
    bt = table.cuda()
    x = torch.zeros((seq, hidden), dtype=BF16, device="cuda")
    pos = torch.zeros(rows, dtype=torch.int32, device="cuda")
    a, b = (torch.zeros((nb, 2, hkv, bs, d), dtype=BF16, device="cuda") for _ in range(2))
    for kw in (dict(rotary=rot), dict(rope_base=1e4), {}):
        step = lambda c: tk.qkv_projection_paged(x, qw, pos, c, bt, hq, hkv, d, **kw)
        pos.copy_(torch.arange(rows))
        step(a.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step(a)
        for i in range(4):
            x.copy_(randn((seq, hidden), BF16, 10 + i))
            pos.copy_(torch.randperm(seq + 30, generator=gen(20 + i))[:rows])
            want = step(b)
            got.fill_(3.0)
            graph.replay()
            torch.cuda.synchronize()
            assert_bit_exact(got.cpu(), want.cpu())
            assert_bit_exact(a.cpu(), b.cpu())
            assert (got.cpu()[pos.cpu() >= seq] == 0).all()


def _packed(x):
    c, s = pref.quantize(x)
    return (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8), s


def test_reused_prompt_equals_a_computed_one(dev):
    """A text at other positions of a new prompt: its K appended there, and its donor's K brought there
    by the scatter, or loaded as it is and shifted, agree to the donor's own rounding, in every layer."""
    layers, hkv, d, bs, n, by = 3, 2, 128, 16, 200, 419
    rot = RotaryEmbedding.from_config(d, 1e6, scaling={"rope_type": "yarn", "factor": 4.0,
                                                       "original_max_position_embeddings": 32768})
    table, nb = _table(n + by, bs, 1)
    bt = table.cuda()
    here = torch.arange(n, dtype=torch.int32).cuda()
    keys = [randn((n, hkv, d), FP32, 10 + i).to(BF16) for i in range(layers)]
    vals = [randn((n, hkv, d), BF16, 20 + i).cuda() for i in range(layers)]
    empty = lambda: [torch.zeros((2, nb, bs, hkv, d), dtype=BF16, device="cuda") for _ in range(layers)]
    old, scattered, shifted = empty(), empty(), empty()
    std = lambda cs: [rc.standard_view(c, "vllm") for c in cs]
    for i in range(layers):
        pc.append_kv_paged(std(old)[i], keys[i].cuda(), vals[i], bt, here, rotary=rot)
    donors = [pc.gather_kv_paged(c, bt, here) for c in std(old)]
    rc.rope_correct_scatter_paged_layers(std(scattered), donors, bt, here, here + by, rotary=rot)
    for i in range(layers):
        pc.append_kv_paged(std(shifted)[i], donors[i][0].transpose(0, 1), donors[i][1].transpose(0, 1), bt,
                           here + by)
    rc.apply_rope_deltas_inplace_layers(shifted, bt, (here + by).tolist(), [by] * n, layout="vllm",
                                        rotary=rot)
    at = here.cpu().long() + by
    for i in range(layers):
        assert_bit_exact(scattered[i].cpu(), shifted[i].cpu())
        rows = scattered[i].cpu()[:, table.long()[at // bs], at % bs]
        want, norm = rref.turn(keys[i], here.cpu() + by, rot.inv_freq, "half", rot.factor)
        # the donor's rounding (each of a pair half a step), turned, and one more
        u = pref.half_step(BF16)
        assert ((rows[0].double() - want).abs() <= u * norm * 2 ** 0.5 + u * want.abs() * (1 + u)
                + 2.0 ** -20 * norm).all()
        assert_bit_exact(rows[1], vals[i].cpu())


def test_batch_with_a_rotary_embedding(dev):
    """KVReuseBatch with an embedding scatters as the per-request calls do, and without rotation as
    without it."""
    hkv, d, bs, layers = 2, 64, 16, 2
    rot = RotaryEmbedding.from_config(d, 1e4)
    tables, nb = _table(16 * 16, bs, 1, spare=0)
    caches = [randn((nb, 2, hkv, bs, d), BF16, 2 + i).cuda() for i in range(layers)]
    plain = [c.clone() for c in caches]
    one = [c.clone() for c in caches]
    reqs = []
    for r in range(2):
        t = torch.arange(0, 100, 2 + r, dtype=torch.int32).cuda()
        reqs.append(ReuseRequest(tables[r * 8:(r + 1) * 8].cuda(),
                                 [randn((2, hkv, 150, d), BF16, 50 + 10 * r + i).cuda()
                                  for i in range(layers)],
                                 (t + 31 * r).to(torch.int32), t,
                                 torch.arange(1, 4, dtype=torch.int32).cuda()))
    batch = KVReuseBatch(caches, reqs, rotary=rot)
    batch.scatter_rope()
    for q in reqs:
        rc.rope_correct_scatter_paged_layers(one, q.donor_kvs, q.block_table, q.donor_positions,
                                             q.target_positions, rotary=rot)
    for a, b in zip(caches, one):
        assert_bit_exact(a.cpu(), b.cpu())
    batch = KVReuseBatch(plain, reqs, rotary=rot)
    batch.scatter_rope(rope=False)
    t, s = reqs[1].target_positions.cpu().long(), reqs[1].donor_positions.cpu().long()
    page = tables[8:].long()[t // bs]
    assert_bit_exact(plain[0].cpu()[page, 0, :, t % bs], reqs[1].donor_kvs[0].cpu()[0, :, s].transpose(0, 1))
    assert not torch.equal(caches[0].cpu()[page, 0, :, t % bs], plain[0].cpu()[page, 0, :, t % bs])
