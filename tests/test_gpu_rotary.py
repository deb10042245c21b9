"""Rotary positions in either layout against 64 bits (tests/rotary_reference.py): rows of new tokens,
appends to pages of every format, donors scattered into pages, K shifted in place."""

from __future__ import annotations

import math

import pytest
import torch

from semblend_amd import paged_cache as pc
from semblend_amd import rope_correction as rc
from semblend_amd.rotary import RotaryEmbedding, apply_rotary

from . import paged_reference as pref
from . import rotary_reference as ref
from .helpers import assert_bit_exact, gen, randn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
SCALED = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 32768}


def _table(n, bs, seed, spare=3):
    need = -(-n // bs)
    return torch.randperm(need + spare, generator=gen(seed))[:need].to(torch.int32), need + spare


# (head_dim, turned elements): whole heads, parts, sizes that 16 bytes do not divide
SIZES = [(128, 128), (64, 64), (64, 32), (128, 64), (96, 96), (80, 32), (512, 512), (8, 4), (24, 20),
         (6, 4), (66, 64)]


@pytest.mark.parametrize("d,n", SIZES)
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_rows(dev, dtype, layout, d, n):
    """Any position (negative and far ones), a factor, one token to many heads."""
    rot = RotaryEmbedding.from_config(d, 5e5, rotary_dim=n, layout=layout, scaling=YARN)
    pos = torch.tensor([0, 1, -1, 31, 131071, -70000, 2 ** 31 - 1, -2 ** 31, 5, 77, 4095],
                       dtype=torch.int64).to(torch.int32)
    q, k = randn((11, 5, d), dtype, 1), randn((11, 2, d), dtype, 2)
    got_q, got_k = apply_rotary(q.cuda(), pos.cuda(), rot, key=k.cuda())
    for got, x in ((got_q, q), (got_k, k)):
        want, norm = ref.turn(x, pos, rot.inv_freq, layout, rot.factor)
        ref.check(got.cpu(), want, norm)
    assert_bit_exact(apply_rotary(q.cuda(), pos.cuda(), rot).cpu(), got_q.cpu())


@pytest.mark.parametrize("num,hq,hk", [(1, 1, 1), (1, 28, 4), (31, 32, 8), (700, 28, 4), (2600, 32, 8),
                                       (9001, 3, 1), (3, 300, 17)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rows_of_every_launch_shape(dev, layout, num, hq, hk):
    """From one token to thousands: the rows a workgroup takes change with both."""
    rot = RotaryEmbedding.from_config(64, 1e6, layout=layout)
    pos = torch.randint(0, 40000, (num,), generator=gen(1)).to(torch.int32)
    q, k = randn((num, hq, 64), BF16, 2), randn((num, hk, 64), BF16, 3)
    got_q, got_k = apply_rotary(q.cuda(), pos.cuda(), rot, key=k.cuda())
    for got, x in ((got_q, q), (got_k, k)):
        ref.check(got.cpu(), *ref.turn(x, pos, rot.inv_freq, layout))


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("n", [64, 32])
def test_rows_in_place_and_strided(dev, dtype, layout, n):
    """Views of a fused projection's output turned in place (what lies between them as it was), heads
    before tokens, odd offsets, unusual last strides: the bits of contiguous inputs."""
    rot = RotaryEmbedding.from_config(64, 1e4, rotary_dim=n, layout=layout)
    num, hq, hk, d = 333, 6, 2, 64
    pos = torch.arange(num, dtype=torch.int32).cuda()
    packed = randn((num, (hq + 2 * hk) * d), dtype, 1).cuda()
    q = packed[:, :hq * d].unflatten(1, (hq, d))
    k = packed[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    want_q, want_k = apply_rotary(q.contiguous(), pos, rot, key=k.contiguous())
    before = packed.clone()
    out = apply_rotary(q, pos, rot, key=k, query_out=q, key_out=k)
    assert out[0] is q and out[1] is k
    assert_bit_exact(q.contiguous().cpu(), want_q.cpu())
    assert_bit_exact(k.contiguous().cpu(), want_k.cpu())
    assert_bit_exact(packed[:, (hq + hk) * d:].contiguous().cpu(),
                     before[:, (hq + hk) * d:].contiguous().cpu())
    q = before[:, :hq * d].unflatten(1, (hq, d))
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.empty(num * hq * d + 1, dtype=dtype, device="cuda")[1:].view(num, hq, d).copy_(q)
    wide = torch.zeros((num, hq, 2 * d), dtype=dtype, device="cuda")
    wide[..., ::2] = q
    for x in (heads_first, odd, wide[..., ::2]):
        assert_bit_exact(apply_rotary(x, pos, rot).cpu().contiguous(), want_q.cpu())
    target = torch.full((num, hq, d + 2), 7.0, dtype=dtype, device="cuda")
    got = apply_rotary(q, pos, rot, query_out=target[..., :d])
    assert_bit_exact(got.contiguous().cpu(), want_q.cpu())
    assert (target[..., d:] == 7.0).all()
    one = before[:1, :d].unflatten(1, (1, d)).expand(num, hq, d)      # one row for all of them
    assert_bit_exact(apply_rotary(one, pos, rot).cpu(), apply_rotary(one.contiguous(), pos, rot).cpu())


def test_rows_of_long_tensors(dev):
    """Offsets past 2^31 bytes and elements."""
    rot = RotaryEmbedding.from_config(128, 1e6)
    num, hq = 40000, 520                                             # 5.3 GB
    q = torch.empty((num, hq, 128), dtype=BF16, device="cuda")
    some = torch.tensor([0, 1, 20011, 39998, 39999])
    rows = randn((5, hq, 128), BF16, 1)
    q[some.cuda()] = rows.cuda()
    pos = torch.arange(num, dtype=torch.int32)
    apply_rotary(q, pos.cuda(), rot, query_out=q)
    ref.check(q[some.cuda()].cpu(), *ref.turn(rows, pos[some], rot.inv_freq, "half"))


def test_group_law(dev):
    """Turned by p and then by q is turned by p + q (two fp32-page roundings), and a norm stays."""
    rot = RotaryEmbedding.from_config(128, 1e4)
    x = randn((50, 2, 128), FP32, 1).cuda()
    p = torch.randint(0, 9000, (50,), generator=gen(2)).to(torch.int32).cuda()
    q = torch.randint(-9000, 9000, (50,), generator=gen(3)).to(torch.int32).cuda()
    two = apply_rotary(apply_rotary(x, p, rot), q, rot)
    one = apply_rotary(x, p + q, rot)
    # three roundings of 2^-24 of values up to the pair's norm (each turned value twice)
    assert float((two - one).abs().max()) <= 4 * 2.0 ** -24 * float(x.abs().max()) * 2 ** 0.5


def test_not_finite(dev):
    """A NaN or an infinity reaches its own pair only."""
    rot = RotaryEmbedding.from_config(64, 1e4, rotary_dim=32)
    x = randn((4, 1, 64), BF16, 1)
    x[0, 0, 3], x[1, 0, 16], x[2, 0, 40] = math.nan, math.inf, math.nan
    got = apply_rotary(x.cuda(), torch.tensor([5, 6, 7, 8], dtype=torch.int32).cuda(), rot).cpu()
    bad = ~got[:, 0].float().isfinite()
    assert bad[0].nonzero().flatten().tolist() == [3, 19]
    assert bad[1].nonzero().flatten().tolist() == [0, 16]
    assert bad[2].nonzero().flatten().tolist() == [40] and not bad[3].any()


# ---- appended to pages ---------------------------------------------------------------------

@pytest.mark.parametrize("d,n", [(128, 128), (64, 32), (80, 80), (6, 4)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_append(dev, dtype, layout, d, n):
    """A ragged batch with padding rows and tokens without a page; other slots as they were."""
    rot = RotaryEmbedding.from_config(d, 1e6, rotary_dim=n, layout=layout, scaling=YARN)
    bs, heads, hq = 16, 3, 6
    t0, _ = _table(70, bs, 1)
    tables = torch.stack([t0, t0 + 8]).to(torch.int32)
    nb = 16
    pos = torch.tensor([65, 66, -1, 68, 69, 0, 1, 2, 500], dtype=torch.int32)
    starts = torch.tensor([0, 5, 8], dtype=torch.int32)
    num = pos.shape[0]
    host = randn((nb, 2, heads, bs, d), dtype, 2)
    cache = host.cuda()
    k, v, q = (randn((num, h, d), dtype, s) for h, s in ((heads, 3), (heads, 4), (hq, 5)))
    q_out = torch.full((num, hq, d), 7.0, dtype=dtype).cuda()
    got_q = pc.append_kv_paged(cache, k.cuda(), v.cuda(), tables.cuda(), pos.cuda(), starts.cuda(),
                               rotary=rot, query=q.cuda(), query_out=q_out)
    assert got_q is q_out
    got, got_q = cache.cpu(), q_out.cpu()
    want_k, norm_k = ref.turn(k, pos, rot.inv_freq, layout, rot.factor)
    want_q, norm_q = ref.turn(q, pos, rot.inv_freq, layout, rot.factor)
    left = torch.ones(host.shape[:4], dtype=torch.bool)
    for t in range(num):
        if t == 2 or t >= 8:
            assert (got_q[t] == 7.0).all()
            continue
        ref.check(got_q[t:t + 1], want_q[t:t + 1], norm_q[t:t + 1])
        page, slot = int(tables[int(t >= 5), int(pos[t]) // bs]), int(pos[t]) % bs
        left[page, :, :, slot] = False
        ref.check(got[page, 0, :, slot][None], want_k[t:t + 1], norm_k[t:t + 1])
        assert_bit_exact(got[page, 1, :, slot], v[t])
    assert_bit_exact(got[left], host[left])


@pytest.mark.parametrize("d,n,layout", [(128, 128, "half"), (64, 64, "half"), (128, 64, "half"),
                                        (128, 64, "interleaved"), (64, 32, "interleaved")])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("num", [1, 40, 2100])
def test_append_4bit_matches_64_bits(dev, dtype, d, n, layout, num):
    """Codes and scales equal to those of the 64-bit result, also where the halves of a row (blocks
    of their own) are of very different size."""
    rot = RotaryEmbedding.from_config(d, 1e6, rotary_dim=n, layout=layout, scaling=YARN)
    bs, heads = 16, 2
    at = torch.arange(num, dtype=torch.int32) + 30011
    table, nb = _table(30011 + num, bs, 1)
    k = randn((num, heads, d), FP32, 3) * torch.where(torch.rand(d, generator=gen(5)) < .1, 9., 1.)
    k = k * torch.exp2(-6.0 * torch.randint(0, 3, (num, heads, d // 32), generator=gen(7))
                       ).repeat_interleave(32, -1)
    k, v = k.to(dtype), randn((num, heads, d), dtype, 4)
    cache = pc.QuantizedKVCache.allocate(nb, heads, bs, d, "cuda")
    pc.append_kv_paged(cache, k.cuda(), v.cuda(), table.cuda(), at.cuda(), rotary=rot)
    page, slot = table.long()[at.long() // bs], at.long() % bs
    for plane, x in ((0, ref.turn(k, at, rot.inv_freq, layout, rot.factor)[0]), (1, v.double())):
        c, s = pref.quantize(x)
        assert torch.equal(cache.scales.cpu()[page, plane, :, slot].long(), s)
        assert torch.equal(cache.codes.cpu()[page, plane, :, slot],
                           (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8))


@pytest.mark.parametrize("n", [128, 64])
def test_append_4bit_small_turns(dev, n):
    """Half pairs of which one element is tiny beside the other: after a small turn the small block
    holds differences of products that fp32 does not settle."""
    rot = RotaryEmbedding.from_config(128, 1e6, rotary_dim=n)
    num, bs = 600, 16
    at = torch.arange(num, dtype=torch.int32)
    k = randn((num, 1, 128), FP32, 3)
    k[..., :n // 2] *= 2.0 ** -15
    table, nb = _table(num, bs, 1)
    for kk in (k.to(BF16), k):
        cache = pc.QuantizedKVCache.allocate(nb, 1, bs, 128, "cuda")
        pc.append_kv_paged(cache, kk.cuda(), kk.cuda(), table.cuda(), at.cuda(), rotary=rot)
        c, s = pref.quantize(ref.turn(kk, at, rot.inv_freq, "half")[0])
        page, slot = table.long()[at.long() // bs], at.long() % bs
        assert torch.equal(cache.scales.cpu()[page, 0, :, slot].long(), s)
        assert torch.equal(cache.codes.cpu()[page, 0, :, slot],
                           (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_append_4bit_of_both_ends_of_the_range(dev, dtype):
    """Half pairs whose first element passes fp32 (not what a scale can hold) under the factor and whose
    second one lies at the smallest scale: each block has its own exponent."""
    rot = RotaryEmbedding(torch.zeros(32), 64, factor=2.0)
    k = torch.empty((2, 1, 64), dtype=FP32)
    k[..., :32] = randn((2, 1, 32), FP32, 1).clamp(-1, 1) * 2.0 ** 127
    k[..., 0] = 1.5 * 2.0 ** 127
    k[..., 32:] = (torch.arange(32) % 8 - 3.0) * 2.0 ** -127
    k = k.to(dtype)
    at = torch.tensor([0, 5], dtype=torch.int32)
    cache = pc.QuantizedKVCache.allocate(1, 1, 16, 64, "cuda")
    table = torch.zeros(1, dtype=torch.int32)
    pc.append_kv_paged(cache, k.cuda(), k.cuda(), table.cuda(), at.cuda(), rotary=rot)
    c, s = pref.quantize(k.double() * 2.0)
    assert torch.equal(cache.scales.cpu()[0, 0, :, at.long()].transpose(0, 1).long(), s)
    assert torch.equal(cache.codes.cpu()[0, 0, :, at.long()].transpose(0, 1),
                       (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8))


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_interleaved_whole_heads_are_rope_base(dev, dtype):
    """The path's own convention given as an embedding: the same bits as ``rope_base``."""
    d, num, bs = 64, 300, 16
    rot = RotaryEmbedding.from_config(d, 1e6, layout="interleaved")
    table, nb = _table(num, bs, 1)
    pos = torch.arange(num, dtype=torch.int32).cuda()
    k, v = randn((num, 2, d), dtype, 1).cuda(), randn((num, 2, d), dtype, 2).cuda()
    a = torch.zeros((nb, 2, 2, bs, d), dtype=dtype, device="cuda")
    b = a.clone()
    pc.append_kv_paged(a, k, v, table.cuda(), pos, rope_base=1e6)
    pc.append_kv_paged(b, k, v, table.cuda(), pos, rotary=rot)
    assert_bit_exact(a.cpu(), b.cpu())


# ---- donors and shifts ---------------------------------------------------------------------

@pytest.mark.parametrize("d,n", [(128, 128), (64, 32), (6, 4)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("pages", ["standard", "vllm", "trt"])
def test_scatter_layers(dev, dtype, layout, d, n, pages):
    """Donor rows into three layers' pages, with pairs out of range; other slots as they were."""
    rot = RotaryEmbedding.from_config(d, 1e6, rotary_dim=n, layout=layout, scaling=YARN)
    bs, heads, layers, donor_len = 16, 3, 3, 90
    table, nb = _table(128, bs, 1)
    table[3] = -1
    table[4] = nb + 2
    tpos = torch.cat([torch.arange(0, 128, 2), torch.tensor([1000, -1, 1, 3])]).to(torch.int32)
    dpos = torch.randint(0, donor_len, (tpos.shape[0],), generator=gen(2)).to(torch.int32)
    dpos[5], dpos[6], dpos[-1] = donor_len, -1, 3        # two out of range, one that does not move
    host = [randn((nb, 2, heads, bs, d), dtype, 10 + i) for i in range(layers)]
    donors = [randn((2, heads, donor_len, d), dtype, 20 + i) for i in range(layers)]
    order = {"standard": (0, 1, 2, 3, 4), "vllm": (1, 0, 3, 2, 4), "trt": (0, 1, 3, 2, 4)}[pages]
    back = [order.index(i) for i in range(5)]
    caches = [x.permute(order).contiguous().cuda().permute(back) for x in host]
    for repeated in (False, True, None):
        got = [x.clone(memory_format=torch.preserve_format) for x in caches]
        rc.rope_correct_scatter_paged_layers(got, [x.cuda() for x in donors], table.cuda(), dpos.cuda(),
                                             tpos.cuda(), repeated_donor_rows=repeated, rotary=rot)
        for layer in range(layers):
            left = torch.ones(host[layer].shape[:4], dtype=torch.bool)
            out = got[layer].cpu()
            for t, s in zip(tpos.tolist(), dpos.tolist()):
                page = int(table[t // bs]) if 0 <= t < 128 else -1
                if not (0 <= page < nb and 0 <= s < donor_len):
                    continue
                left[page, :, :, t % bs] = False
                want, norm = ref.turn(donors[layer][0, :, s][None], torch.tensor([t - s]),
                                      rot.inv_freq, layout)
                ref.check(out[page, 0, :, t % bs][None], want, norm if t != s else 0 * norm)
                assert_bit_exact(out[page, 1, :, t % bs], donors[layer][1, :, s])
            assert_bit_exact(out[left], host[layer][left])


@pytest.mark.parametrize("layers,heads,num", [(1, 1, 1), (1, 8, 4000), (28, 4, 700), (40, 8, 300),
                                              (2, 2, 9000)])
def test_scatter_of_every_launch_shape(dev, layers, heads, num):
    rot = RotaryEmbedding.from_config(64, 1e6, scaling=SCALED)
    bs = 16
    table, nb = _table(num, bs, 1)
    dpos = torch.randperm(num, generator=gen(2)).to(torch.int32)
    tpos = torch.arange(num, dtype=torch.int32)
    donors = torch.randn((layers, 2, heads, num, 64), generator=torch.Generator("cuda").manual_seed(3),
                         device="cuda", dtype=BF16)
    caches = torch.zeros((layers, nb, 2, heads, bs, 64), dtype=BF16, device="cuda")
    rc.rope_correct_scatter_paged_layers(list(caches), list(donors), table.cuda(), dpos.cuda(),
                                         tpos.cuda(), rotary=rot)
    page, slot = table.long()[tpos.long() // bs], tpos.long() % bs
    got = caches.cpu()[:, page, :, :, slot]                            # [T, L, 2, H, D]
    src = donors.cpu()[:, :, :, dpos.long()].permute(3, 0, 1, 2, 4)    # [T, L, 2, H, D]
    assert_bit_exact(got[:, :, 1].contiguous(), src[:, :, 1].contiguous())
    want, norm = ref.turn(src[:, :, 0].flatten(1, 2), tpos - dpos, rot.inv_freq, "half")
    ref.check(got[:, :, 0].flatten(1, 2), want, norm)


@pytest.mark.parametrize("d,n", [(128, 128), (64, 32), (6, 4)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("num", [7, 300])
def test_shift_layers(dev, dtype, layout, d, n, num):
    """K in place over several layers on the vLLM layout, positions in the launch and uploaded, one of
    them listed twice, deltas of 0 and positions behind the table; V and other slots as they were."""
    rot = RotaryEmbedding.from_config(d, 1e6, rotary_dim=n, layout=layout, scaling=YARN)
    bs, heads, layers = 16, 3, 2
    table, nb = _table(320, bs, 1)
    table[1] = -1
    pos = torch.randperm(320, generator=gen(2))[:num].tolist()
    delta = torch.randint(-4096, 4097, (num,), generator=gen(3)).tolist()
    delta[1] = 0
    pos[4] = pos[0]                                                    # turned twice
    pos[5] = 5000
    host = [randn((nb, 2, heads, bs, d), dtype, 10 + i) for i in range(layers)]
    caches = [x.permute(1, 0, 3, 2, 4).contiguous().cuda() for x in host]
    done = rc.apply_rope_deltas_inplace_layers(caches, table.cuda(), pos, delta, layout="vllm", rotary=rot)
    assert done == layers * sum(x != 0 and p < 320 for p, x in zip(pos, delta))
    for layer in range(layers):
        got = caches[layer].cpu().permute(1, 0, 3, 2, 4)
        assert_bit_exact(got[:, 1].contiguous(), host[layer][:, 1].contiguous())
        left = torch.ones(host[layer][:, 0].shape[:3], dtype=torch.bool)
        for i, (p, x) in enumerate(zip(pos, delta)):
            page = int(table[p // bs]) if p < 320 else -1
            if page < 0 or x == 0:
                continue
            left[page, :, p % bs] = False
            if i in (0, 4):
                continue
            want, norm = ref.turn(host[layer][page, 0, :, p % bs][None], torch.tensor([x]), rot.inv_freq,
                                  layout)
            ref.check(got[page, 0, :, p % bs][None], want, norm)
        assert_bit_exact(got[:, 0][left], host[layer][:, 0][left])
        page = int(table[pos[0] // bs])
        if page >= 0 and delta[0] and delta[4]:
            row = host[layer][page, 0, :, pos[0] % bs][None].cuda()
            for x in (delta[0], delta[4]):
                one = RotaryEmbedding(rot.inv_freq, d, layout)         # (no factor)
                row = apply_rotary(row, torch.tensor([x], dtype=torch.int32).cuda(), one)
            assert_bit_exact(got[page, 0, :, pos[0] % bs], row[0].cpu())


def test_scatter_equals_shift_and_append(dev):
    """Three ways of one row to its new position: appended there, its donor scattered there, and
    scattered unturned and then shifted (fp32 pages; a rounding each)."""
    rot = RotaryEmbedding.from_config(128, 1e6, scaling=SCALED)
    bs, heads, num, by = 16, 2, 100, 33
    table, nb = _table(num + by, bs, 1)
    bt = table.cuda()
    here = torch.arange(num, dtype=torch.int32).cuda()
    k, v = randn((num, heads, 128), FP32, 2).cuda(), randn((num, heads, 128), FP32, 3).cuda()
    empty = torch.zeros((nb, 2, heads, bs, 128), device="cuda")
    donor_cache, a, b, c = (empty.clone() for _ in range(4))
    pc.append_kv_paged(donor_cache, k, v, bt, here, rotary=rot)
    donor = pc.gather_kv_paged(donor_cache, bt, here)
    pc.append_kv_paged(a, k, v, bt, here + by, rotary=rot)
    rc.rope_correct_scatter_paged_layers([b], [donor], bt, here, here + by, rotary=rot)
    pc.append_kv_paged(c, donor[0].transpose(0, 1), donor[1].transpose(0, 1), bt, here + by)
    rc.apply_rope_deltas_inplace_layers([c], bt, (here + by).tolist(), [by] * num, rotary=rot)
    assert_bit_exact(b.cpu(), c.cpu())
    assert float((a - b).abs().max()) <= 3 * 2.0 ** -24 * 2 ** 0.5 * float(k.abs().max()) * 2
    d = empty.clone()
    pc.append_kv_paged(d, donor[0].transpose(0, 1), donor[1].transpose(0, 1), bt, here + by,
                       rotary=rot, rotations=torch.full_like(here, by))
    assert_bit_exact(b.cpu(), d.cpu())


# ---- graphs, streams, gradients ------------------------------------------------------------

def test_captured_step(dev):
    """Append, rows and a scatter captured once and replayed with new positions in the same tensors,
    eager work between the replays."""
    rot = RotaryEmbedding.from_config(64, 1e6)
    bs, heads, num = 16, 2, 24
    table, nb = _table(256, bs, 1)
    bt = table.cuda()
    pos = torch.arange(num, dtype=torch.int32).cuda()
    dpos = torch.arange(num, dtype=torch.int32).cuda()
    k, v, q = (randn((num, h, 64), BF16, s).cuda() for h, s in ((heads, 1), (heads, 2), (6, 3)))
    donor = randn((2, heads, 64, 64), BF16, 4).cuda()
    cache, other = (torch.zeros((nb, 2, heads, bs, 64), dtype=BF16, device="cuda") for _ in range(2))
    q_out, q_two = torch.empty_like(q), torch.empty_like(q)

    def step(c, o):
        pc.append_kv_paged(c, k, v, bt, pos, rotary=rot, query=q, query_out=q_out)
        apply_rotary(q, pos, rot, query_out=q_two)
        rc.rope_correct_scatter_paged_layers([o], [donor], bt, dpos, pos, rotary=rot)

    step(cache, other)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(cache, other)
    for start in (3, 50, 111):
        pos.copy_(torch.arange(start, start + num, dtype=torch.int32))
        want = [torch.zeros_like(cache), torch.zeros_like(other)]
        step(*want)
        q_want = q_out.clone()
        q_out.zero_(), q_two.zero_(), cache.zero_(), other.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert_bit_exact(cache.cpu(), want[0].cpu())
        assert_bit_exact(other.cpu(), want[1].cpu())
        assert_bit_exact(q_out.cpu(), q_want.cpu())
        assert_bit_exact(q_two.cpu(), q_want.cpu())


def test_first_call_inside_a_capture_is_refused(dev):
    rot = RotaryEmbedding.from_config(64, 1e4)
    q = randn((4, 2, 64), BF16, 1).cuda()
    pos = torch.arange(4, dtype=torch.int32).cuda()
    out = torch.empty_like(q)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="captured"):
            apply_rotary(q, pos, rot, query_out=out)
        out.copy_(q)
    assert_bit_exact(apply_rotary(q, pos, rot, query_out=out).cpu(), apply_rotary(q, pos, rot).cpu())


def test_other_stream(dev):
    rot = RotaryEmbedding.from_config(128, 1e4)
    q = randn((512, 8, 128), BF16, 1).cuda()
    pos = torch.arange(512, dtype=torch.int32).cuda()
    want = apply_rotary(q, pos, rot).cpu()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        moved = q * 1.0
        got = apply_rotary(moved, pos, rot)
    side.synchronize()
    assert_bit_exact(got.cpu(), want)


def test_gradient_is_refused(dev):
    rot = RotaryEmbedding.from_config(64, 1e4)
    q = randn((4, 2, 64), FP32, 1).cuda().requires_grad_()
    k = randn((4, 2, 64), FP32, 1).cuda()
    out, out_k = apply_rotary(q, [0, 1, 2, 3], rot, key=k)
    assert not out_k.requires_grad
    with pytest.raises(RuntimeError, match="no backward pass"):
        out.sum().backward()
    with torch.no_grad():
        assert not apply_rotary(q, [0, 1, 2, 3], rot).requires_grad
