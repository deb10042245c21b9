"""Appending to, reading and attending over the paged caches of a serving batch, against 64 bits
(tests/paged_reference.py): every format, page layout and head size the entry points take, masks
that leave rows empty, padding, unusual strides, graphs and streams."""

from __future__ import annotations

import math

import pytest
import torch

from semblend_amd import paged_cache as pc
from semblend_amd import rope_correction as rc

from . import paged_reference as ref
from .helpers import assert_bit_exact, gen, randn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _tables(lens, bs, seed, spare=3, width=None):
    """(tables [R, max_blocks] with -1 behind each request's pages, pages in the pool)."""
    need = [-(-n // bs) for n in lens]
    pool = sum(need) + spare
    perm = torch.randperm(pool, generator=gen(seed)).to(torch.int32)
    t = torch.full((len(lens), width or max(max(need), 1)), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        t[i, :n] = perm[at:at + n]
        at += n
    return t, pool


def _starts(rows):
    s = [0]
    for r in rows:
        s.append(s[-1] + r)
    return s


def _cache(nb, heads, bs, d, dtype, seed, layout="standard"):
    """(host values [NB, 2, H, bs, D], device view in that shape on the layout's storage)."""
    x = randn((nb, 2, heads, bs, d), dtype, seed)
    order = {"standard": (0, 1, 2, 3, 4), "vllm": (1, 0, 3, 2, 4), "trt": (0, 1, 3, 2, 4)}[layout]
    dev = x.permute(order).contiguous().cuda()
    return x, dev.permute([order.index(i) for i in range(5)])


def _quant_cache(nb, heads, bs, d, seed, special=False):
    g = gen(seed)
    codes = torch.randint(0, 256, (nb, 2, heads, bs, d // 2), generator=g, dtype=torch.uint8)
    scales = torch.randint(123, 129, (nb, 2, heads, bs, d // 32), generator=g, dtype=torch.uint8)
    return codes, scales, pc.QuantizedKVCache(codes.cuda(), scales.cuda())


# ---- append --------------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["standard", "vllm", "trt"])
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (FP16, 64), (FP32, 128), (BF16, 80), (FP32, 6),
                                     (FP16, 512), (BF16, 2)])
def test_append_ragged(dev, dtype, d, layout):
    """A ragged batch with padding of every kind: values, and every other slot as it was."""
    bs, heads, hq, base = 16, 3, 6, 1e4
    lens, rows = [70, 33, 1, 500], [5, 33, 1, 0]
    tables, nb = _tables(lens, bs, 1)
    starts = _starts(rows)
    num = starts[-1] + 4                     # four rows behind the last request
    pos = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, rows)]
                    + [torch.arange(4)]).to(torch.int32)
    pos[2] = -1                              # padding inside a request
    tables[0, 4] = nb + 5                    # position 66 on: no page of the pool
    pos[7] = tables.shape[1] * bs + 3        # behind the table
    host, cache = _cache(nb, heads, bs, d, dtype, 2, layout)
    k, v, q = (randn((num, h, d), dtype, s) for h, s in ((heads, 3), (heads, 4), (hq, 5)))
    q_out = torch.full((num, hq, d), 7.0, dtype=dtype).cuda()
    got_q = pc.append_kv_paged(cache, k.cuda(), v.cuda(), tables.cuda(), pos.cuda(),
                               row_starts=torch.tensor(starts, dtype=torch.int32).cuda(),
                               rope_base=base, query=q.cuda(), query_out=q_out)
    assert got_q is q_out
    got, got_q = cache.cpu(), q_out.cpu()
    want_k, want_q = ref.rotate(k, pos, base), ref.rotate(q, pos, base)
    # one rounding; 16-bit rotations are fp32: four roundings of 2^-24 of the pair's norm
    noise = (2.0 ** -50 if dtype == FP32 else 2.0 ** -22)
    touched = torch.zeros(host.shape[:4], dtype=torch.bool)
    for i, r in enumerate(rows):
        for t in range(starts[i], starts[i] + r):
            p = int(pos[t])
            if p < 0:
                assert (got_q[t] == 7.0).all()
                continue
            err = (got_q[t].double() - want_q[t]).abs()
            tol = ref.half_step(dtype) * want_q[t].abs() + noise * q[t].double().abs().amax() * 2
            assert (err <= tol + torch.finfo(dtype).tiny).all(), (t, float(err.max()))
            if p // bs >= tables.shape[1] or not 0 <= int(tables[i, p // bs]) < nb:
                continue
            page = int(tables[i, p // bs])
            touched[page, :, :, p % bs] = True
            err = (got[page, 0, :, p % bs].double() - want_k[t]).abs()
            tol = ref.half_step(dtype) * want_k[t].abs() + noise * k[t].double().abs().amax() * 2
            assert (err <= tol + torch.finfo(dtype).tiny).all(), (t, float(err.max()))
            assert_bit_exact(got[page, 1, :, p % bs], v[t])
    assert_bit_exact(got[~touched], host[~touched])
    assert (got_q[starts[-1]:] == 7.0).all()


@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_append_strides_and_alignment(dev, dtype, quant):
    """Keys cut out of a packed QKV buffer at an odd offset, and heads-major values, give what
    contiguous ones give; without rope_base K is copied."""
    bs, heads, d, num = 16, 2, 64, 45
    tables, nb = _tables([num], bs, 1)
    pos = torch.arange(num, dtype=torch.int32).cuda()
    buf = randn((num, 3 * heads * d + 1), dtype, 2).cuda()
    k = buf[:, 1:1 + heads * d].unflatten(1, (heads, d))
    v = randn((heads, num, d), dtype, 3).cuda().transpose(0, 1)
    wide = randn((num, heads, 2 * d), dtype, 4).cuda()[..., ::2]   # last stride 2

    def run(kk, vv, base):
        c = pc.QuantizedKVCache.allocate(nb, heads, bs, d, "cuda") if quant else \
            torch.zeros((nb, 2, heads, bs, d), dtype=dtype, device="cuda")
        pc.append_kv_paged(c, kk, vv, tables[0].cuda(), pos, rope_base=base)
        return (c.codes, c.scales) if quant else (c,)

    for base in (None, 1e4):
        for kk, vv in ((k, v), (wide, wide)):
            for a, b in zip(run(kk, vv, base), run(kk.contiguous(), vv.contiguous(), base)):
                assert_bit_exact(a.contiguous(), b.contiguous())
    if not quant:
        got = pc.gather_kv_paged(run(k, v, None)[0], tables[0].cuda(), num_rows=num)
        assert_bit_exact(got[0].transpose(0, 1).contiguous(), k.contiguous())


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (FP16, 64), (FP32, 96), (BF16, 32)])
@pytest.mark.parametrize("num", [1, 17, 2500])
def test_append_4bit_matches_64_bits(dev, dtype, d, num):
    """Codes and scale bytes equal to the 64-bit quantiser's, K rotated at far positions; other
    rows of the pages as they were."""
    bs, heads, base = 16, 2, 1e6
    at = torch.arange(num, dtype=torch.int32) + 30011
    tables, nb = _tables([30011 + num], bs, 1)
    codes, scales, cache = _quant_cache(nb, heads, bs, d, 2)
    k = randn((num, heads, d), dtype, 3) * torch.where(torch.rand(d, generator=gen(5)) < .1, 9., 1.)
    k, v = k.to(dtype), randn((num, heads, d), dtype, 4)
    pc.append_kv_paged(cache, k.cuda(), v.cuda(), tables[0].cuda(), at.cuda(), rope_base=base)
    page, slot = tables[0].long()[at.long() // bs], at.long() % bs
    want_c, want_s = codes.clone(), scales.clone()
    for plane, x in ((0, ref.rotate(k, at, base)), (1, v.double())):
        c, s = ref.quantize(x)
        want_c[page, plane, :, slot] = (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8)
        want_s[page, plane, :, slot] = s.to(torch.uint8)
    assert torch.equal(cache.scales.cpu(), want_s)
    assert torch.equal(cache.codes.cpu(), want_c)
    got = pc.gather_kv_paged(cache, tables[0].cuda(), at.cuda(), dtype=FP32)
    want = ref.dequantize(want_c, want_s)[page, :, :, slot].permute(1, 2, 0, 3)
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_append_4bit_ties_zeros_and_not_finite(dev, dtype):
    """Every border between two codes and the values beside it at scales over the dtype's range,
    zero blocks (of either sign), blocks with a NaN or an infinity."""
    bs, heads, d = 16, 1, 64
    lo, hi = {BF16: (-126, 120), FP16: (-14, 12), FP32: (-126, 120)}[dtype]
    borders = torch.tensor([.25, .75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.5, 7.0])
    eps = torch.finfo(dtype).eps
    around = torch.cat([borders, borders * (1 - eps), borders * (1 + eps)]).to(dtype)
    rows = []
    for e in range(lo, hi, 3):
        block = torch.zeros(64, dtype=torch.float64)
        block[:27] = around.double()
        block[32:59] = -around.double().flip(0).clamp(max=7.0)
        rows.append(block * 2.0 ** e)
    x = torch.stack(rows).to(dtype)
    extra = torch.zeros((8, 64), dtype=dtype)
    extra[1] = -0.0
    extra[2, 3], extra[3, 40], extra[4, 0] = math.nan, math.inf, -math.inf
    extra[5] = torch.finfo(dtype).max
    extra[6, ::2] = torch.finfo(dtype).smallest_normal
    extra[7, 5] = torch.finfo(dtype).tiny / 4
    x = torch.cat([x, extra])[:, None, :]
    num = x.shape[0]
    tables, nb = _tables([num], bs, 1)
    cache = pc.QuantizedKVCache.allocate(nb, heads, bs, d, "cuda")
    pc.append_kv_paged(cache, x.cuda(), x.flip(0).cuda(), tables[0].cuda(),
                       torch.arange(num, dtype=torch.int32).cuda())
    page, slot = tables[0].long()[torch.arange(num) // bs], torch.arange(num) % bs
    for plane, y in ((0, x), (1, x.flip(0))):
        c, s = ref.quantize(y.double())
        got_s = cache.scales.cpu()[page, plane, :, slot].long()
        got_c = cache.codes.cpu()[page, plane, :, slot]
        assert torch.equal(got_s, s)
        assert torch.equal(got_c, (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8))
    back = pc.gather_kv_paged(cache, tables[0].cuda(), num_rows=num, dtype=FP32).cpu()
    bad = ~x[:, 0].float().unflatten(1, (2, 32)).isfinite().all(-1)
    assert torch.equal(back[0, 0].unflatten(1, (2, 32)).isnan().all(-1), bad)
    assert torch.equal(back[0, 0].unflatten(1, (2, 32)).isnan().any(-1), bad)


def test_append_rotations_and_donor(dev):
    """A donor buffer read from one request's pages and appended to another's, rotated by the
    difference of the positions, equals appending the keys there in the first place."""
    bs, heads, d, n, base = 16, 2, 64, 100, 1e4
    tables, nb = _tables([n, n + 40], bs, 1)
    t = tables.cuda()
    k, v = randn((n, heads, d), FP32, 2).cuda(), randn((n, heads, d), FP32, 3).cuda()
    here = torch.arange(n, dtype=torch.int32).cuda()
    there = here + 40
    cache = torch.zeros((nb, 2, heads, bs, d), device="cuda")
    pc.append_kv_paged(cache, k, v, t[0], here, rope_base=base)
    donor = pc.gather_kv_paged(cache, t[0], here)
    moved, direct = cache.clone(), cache.clone()
    pc.append_kv_paged(moved, donor[0].transpose(0, 1), donor[1].transpose(0, 1), t[1], there,
                       rope_base=base, rotations=there - here)
    pc.append_kv_paged(direct, k, v, t[1], there, rope_base=base)
    # two fp32 roundings against one
    torch.testing.assert_close(moved, direct, atol=2 ** -22 * 8.0, rtol=0)
    scattered = cache.clone()
    rc.rope_correct_scatter_paged(scattered, donor, t[1], here, there, rope_base=base)
    # (its angle is the fp32 product of 40 and the frequency: 2^-24 * 40 of an angle more)
    torch.testing.assert_close(moved, scattered, atol=8.0 * (2 ** -22 + 40 * 2 ** -24), rtol=0)


def test_append_matches_projection_write(dev):
    """The same K rows as qkv_projection_paged writes at the same positions (its angles are fp32
    products: 2^-24 of the angle apart, and a rounding each)."""
    from semblend_amd import triton_kernels as tk

    bs, heads, d, n, base = 16, 2, 64, 40, 1e6
    tables, nb = _tables([512], bs, 1)
    bt = tables[0].cuda()
    x = randn((512, 4 * d), BF16, 2).cuda()
    w = torch.eye(4 * d, dtype=BF16).cuda()        # no query head but two, K and V as they are
    w = torch.cat([w[:2 * d], w[:2 * d], w[2 * d:]])
    pos = torch.randperm(512, generator=gen(3))[:n].sort().values.to(torch.int32).cuda()
    a = torch.zeros((nb, 2, heads, bs, d), dtype=BF16, device="cuda")
    b = a.clone()
    q = tk.qkv_projection_paged(x, w, pos, a, bt, heads, heads, d, rope_base=base)
    rows = x[pos.long()].view(n, 4, d)
    got = pc.append_kv_paged(b, rows[:, :2], rows[:, 2:], bt, pos, rope_base=base,
                             query=rows[:, :2])
    assert_bit_exact(a[:, 1], b[:, 1])
    for y, z in ((a[:, 0], b[:, 0]), (q, got)):
        err = (y.double() - z.double()).abs()
        assert (err <= 2 * ref.half_step(BF16) * y.double().abs() + 512 * 2 ** -24 * 8).all()


# ---- gather --------------------------------------------------------------------------------

@pytest.mark.parametrize("layout", ["standard", "vllm"])
@pytest.mark.parametrize("dtype,d", [(BF16, 128), (FP16, 64), (FP32, 64), (BF16, 6)])
def test_gather_16bit(dev, dtype, d, layout):
    bs, heads, n = 24, 3, 301
    tables, nb = _tables([n], bs, 1)
    tables[0, 3] = -1
    host, cache = _cache(nb, heads, bs, d, dtype, 2, layout)
    pos = torch.randint(-3, n + 60, (77,), generator=gen(4)).to(torch.int32)
    got = pc.gather_kv_paged(cache, tables[0].cuda(), pos.cuda()).cpu()
    for i, p in enumerate(pos.tolist()):
        page = int(tables[0, p // bs]) if 0 <= p < tables.shape[1] * bs else -1
        want = host[page, :, :, p % bs] if page >= 0 else torch.zeros((2, heads, d), dtype=dtype)
        assert_bit_exact(got[:, :, i], want)
    out = torch.zeros((2, heads, n, d + 8), dtype=dtype, device="cuda")[..., :d]
    full = pc.gather_kv_paged(cache, tables[0].cuda(), num_rows=n, out=out)
    assert full is out
    assert_bit_exact(full[:, :, 100].cpu(), host[tables[0, 100 // bs].item(), :, :, 100 % bs])


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("d", [32, 64, 128])
def test_gather_4bit_every_byte(dev, dtype, d):
    """All 256 code bytes under every scale byte (NaN under 255), rounded once to the dtype."""
    bs = 32
    codes = torch.arange(256, dtype=torch.uint8).repeat(256 * 16 // 256 * 64)[:256 * 2 * bs * d // 2]
    codes = codes.view(-1, 2, 1, bs, d // 2).clone()
    scales = torch.arange(256, dtype=torch.uint8).repeat_interleave(d // 32)
    scales = scales.repeat(codes.numel() // (d // 2) // 256 + 1)[:codes[..., 0].numel() * (d // 32)]
    scales = scales.view(*codes.shape[:4], d // 32).clone()
    cache = pc.QuantizedKVCache(codes.cuda(), scales.cuda())
    nb = codes.shape[0]
    got = pc.gather_kv_paged(cache, torch.arange(nb, dtype=torch.int32).cuda(), dtype=dtype).cpu()
    want = ref.dequantize(codes, scales).permute(1, 2, 0, 3, 4).flatten(2, 3)
    # (scale byte 0 lies below fp32's and bf16's normal numbers, where results may be flushed)
    small = want.abs() < 2.0 ** -125
    assert torch.equal(got.isnan(), want.isnan())
    same = (got == want.to(dtype)) | got.isnan() | small
    assert same.all()
    assert (got[small].double().abs() <= 2.0 ** -125).all()


# ---- attention -----------------------------------------------------------------------------

def _attend_case(dtype, d, hq, hkv, bs, lens, rows, window, sinks, quant=False, layout="standard",
                 positions=None, seed=0, scale=None, max_rows=None, width=None):
    tables, nb = _tables(lens, bs, seed + 1, width=width)
    starts = None if rows is None else _starts(rows)
    if positions is None:
        rr = rows or [1] * len(lens)
        positions = torch.cat([torch.arange(n - r, n) for n, r in zip(lens, rr)]).to(torch.int32)
    if quant:
        codes, scales, cache = _quant_cache(nb, hkv, bs, d, seed + 2)
        c64 = ref.dequantize(codes, scales)
    else:
        host, cache = _cache(nb, hkv, bs, d, dtype, seed + 2, layout)
        c64 = host.double()
    q = (randn((positions.numel(), hq, d), FP32, seed + 3) * 1.5).to(dtype)
    sc = d ** -0.5 if scale is None else scale
    want, mass, serr = ref.attention(q, c64, tables, positions, starts, window, sinks, sc)
    out = torch.full(q.shape, 3.0, dtype=dtype).cuda()
    got = pc.paged_attention(q.cuda(), cache, tables.cuda(), positions.cuda(),
                             None if starts is None else
                             torch.tensor(starts, dtype=torch.int32).cuda(),
                             max_rows=max_rows, window=window, sinks=sinks, scale=scale, out=out)
    assert got is out
    got = got.cpu()
    pad = want.isnan()
    assert (got[pad] == 3.0).all()
    bound = ref.attention_bound(want, mass, serr, dtype, max(lens))
    err = torch.where(pad, torch.zeros_like(want), (got.double() - want).abs())
    worst = (err / bound.clamp_min(1e-30)).masked_fill(pad, 0.0)
    assert (worst <= 1).all(), f"{float(worst.max()):.3f} of the bound, error {float(err.max()):.3g}"
    return got


FORMATS = [(BF16, False), (FP16, False), (FP32, False), (BF16, True), (FP16, True), (FP32, True)]


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("d,hq,hkv,bs", [(128, 28, 4, 16), (64, 14, 2, 16), (128, 8, 8, 32),
                                         (64, 20, 1, 1), (128, 5, 1, 24), (96, 6, 2, 16),
                                         (32, 4, 4, 8)])
@pytest.mark.parametrize("window,sinks", [(None, 0), (37, 0), (64, 4), (1, 0), (200, 70)])
def test_decode(dev, dtype, quant, d, hq, hkv, bs, window, sinks):
    """One row per request, lengths from one token on, ends inside pages and tiles."""
    _attend_case(dtype, d, hq, hkv, bs, [1, 2, 31, 32, 33, 200, 517], None, window, sinks, quant)


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4), (17, 0)])
@pytest.mark.parametrize("d,hq,hkv,bs", [(128, 28, 4, 16), (64, 14, 2, 32), (128, 4, 2, 24)])
def test_mixed_batch(dev, dtype, quant, d, hq, hkv, bs, window, sinks):
    """Chunks of every size between single tokens and empty requests."""
    _attend_case(dtype, d, hq, hkv, bs, [300, 5, 64, 129, 1, 700], [90, 1, 64, 3, 0, 40], window,
                 sinks, quant)


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("layout", ["vllm", "trt"])
def test_layouts_and_scattered_rows(dev, dtype, quant, layout):
    """Recomputed rows scattered over the context and out of order."""
    pos = torch.randperm(400, generator=gen(9))[:150].to(torch.int32)
    _attend_case(dtype, 64, 14, 2, 16, [400], [150], 90, 4, quant, "standard" if quant else layout,
                 positions=pos)


@pytest.mark.parametrize("dtype,quant", [(BF16, False), (FP32, False), (FP16, True)])
@pytest.mark.parametrize("rows,max_rows", [([1, 1, 1], 1), ([2, 3, 1], 3), ([2, 3, 1], None),
                                           ([40, 1, 7], 2), ([40, 1, 7], 1000)])
def test_max_rows_is_a_hint(dev, dtype, quant, rows, max_rows):
    _attend_case(dtype, 128, 28, 4, 16, [150, 90, 61], rows, None, 0, quant, max_rows=max_rows)


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("hq,hkv", [(28, 4), (8, 2), (20, 1)])
def test_requests_of_a_few_rows(dev, dtype, quant, hq, hkv):
    """Requests on both sides of where their rows change kernels (48 rows and heads of a group), of
    one to three row tiles of 16 each, without and with others of many rows."""
    for extra in ([], [70]):
        rows = [7, 6, 5, 1, 12, 13, 2, 3, 0, 7] + extra
        _attend_case(dtype, 64, hq, hkv, 16, [30 + 41 * i for i in range(len(rows))], rows, None, 0,
                     quant)
        _attend_case(dtype, 128, hq, hkv, 16, [30 + 41 * i for i in range(len(rows))], rows, 50, 3,
                     quant, max_rows=max(rows))


@pytest.mark.parametrize("dtype,quant", FORMATS)
def test_long_context_is_split(dev, dtype, quant):
    """Few items over a long context: the key ranges are split and joined."""
    _attend_case(dtype, 64, 4, 2, 16, [6000], None, None, 0, quant)
    _attend_case(dtype, 64, 4, 2, 16, [6000, 3], [20, 1], None, 0, quant)
    _attend_case(dtype, 64, 4, 2, 16, [5000], None, 2900, 33, quant)


@pytest.mark.parametrize("dtype,quant", FORMATS)
def test_padding_and_rows_that_see_nothing(dev, dtype, quant):
    """Negative positions stay as they are, also between live rows; rows whose window lies behind
    the table, or whose pages are none of the pool's, get zeros; rows behind the last request
    stay."""
    d, hq, hkv, bs = 64, 14, 2, 16
    tables, nb = _tables([64, 64, 64], bs, 1)
    tables[1] = -1
    tables[2, 1:3] = nb + 1
    if quant:
        codes, scales, cache = _quant_cache(nb, hkv, bs, d, 2)
        c64 = ref.dequantize(codes, scales)
    else:
        host, cache = _cache(nb, hkv, bs, d, dtype, 2)
        c64 = host.double()
    for rows in ([4, 3, 3], [70, 3, 41]):
        starts = _starts(rows)
        num = starts[-1] + 5
        pos = torch.randint(0, 64, (num,), generator=gen(3)).to(torch.int32)
        pos[1] = -1
        pos[2] = 500                      # the window (8) ends behind the 64 keys of the table
        pos[starts[2]] = 40               # its window: pages 1 and 2, none of the pool's
        pos[starts[2] + 1] = 70           # window 63..70, one key in the table
        q = randn((num, hq, d), dtype, 4)
        want, mass, serr = ref.attention(q, c64, tables, pos, starts, 8, 0, d ** -0.5)
        out = torch.full(q.shape, 3.0, dtype=dtype).cuda()
        pc.paged_attention(q.cuda(), cache, tables.cuda(), pos.cuda(),
                           torch.tensor(starts, dtype=torch.int32).cuda(), window=8, out=out)
        got = out.cpu()
        assert (got[1] == 3.0).all() and (got[starts[-1]:] == 3.0).all()
        assert (got[2] == 0).all() and (got[starts[1]:starts[2]] == 0).all()
        assert (got[starts[2]] == 0).all()
        live = ~want.isnan()
        bound = ref.attention_bound(want, mass, serr, dtype, 64)
        assert ((got.double() - want).abs()[live] <= bound[live]).all()


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("rows", [1, 3, 90])
def test_masked_places_may_hold_anything(dev, dtype, quant, rows):
    """NaN and infinities in keys that a row does not see: behind its position, between the sinks
    and the window, in slots behind the context. Rows that do see one get what the sum gives."""
    d, hq, hkv, bs, n = 64, 14, 2, 16, 150
    tables, nb = _tables([n], bs, 1, spare=0)
    pos = torch.arange(n - rows, n, dtype=torch.int32)
    t = torch.arange(tables.shape[1] * bs)
    if quant:
        codes, scales, cache = _quant_cache(nb, hkv, bs, d, 2)
    else:
        host, _ = _cache(nb, hkv, bs, d, dtype, 2)
    kinds = (math.nan,) if quant else (math.nan, math.inf, -math.inf)
    window, sinks = 20, 3
    for bad_at in ([n, n + 3], [5, 70] if rows < 90 else [5, 30], [n - 1] if rows > 1 else [5],
                   [max(0, n - rows - 19)], [0]):
        for kind in kinds:
            x = torch.tensor(bad_at)
            page, slot = tables[0].long()[x // bs], x % bs
            if quant:
                s = scales.clone()
                s[page, :, :, slot, 1] = 255
                c = pc.QuantizedKVCache(codes.cuda(), s.cuda())
                c64 = ref.dequantize(codes, s)
            else:
                h = host.clone()
                h[page, :, :, slot, 5::7] = kind
                c, c64 = h.cuda(), h.double()
            q = randn((rows, hq, d), dtype, 4)
            want, mass, serr = ref.attention(q, c64, tables, pos, [0, rows], window, sinks, .125)
            # (the definition's sum over seen keys only; a seen -inf key gives a score of either
            # sign, so only rows without one are compared as numbers)
            got = pc.paged_attention(q.cuda(), c, tables[0].cuda(), pos.cuda(), window=window,
                                     sinks=sinks, scale=.125).cpu()
            sees_bad = torch.tensor([[bool(ref.visible(int(p), torch.tensor([b]), window, sinks))
                                      for b in bad_at] for p in pos]).any(1)
            clean = ~sees_bad
            assert got[clean].isfinite().all(), (bad_at, kind)
            bound = ref.attention_bound(want, mass, serr, dtype, n)
            assert ((got.double() - want).abs()[clean] <= bound[clean]).all()
            if sees_bad.any() and kind != kind:
                assert not got[sees_bad].isfinite().all(-1).any()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("rows", [1, 60])
def test_seen_infinite_values(dev, dtype, rows):
    """A seen V of +inf gives +inf in its columns, +inf and -inf together NaN, whether the tile is
    seen whole or in part."""
    d, hq, hkv, bs, n = 64, 8, 2, 16, 200
    tables, nb = _tables([n], bs, 1)
    host, _ = _cache(nb, hkv, bs, d, dtype, 2)
    for at in (40, n - 3 - rows):
        h = host.clone()
        page, slot = int(tables[0, at // bs]), at % bs
        page2, slot2 = int(tables[0, (at - 2) // bs]), (at - 2) % bs
        h[page, 1, :, slot, 3] = math.inf
        h[page, 1, :, slot, 9] = math.inf
        h[page2, 1, :, slot2, 9] = -math.inf
        h[page2, 1, :, slot2, 11] = -math.inf
        q = randn((rows, hq, d), dtype, 4)
        pos = torch.arange(n - rows, n, dtype=torch.int32)
        got = pc.paged_attention(q.cuda(), h.cuda(), tables[0].cuda(), pos.cuda()).cpu().float()
        assert (got[..., 3] == math.inf).all() and (got[..., 11] == -math.inf).all()
        assert got[..., 9].isnan().all()
        rest = [i for i in range(d) if i not in (3, 9, 11)]
        assert got[..., rest].isfinite().all()


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("rows", [1, 50])
def test_rising_scores_and_scales(dev, dtype, quant, rows):
    """Large and rising logits (the reference moves many times); scales of other signs."""
    for scale in (3.0, 0.0, -0.4, 1e-39):
        _attend_case(dtype, 64, 4, 2, 16, [333], [rows], None, 0, quant, scale=scale)


@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_unaligned_and_strided_rows(dev, dtype):
    """Queries cut from a packed buffer (aligned or not), outputs into one, transposed heads."""
    d, hq, hkv, bs, n = 64, 8, 2, 16, 90
    tables, nb = _tables([n], bs, 1)
    host, cache = _cache(nb, hkv, bs, d, dtype, 2)
    pos = torch.arange(20, 90, dtype=torch.int32).cuda()
    buf = randn((70, hq * d + 16), dtype, 3).cuda()
    bt = tables[0].cuda()
    for shift in (0, 8, 1):
        q = buf[:, shift:shift + hq * d].unflatten(1, (hq, d))
        want = pc.paged_attention(q.contiguous(), cache, bt, pos, window=30, sinks=2)
        out = torch.zeros((70, 2 * hq * d + 1), dtype=dtype, device="cuda")
        view = out[:, shift:shift + hq * d].unflatten(1, (hq, d))
        got = pc.paged_attention(q, cache, bt, pos, window=30, sinks=2, out=view)
        u = ref.half_step(dtype)
        tol = 4 * u if dtype != FP32 else 2 ** -18   # another kernel's roundings
        torch.testing.assert_close(got.float(), want.float(), atol=4 * tol, rtol=tol)
        assert (out[:, shift + hq * d:] == 0).all()
    heads_major = buf[:, :hq * d].unflatten(1, (hq, d)).transpose(0, 1).contiguous()
    got = pc.paged_attention(heads_major.transpose(0, 1), cache, bt, pos, window=30, sinks=2)
    want = pc.paged_attention(heads_major.transpose(0, 1).contiguous(), cache, bt, pos, window=30,
                              sinks=2)
    assert_bit_exact(got.contiguous(), want)


def test_tables_of_other_types_and_strides(dev):
    d, hq, hkv, bs = 64, 4, 2, 16
    tables, nb = _tables([60, 33], bs, 1)
    _, cache = _cache(nb, hkv, bs, d, BF16, 2)
    q = randn((2, hq, d), BF16, 3).cuda()
    pos = torch.tensor([59, 32], dtype=torch.int32).cuda()
    want = pc.paged_attention(q, cache, tables.cuda(), pos)
    wide = torch.full((2, 40), 12345, dtype=torch.int32).cuda()
    wide[:, 5:5 + tables.shape[1]] = tables.cuda()
    for bt in (tables.long().cuda(), tables, wide[:, 5:5 + tables.shape[1]],
               tables.t().contiguous().cuda().t()):
        assert_bit_exact(pc.paged_attention(q, cache, bt, pos), want)
    assert_bit_exact(pc.paged_attention(q, cache, tables.cuda(), pos.long()), want)
    assert_bit_exact(pc.paged_attention(q[1:], cache, tables[1].cuda(), [32]), want[1:])


@pytest.mark.parametrize("quant", [False, True])
def test_offsets_past_32_bits(dev, quant):
    """Pages far into a pool of more than 4 GiB (2 GiB of scales' codes for 4 bits)."""
    d, hq, hkv, bs = 128, 8, 8, 16
    page = 2 * hkv * bs * (d // 2 if quant else 2 * d)
    nb = (9 << 29) // page
    tables = torch.tensor([[nb - 1, 3, nb - 7, nb // 2]], dtype=torch.int32)
    ids = tables[0].long()
    if quant:
        codes, scales, _ = _quant_cache(4, hkv, bs, d, 2)
        cache = pc.QuantizedKVCache(
            torch.empty((nb, 2, hkv, bs, d // 2), dtype=torch.uint8, device="cuda"),
            torch.empty((nb, 2, hkv, bs, d // 32), dtype=torch.uint8, device="cuda"))
        cache.codes[ids.cuda()], cache.scales[ids.cuda()] = codes.cuda(), scales.cuda()
        small = pc.QuantizedKVCache(codes.cuda(), scales.cuda())
    else:
        host, small = _cache(4, hkv, bs, d, BF16, 2)
        cache = torch.empty((nb, 2, hkv, bs, d), dtype=BF16, device="cuda")
        cache[ids.cuda()] = small
    near = torch.arange(4, dtype=torch.int32)[None].cuda()
    k, v = (randn((2, hkv, d), BF16, s).cuda() for s in (3, 4))
    for rows in (1, 50):
        pos = torch.arange(60 - rows, 60, dtype=torch.int32).cuda()
        q = randn((rows, hq, d), BF16, 5).cuda()
        at = torch.tensor([60, 17], dtype=torch.int32).cuda()
        for c, t in ((cache, tables.cuda()), (small, near)):
            pc.append_kv_paged(c, k, v, t[0], at, rope_base=1e4)
        assert_bit_exact(pc.paged_attention(q, cache, tables[0].cuda(), pos),
                         pc.paged_attention(q, small, near[0], pos))
        assert_bit_exact(pc.gather_kv_paged(cache, tables[0].cuda()),
                         pc.gather_kv_paged(small, near[0]))


def test_many_requests(dev):
    """More requests than one scan step, most of them empty or padding."""
    d, hq, hkv, bs, n = 64, 14, 2, 16, 150
    lens = [1 + (37 * i) % 90 for i in range(n)]
    rows = [0 if i % 3 == 0 else 1 + (i % 7 == 0) * min(20, lens[i] - 1) for i in range(n)]
    for dtype, quant in ((BF16, False), (FP16, True), (FP32, False)):
        _attend_case(dtype, d, hq, hkv, bs, lens, rows, 50, 2, quant)


@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("hkv,hq,d,num", [(150, 300, 4, 3), (1, 1, 2, 700), (130, 1, 512, 2),
                                          (7, 3, 32, 5000)])
def test_append_many_heads_or_tokens(dev, dtype, hkv, hq, d, num):
    """Tokens of more rows than a workgroup takes, and rows of a few bytes: V exactly, K and the
    query rotated (two products and a sum in fp32 at most, and one rounding)."""
    bs = 16
    tables, nb = _tables([num], bs, 1)
    _, cache = _cache(nb, hkv, bs, d, dtype, 2)
    k, v = (randn((num, hkv, d), dtype, s) for s in (3, 4))
    q = randn((num, hq, d), dtype, 5)
    pos = torch.randperm(num, generator=gen(6)).to(torch.int32)
    got_q = pc.append_kv_paged(cache, k.cuda(), v.cuda(), tables[0].cuda(), pos.cuda(),
                               rope_base=1e4, query=q.cuda()).cpu()
    rows = cache.cpu()[tables[0].long()[(pos // bs).long()], :, :, (pos % bs).long()]
    assert_bit_exact(rows[:, 1], v)
    for got, x in ((rows[:, 0], k), (got_q, q)):
        want = ref.rotate(x, pos, 1e4)
        norm = x.double().unflatten(-1, (-1, 2)).norm(dim=-1).repeat_interleave(2, -1)
        bound = want.abs() * ref.half_step(dtype) + norm * 2.0 ** -21
        assert ((got.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("dtype,quant", FORMATS)
def test_one_row_of_several_requests(dev, dtype, quant):
    """A batch of one row whose request is not the first, and one whose only row is padding: the
    context is long enough to be split."""
    _attend_case(dtype, 64, 4, 2, 16, [10, 6000, 10], [0, 1, 0], None, 0, quant)
    _attend_case(dtype, 64, 40, 1, 16, [10, 6000, 10], [0, 1, 0], None, 0, quant)
    _attend_case(dtype, 64, 4, 2, 16, [6000], [0], None, 0, quant,
                 positions=torch.tensor([5999], dtype=torch.int32))


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("window,sinks", [(None, 0), (1, 0), (5, 4), (2 ** 31 + 5, 2 ** 40)])
def test_largest_position(dev, dtype, quant, window, sinks):
    """Rows at 2^31 - 1 see the whole table, or the first tokens, or nothing."""
    for rows in (1, 60):
        pos = torch.full((rows,), 2 ** 31 - 1, dtype=torch.int32)
        pos[rows // 2:] -= torch.arange(rows - rows // 2, dtype=torch.int32)
        for d in (64, 96):
            _attend_case(dtype, d, 4, 2, 16, [100], [rows], window, sinks, quant, positions=pos)


@pytest.mark.parametrize("dtype,quant", FORMATS)
def test_output_in_place_of_the_query(dev, dtype, quant):
    d, hq, hkv, bs = 64, 14, 2, 16
    tables, nb = _tables([3000, 90], bs, 1)
    cache = _quant_cache(nb, hkv, bs, d, 2)[2] if quant else _cache(nb, hkv, bs, d, dtype, 2)[1]
    for rows in (None, [70, 1]):
        lens = rows or [1, 1]
        pos = torch.cat([torch.arange(n - r, n) for n, r in zip([3000, 90], lens)]).int().cuda()
        rs = None if rows is None else torch.tensor(_starts(rows), dtype=torch.int32).cuda()
        q = randn((pos.numel(), hq, d), dtype, 3).cuda()
        want = pc.paged_attention(q, cache, tables.cuda(), pos, rs)
        got = pc.paged_attention(q, cache, tables.cuda(), pos, rs, out=q)
        assert got is q
        assert_bit_exact(got, want)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("pad", [0, 12])
def test_codes_and_scales_in_one_row(dev, dtype, pad):
    """Codes and scale bytes of a row side by side (rows of 68 bytes, or padded to 80, so that the
    codes stay aligned), pages apart: strides that are no multiples of each other."""
    d, hq, hkv, bs = 128, 28, 4, 16
    tables, nb = _tables([400, 33], bs, 1)
    codes, scales, cache = _quant_cache(nb, hkv, bs, d, 2)
    width = d // 2 + d // 32 + pad
    both = torch.zeros((nb, 3, hkv, bs, width), dtype=torch.uint8, device="cuda")[:, :2]
    other = pc.QuantizedKVCache(both[..., :d // 2], both[..., d // 2:d // 2 + d // 32])
    other.codes.copy_(codes)
    other.scales.copy_(scales)
    t = tables.cuda()
    for rows in ([1, 1], [100, 3]):
        pos = torch.cat([torch.arange(n - r, n) for n, r in zip([400, 33], rows)]).int().cuda()
        rs = torch.tensor(_starts(rows), dtype=torch.int32).cuda()
        k, v = (randn((pos.numel(), hkv, d), dtype, s).cuda() for s in (3, 4))
        q = randn((pos.numel(), hq, d), dtype, 5).cuda()
        for c in (cache, other):
            pc.append_kv_paged(c, k, v, t, pos, rs, rope_base=1e4)
        assert torch.equal(cache.codes, other.codes) and torch.equal(cache.scales, other.scales)
        want, mass, serr = ref.attention(q.cpu(), ref.dequantize(cache.codes.cpu(),
                                                                 cache.scales.cpu()), tables,
                                         pos.cpu(), _starts(rows), 50, 4, d ** -0.5)
        got = pc.paged_attention(q, other, t, pos, rs, window=50, sinks=4).cpu()
        assert ((got.double() - want).abs() <= ref.attention_bound(want, mass, serr, dtype,
                                                                   400)).all()
    assert_bit_exact(pc.gather_kv_paged(other, t[0]), pc.gather_kv_paged(cache, t[0]))
    if pad:
        assert (both[..., d // 2 + d // 32:] == 0).all()


@pytest.mark.parametrize("quant", [False, True])
def test_append_tokens_of_no_request_or_slot(dev, quant):
    """Tokens before the first request's and behind the last one's are left out, and so are slots
    behind the table, up to position 2^31 - 1 (whose query is rotated all the same)."""
    d, hq, hkv, bs = 64, 4, 2, 16
    tables, nb = _tables([64, 64], bs, 1)
    cache = _quant_cache(nb, hkv, bs, d, 2)[2] if quant else _cache(nb, hkv, bs, d, BF16, 2)[1]
    parts = (cache.codes, cache.scales) if quant else (cache,)
    before = [p.clone() for p in parts]
    pos = torch.tensor([3, 4, 2 ** 31 - 1, 64, 5, 6], dtype=torch.int32)
    q = randn((6, hq, d), BF16, 3)
    out = torch.full(q.shape, 3.0, dtype=BF16).cuda()
    got = pc.append_kv_paged(cache, randn((6, hkv, d), BF16, 4).cuda(),
                             randn((6, hkv, d), BF16, 5).cuda(), tables.cuda(), pos.cuda(),
                             torch.tensor([2, 3, 4], dtype=torch.int32).cuda(), rope_base=1e4,
                             query=q.cuda(), query_out=out).cpu()
    for p, b in zip(parts, before):
        assert torch.equal(p.cpu(), b.cpu())
    rows = [0, 1, 4, 5]
    assert (got[rows] == 3.0).all()
    # (interleaved sums of two products in fp32, 2^-22 of the pair's norm, and one rounding)
    want = ref.rotate(q, pos, 1e4)
    norm = q.double().unflatten(-1, (-1, 2)).norm(dim=-1).repeat_interleave(2, -1)
    err = (got.double() - want).abs()
    bound = want.abs() * ref.half_step(BF16) + norm * 2.0 ** -21
    assert (err <= bound)[2:4].all()


@pytest.mark.parametrize("n", [2048, 2049])
@pytest.mark.parametrize("dtype,quant", [(BF16, False), (FP16, True), (FP32, False)])
def test_very_many_single_rows(dev, dtype, quant, n):
    """Decode steps on both sides of the most rows whose items are balanced, with tables of 9600
    keys: padding rows, one long row, the others short."""
    lens = [1 + (37 * i) % 40 for i in range(n)]
    lens[n // 2] = 5000
    pos = torch.tensor([-1 if i % 5 == 3 else x - 1 for i, x in enumerate(lens)], dtype=torch.int32)
    pos[n // 2] = 4999
    _attend_case(dtype, 64, 3, 1, 16, lens, None, None, 0, quant, positions=pos, width=600)


# ---- together, captured, on other streams -----------------------------------------------------

@pytest.mark.parametrize("quant", [False, True])
def test_prompt_then_decode(dev, quant):
    """A prompt appended in chunks and attended under a window, then decode steps of a batch, as a
    server runs them, against 64 bits on the caches the appends left."""
    d, hq, hkv, bs, base, window, sinks = 64, 14, 2, 16, 1e4, 60, 4
    lens = [150, 40]
    tables, nb = _tables([n + 8 for n in lens], bs, 1)
    t = tables.cuda()
    cache = pc.QuantizedKVCache.allocate(nb, hkv, bs, d, "cuda") if quant else \
        torch.zeros((nb, 2, hkv, bs, d), dtype=BF16, device="cuda")

    def step(rows, pos, seed):
        starts = _starts(rows)
        num = starts[-1]
        k, v = (randn((num, hkv, d), BF16, seed + i) for i in (0, 1))
        q = randn((num, hq, d), BF16, seed + 2)
        rs = torch.tensor(starts, dtype=torch.int32).cuda()
        qr = pc.append_kv_paged(cache, k.cuda(), v.cuda(), t, pos.cuda(), row_starts=rs,
                                rope_base=base, query=q.cuda())
        got = pc.paged_attention(qr, cache, t, pos.cuda(), row_starts=rs, window=window,
                                 sinks=sinks).cpu()
        c64 = (ref.dequantize(cache.codes.cpu(), cache.scales.cpu()) if quant
               else cache.cpu().double())
        want, mass, serr = ref.attention(qr.cpu(), c64, tables, pos, starts, window, sinks,
                                         d ** -0.5)
        bound = ref.attention_bound(want, mass, serr, BF16, 200)
        assert ((got.double() - want).abs() <= bound).all()

    step([100, 40], torch.cat([torch.arange(100), torch.arange(40)]).to(torch.int32), 10)
    step([50, 1], torch.cat([torch.arange(100, 150), torch.tensor([40])]).to(torch.int32), 20)
    for i in range(3):
        step([1, 1], torch.tensor([150 + i, 41 + i], dtype=torch.int32), 30 + 5 * i)


@pytest.mark.parametrize("quant", [False, True])
def test_graph_decode_step(dev, quant):
    """One captured step (append, attention) replayed with new positions and tokens, eager work
    and other captured steps between the replays; a second graph shares nothing with it."""
    d, hq, hkv, bs, n = 128, 28, 4, 16, 4000
    tables, nb = _tables([n, 700, 90], bs, 1)
    t = tables.cuda()
    if quant:
        _, _, cache = _quant_cache(nb, hkv, bs, d, 2)
        copy = pc.QuantizedKVCache(cache.codes.clone(), cache.scales.clone())
    else:
        _, cache = _cache(nb, hkv, bs, d, BF16, 2)
        copy = cache.clone()
    k, v, q = (torch.zeros((3, h, d), dtype=BF16, device="cuda") for h in (hkv, hkv, hq))
    pos = torch.tensor([5, 6, 7], dtype=torch.int32).cuda()

    def step(c, outs=(None, None)):
        qr = pc.append_kv_paged(c, k, v, t, pos, rope_base=1e6, query=q)
        return (pc.paged_attention(qr, c, t, pos, out=outs[0]),
                pc.paged_attention(qr, c, t, pos, window=100, sinks=4, out=outs[1]))

    step(copy), step(cache)      # (both caches hold this step's tokens; nothing is captured yet)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        # (outputs of the caller's: memory that a graph allocates serves it for other things, so
        # padding rows could not be seen to stay as they were)
        out = (torch.empty_like(q), torch.empty_like(q))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(cache, out)
        graphs.append((g, out))
    for r in range(4):
        for x, s in ((k, 1), (v, 2), (q, 3)):
            x.copy_(randn(tuple(x.shape), BF16, 100 * r + s).cuda())
        pos.copy_(torch.tensor([n - 1 - r, [699, -1, 3, 250][r], r], dtype=torch.int32).cuda())
        g, out = graphs[r % 2]
        if r == 1:
            for o in out:
                o.fill_(2.0)
        g.replay()
        want = step(copy)
        torch.cuda.synchronize()
        live = (pos >= 0)
        for a, b in zip(out, want):
            assert_bit_exact(a[live], b[live])
        if r == 1:
            assert all((o[1] == 2.0).all() for o in out)
        if quant:
            assert torch.equal(cache.codes, copy.codes) and torch.equal(cache.scales, copy.scales)
        else:
            assert_bit_exact(cache, copy)


def test_other_stream(dev):
    """Calls on a side stream, two at once on two streams, give what the default stream gives."""
    d, hq, hkv, bs, n = 128, 28, 4, 16, 3000
    tables, nb = _tables([n], bs, 1)
    _, cache = _cache(nb, hkv, bs, d, BF16, 2)
    q = randn((1, hq, d), BF16, 3).cuda()
    q2 = randn((130, hq, d), BF16, 4).cuda()
    pos = torch.tensor([n - 1], dtype=torch.int32).cuda()
    pos2 = torch.arange(n - 130, n, dtype=torch.int32).cuda()
    bt = tables[0].cuda()
    want = (pc.paged_attention(q, cache, bt, pos), pc.paged_attention(q2, cache, bt, pos2))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = []
    for s, (x, p) in zip(streams, ((q, pos), (q2, pos2))):
        with torch.cuda.stream(s):
            got.append([pc.paged_attention(x, cache, bt, p) for _ in range(5)])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for x in g:
            assert_bit_exact(x, w)


def test_repeated_calls_are_bit_identical(dev):
    """No atomics, no order of arrival: the same call gives the same bits."""
    d, hq, hkv, bs = 128, 32, 8, 16
    tables, nb = _tables([5000, 300], bs, 1)
    _, _, cache = _quant_cache(nb, hkv, bs, d, 2)
    pos = torch.tensor([4999, 299], dtype=torch.int32).cuda()
    q = randn((2, hq, d), BF16, 3).cuda()
    want = pc.paged_attention(q, cache, tables.cuda(), pos)
    for _ in range(3):
        assert_bit_exact(pc.paged_attention(q, cache, tables.cuda(), pos), want)


# ---- 4-bit blocks of any scale ----------------------------------------------------------------

def _any_scale_case(dtype, d, rows, byte, bad_at, minus_page):
    """Blocks of scale byte `byte` with random codes in K and V of the positions `bad_at`, and in
    page 0, which is no page of the request (a table entry of -1 in the middle)."""
    hq, hkv, bs, n, window, sinks = 14, 2, 16, 150, 20, 3
    tables = torch.randperm(10, generator=gen(1))[None].to(torch.int32) + 1
    if minus_page:
        tables[0, (n - 10) // bs] = -1
    codes, scales, _ = _quant_cache(11, hkv, bs, d, 2)
    x = torch.tensor(bad_at)
    page, slot = tables[0].long()[x // bs], x % bs
    scales[page, :, :, slot] = byte
    scales[0] = byte
    cache = pc.QuantizedKVCache(codes.cuda(), scales.cuda())
    pos = torch.arange(n - rows, n, dtype=torch.int32)
    q = randn((rows, hq, d), dtype, 4)
    want, mass, serr = ref.attention(q, ref.dequantize(codes, scales), tables, pos, [0, rows], window,
                                     sinks, .125)
    got = pc.paged_attention(q.cuda(), cache, tables[0].cuda(), pos.cuda(), window=window,
                             sinks=sinks, scale=.125).cpu()
    clean = ~torch.tensor([[bool(ref.visible(int(p), torch.tensor([b]), window, sinks))
                            for b in bad_at] for p in pos]).any(1)
    assert clean.any()
    assert got[clean].isfinite().all()
    bound = ref.attention_bound(want, mass, serr, dtype, n)
    assert ((got.double() - want).abs()[clean] <= bound[clean]).all()


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 3, 90])
@pytest.mark.parametrize("byte", [142, 143, 200, 252, 253, 254, 255])
def test_masked_4bit_blocks_of_any_scale(dev, dtype, d, rows, byte):
    """Blocks that a row does not see may have any scale byte, those whose values are infinite in
    the query's type (fp16 from 143 on, bf16 from 253 on) among them."""
    n = 150
    _any_scale_case(dtype, d, rows, byte, [n, n + 3], False)
    _any_scale_case(dtype, d, rows, byte, [n + 1], True)
    if rows < 90:
        _any_scale_case(dtype, d, rows, byte, [5, 70], False)
    if rows > 1:
        _any_scale_case(dtype, d, rows, byte, [n - 1], False)


@pytest.mark.parametrize("dtype,byte", [(BF16, 253), (BF16, 254), (FP16, 143)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 60])
def test_seen_4bit_values_beside_infinite_ones(dev, dtype, byte, d, rows):
    """A block of V that holds an infinity in the query's type (one column of each block here), seen
    whole or in part: an infinity of its sign there, the sums of the other columns as ever."""
    hq, hkv, bs, n = 8, 2, 16, 200
    tables, nb = _tables([n], bs, 1)
    codes, scales, _ = _quant_cache(nb, hkv, bs, d, 2)
    small = 1 if byte == 254 else 5                      # up to 2^126, 3 * 2^126, 3 * 2^16
    for at in (40, n - 3 - rows):
        c, s = codes.clone(), scales.clone()
        page, slot = int(tables[0, at // bs]), at % bs
        v = torch.randint(0, small + 1, (hkv, d), generator=gen(3)) + 8 * (torch.arange(d) % 2)
        v[:, 3::32], v[:, 8::32] = 7, 15                 # 6 and -6 times the power
        c[page, 1, :, slot] = (v[:, 0::2] | v[:, 1::2] << 4).to(torch.uint8)
        s[page, 1, :, slot] = byte
        q = randn((rows, hq, d), dtype, 4) * .25
        pos = torch.arange(n - rows, n, dtype=torch.int32)
        want, mass, serr = ref.attention(q, ref.dequantize(c, s), tables, pos, [0, rows], None, 0,
                                         .01)
        got = pc.paged_attention(q.cuda(), pc.QuantizedKVCache(c.cuda(), s.cuda()), tables[0].cuda(),
                                 pos.cuda(), scale=.01).cpu()
        assert (got[..., 3::32] == math.inf).all() and (got[..., 8::32] == -math.inf).all()
        rest = [i for i in range(d) if i % 32 not in (3, 8)]
        bound = ref.attention_bound(want, mass, serr, dtype, n)
        assert ((got.double() - want).abs() <= bound)[..., rest].all()


@pytest.mark.parametrize("dtype,quant", FORMATS)
@pytest.mark.parametrize("d", [64, 96])
@pytest.mark.parametrize("rows", [1, 60])
def test_seen_nan_score_before_finite_ones(dev, dtype, quant, d, rows):
    """A first key whose score is NaN, alone in the first key tile that a row sees (later tiles hold
    finite scores): the row is NaN, whichever kernel takes the call."""
    hq, hkv, bs, n = 14, 2, 16, 700
    tables, nb = _tables([n], bs, 1)
    pos = torch.arange(n - rows, n, dtype=torch.int32)
    if quant:
        codes, scales, _ = _quant_cache(nb, hkv, bs, d, 2)
        scales[int(tables[0, 0]), 0, :, 0] = 255
        cache = pc.QuantizedKVCache(codes.cuda(), scales.cuda())
    else:
        host, _ = _cache(nb, hkv, bs, d, dtype, 2)
        host[int(tables[0, 0]), 0, :, 0] = math.nan
        cache = host.cuda()
    q = randn((rows, hq, d), dtype, 4).cuda()
    for window, sinks, nan in ((20, 1, True), (300, 3, True), (20, 0, False)):
        got = pc.paged_attention(q, cache, tables[0].cuda(), pos.cuda(), window=window, sinks=sinks)
        assert got.isnan().all() if nan else got.isfinite().all()


@pytest.mark.parametrize("plane", [0, 1])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", [1, 60])
def test_largest_4bit_values_of_fp16_queries(dev, plane, d, rows):
    """fp16 queries over 4-bit pages take values below 2^18: every fourth key's K or V has blocks of
    scale byte 142 (up to 6 * 2^15), and rows see them in whole tiles and in part."""
    hq, hkv, bs, n = 8, 2, 16, 200
    tables, nb = _tables([n], bs, 1)
    codes, scales, _ = _quant_cache(nb, hkv, bs, d, 2)
    at = torch.arange(0, n, 4)
    scales[tables[0].long()[at // bs], plane, :, at % bs] = 142
    cache = pc.QuantizedKVCache(codes.cuda(), scales.cuda())
    pos = torch.arange(n - rows, n, dtype=torch.int32)
    q = randn((rows, hq, d), FP16, 4)
    scale = 1e-6 if plane == 0 else .01
    for window, sinks in ((None, 0), (90, 4)):
        want, mass, serr = ref.attention(q, ref.dequantize(codes, scales), tables, pos, [0, rows],
                                         window, sinks, scale)
        assert want.abs().amax() < 65504 * (1 if plane else 2 ** -8)
        got = pc.paged_attention(q.cuda(), cache, tables[0].cuda(), pos.cuda(), window=window,
                                 sinks=sinks, scale=scale).cpu()
        bound = ref.attention_bound(want, mass, serr, FP16, n)
        assert ((got.double() - want).abs() <= bound).all()


# ---- prompt chunks whose keys are split ---------------------------------------------------------

HALVES = [f for f in FORMATS if f[0] != FP32]


def _planned_bytes(rows, requests, hq, hkv, d, bs, width, window, sinks, dtype, quant):
    from semblend_amd import _lib

    return _lib.size_query("sb_paged_attention_workspace_size", rows, requests, int(requests > 1),
                           rows, hq, hkv, d, bs, width, window or 0, sinks, _lib.SB_DTYPE[dtype],
                           _lib.SB_DTYPE_MXFP4 if quant else _lib.SB_DTYPE[dtype])


@pytest.mark.parametrize("dtype,quant", HALVES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window,sinks", [(None, 0), (2900, 33)])
def test_chunk_over_a_long_context_is_split(dev, dtype, quant, d, window, sinks):
    """Chunks on the rows kernel, of one row tile and of three (the last not full), whose key lists
    are cut into several parts: alone, beside a single token, and with padding between their rows."""
    hq, hkv, bs, n = 4, 2, 16, 6000
    for rows in (70, 300):
        tiles = -(-rows * 2 // 256)
        part = 4 * (d + 2) * 256 * tiles * hkv    # bytes of one part of every row tile
        planned = _planned_bytes(rows, 1, hq, hkv, d, bs, n // bs, window, sinks, dtype, quant)
        assert planned >= 3 * part, (planned, part)
        pos = torch.arange(n - rows, n, dtype=torch.int32)
        _attend_case(dtype, d, hq, hkv, bs, [n], [rows], window, sinks, quant, positions=pos)
        pos = torch.cat([pos, torch.tensor([2], dtype=torch.int32)])
        pos[3:9], pos[rows - 1] = -1, -1
        _attend_case(dtype, d, hq, hkv, bs, [n, 3], [rows, 1], window, sinks, quant, positions=pos)


@pytest.mark.parametrize("dtype,quant", HALVES)
@pytest.mark.parametrize("hq,hkv", [(8, 2), (28, 4)])
def test_chunks_among_many_single_rows(dev, dtype, quant, hq, hkv):
    """One or several long chunks in a batch of many requests, most of them of one row or none: the
    chunks' keys are split."""
    d, bs, n = 64, 16, 140
    lens = [1 + (37 * i) % 400 for i in range(n)]
    for chunks in ({100: 90}, {0: 33, 70: 150, 71: 64, 139: 20}):
        rows = [chunks.get(i, 0 if i % 5 == 0 else 1) for i in range(n)]
        ctx = [4000 + i if i in chunks else x for i, x in enumerate(lens)]
        assert _planned_bytes(sum(rows), n, hq, hkv, d, bs, 259, None, 0, dtype, quant) > 0
        _attend_case(dtype, d, hq, hkv, bs, ctx, rows, None, 0, quant, width=259)
        _attend_case(dtype, d, hq, hkv, bs, ctx, rows, 3000, 5, quant, width=259)


@pytest.mark.parametrize("dtype,quant", HALVES)
def test_tables_much_wider_than_the_contexts(dev, dtype, quant):
    """A captured step's tables are as wide as the longest context it may meet: chunks and single
    tokens of a few hundred keys under tables of 128K."""
    for d, rows in ((64, [90]), (128, [90]), (64, [90, 1, 40]), (128, [1, 300, 1])):
        _attend_case(dtype, d, 14, 2, 16, [700, 40, 333][:len(rows)] if rows[0] > 1 else
                     [30, 700, 64], rows, None, 0, quant, width=8192)


@pytest.mark.parametrize("quant", [False, True])
def test_graph_of_a_mixed_batch(dev, quant):
    """A captured call of a chunk beside single tokens (both kernels and their merges), replayed with
    other positions, rows per request and pages, eager calls between the replays."""
    d, hq, hkv, bs, n = 128, 28, 4, 16, 4000
    tables, nb = _tables([n, n, 90], bs, 1)
    cache = _quant_cache(nb, hkv, bs, d, 2)[2] if quant else _cache(nb, hkv, bs, d, BF16, 2)[1]
    num = 90
    t = tables.cuda()
    pos = torch.zeros(num, dtype=torch.int32, device="cuda")
    starts = torch.zeros(4, dtype=torch.int32, device="cuda")
    q = torch.zeros((num, hq, d), dtype=BF16, device="cuda")
    out = torch.empty_like(q)

    def step(o):
        return pc.paged_attention(q, cache, t, pos, starts, window=3500, sinks=4, out=o)

    step(torch.empty_like(q))
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(out)
    for r, rows in enumerate(([80, 1, 1], [1, 60, 20], [0, 88, 2], [80, 1, 1])):
        starts.copy_(torch.tensor(_starts(rows), dtype=torch.int32).cuda())
        ctx = [n - 7 * r, n - 9, 90 - r]
        p = torch.cat([torch.arange(c - x, c) for c, x in zip(ctx, rows)])
        pos.copy_(torch.cat([p, torch.full((num - len(p),), 5)]).to(torch.int32).cuda())
        q.copy_(randn((num, hq, d), BF16, 10 + r).cuda())
        t.copy_(tables.flip(1) if r == 2 else tables)
        out.fill_(2.0)
        want = torch.full_like(q, 2.0)
        g.replay()
        step(want)
        torch.cuda.synchronize()
        assert_bit_exact(out, want)
        assert (out[len(p):] == 2.0).all()
        assert not (out[:len(p)] == 2.0).all(-1).any()


@pytest.mark.parametrize("dtype,quant", HALVES)
def test_repeated_mixed_calls_are_bit_identical(dev, dtype, quant):
    d, hq, hkv, bs, rows = 128, 32, 8, 16, [200, 1, 1, 30]
    tables, nb = _tables([5000, 300, 4000, 90], bs, 1)
    cache = _quant_cache(nb, hkv, bs, d, 2)[2] if quant else _cache(nb, hkv, bs, d, dtype, 2)[1]
    starts = torch.tensor(_starts(rows), dtype=torch.int32).cuda()
    pos = torch.cat([torch.arange(n - r, n) for n, r in zip([5000, 300, 4000, 90], rows)])
    q = randn((sum(rows), hq, d), dtype, 3).cuda()
    args = (q, cache, tables.cuda(), pos.int().cuda(), starts)
    want = pc.paged_attention(*args)
    for _ in range(3):
        assert_bit_exact(pc.paged_attention(*args), want)


@pytest.mark.parametrize("dtype,quant", HALVES)
@pytest.mark.parametrize("chunks", [2, 6, 20, 70])
def test_row_tiles_share_the_partials(dev, dtype, quant, chunks):
    """Requests of a few more rows than the decode kernel takes: many row tiles that are little
    filled, so that the parts of each go from the most to one; empty requests between them."""
    d, hq, hkv, bs = 64, 28, 4, 16
    rows = [3 + i % 2 if i % 2 else 0 for i in range(2 * chunks)]
    lens = [1500 + 31 * i for i in range(2 * chunks)]
    for window, sinks in ((None, 0), (700, 70)):
        _attend_case(dtype, d, hq, hkv, bs, lens, rows, window, sinks, quant, width=400)


@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_append_4bit_largest_rotated_keys(dev, dtype):
    """Rotated keys of the dtype's largest values, whose pairs' sums may pass fp32: codes and scale
    bytes are the 64-bit quantiser's; blocks with an infinity or a NaN beside them are NaN."""
    bs, heads, d, num, base = 16, 2, 64, 70, 1e4
    tables, nb = _tables([num], bs, 1)
    codes, scales, cache = _quant_cache(nb, heads, bs, d, 2)
    top = torch.finfo(dtype).max
    k = (torch.rand((num, heads, d), generator=gen(3)) * 2 - 1).double()
    k[:, :, ::5] = k[:, :, ::5].sign()                  # +-max, in some blocks beside small values
    k[40:, 0, 1::2] *= 1e-3
    k = (k * top).to(dtype)
    k[50, 0, 3], k[51, 1, 40], k[52, 0, 63] = math.inf, math.nan, -math.inf
    v = randn((num, heads, d), dtype, 4)
    at = torch.arange(num, dtype=torch.int32)
    pc.append_kv_paged(cache, k.cuda(), v.cuda(), tables[0].cuda(), at.cuda(), rope_base=base)
    page, slot = tables[0].long()[at.long() // bs], at.long() % bs
    c, s = ref.quantize(ref.rotate(k, at, base))
    assert (s == 255).any(-1).sum() == 3 and (dtype == FP16 or (s == 253).sum() > 100)
    assert torch.equal(cache.scales.cpu()[page, 0, :, slot].long(), s)
    assert torch.equal(cache.codes.cpu()[page, 0, :, slot],
                       (c[..., 0::2] | c[..., 1::2] << 4).to(torch.uint8))
