"""Every form of a product with 4-bit weights against 64 bits, at sizes held to their forms on the CPU
(tests/test_quantized_forms.py); strides, values that are not finite, captures and streams where many rows
run."""

from __future__ import annotations

import math

import pytest
import torch

from semblend_amd import _lib
from semblend_amd.quantized import QuantizedLinear, quantized_linear

from . import quantized_forms as forms
from . import quantized_reference as ref
from .helpers import assert_bit_exact, gen, randn

pytestmark = pytest.mark.gpu

BF16, FP16 = torch.bfloat16, torch.float16


def _weight(n, k, group, dtype, seed, zeros=True):
    codes, scales, z = ref.make(n, k, group, dtype, seed, zeros)
    w = QuantizedLinear(codes.cuda(), scales.cuda(), None if z is None else z.cuda())
    return codes, scales, z, w


def _some(n, most=200):
    """Features to look at: all, or some with the first and last tiles."""
    if n <= most:
        return torch.arange(n)
    at = torch.cat([torch.arange(40), torch.randperm(n, generator=gen(1))[:most - 110], torch.arange(n - 70, n)])
    return at.unique()


def _check(got, x, codes, scales, z, bias=None):
    at = _some(codes.shape[0])
    ref.check(got.cpu()[:, at], *forms.linear(x, codes[at], scales[at], None if z is None else z[at],
                                              None if bias is None else bias[at]))


def _launches(call):
    """(result, launches of the few-rows kernel, of the tiles, of the sums, of the merge)."""
    torch.cuda.synchronize()
    _lib.kernel_timing(True)
    try:
        out = call()
        torch.cuda.synchronize()
        return out, [_lib.kernel_time(k)[1] for k in ("w4_rows", "w4_tiles", "w4_sums", "w4_merge")]
    finally:
        _lib.kernel_timing(False)


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("size", forms.ROWS, ids=lambda s: "x".join(map(str, s)))
def test_few_rows(dev, size, dtype):
    m, n, k, group = size
    codes, scales, z, w = _weight(n, k, group, dtype, 1)
    x, b = randn((m, k), dtype, 2), randn((n,), dtype, 3)
    got, ran = _launches(lambda: quantized_linear(x.cuda(), w, bias=b.cuda()))
    assert ran == [1, 0, 0, 0]
    _check(got, x, codes, scales, z, b)


@pytest.mark.parametrize("size", forms.ROWS_ONCE, ids=lambda s: "x".join(map(str, s)))
def test_few_rows_codes_read_once(dev, size):
    """(Inputs made on the device: 400 million codes.)"""
    m, n, k, group = size
    g = torch.Generator("cuda").manual_seed(1)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8, device="cuda")
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8, device="cuda")
    for dtype in (BF16, FP16):
        scales = ((torch.rand(z.shape, generator=g, device="cuda") + 0.5) / 64).to(dtype)
        w = QuantizedLinear(codes, scales, z)
        x = randn((m, k), dtype, 2)
        got, ran = _launches(lambda: quantized_linear(x.cuda(), w))
        assert ran == [1, 0, 0, 0]
        at = _some(n, 400).cuda()
        ref.check(got[:, at].cpu(), *forms.linear(x, codes[at].cpu(), scales[at].cpu(), z[at].cpu()))


@pytest.mark.parametrize("zeros", [True, False])
@pytest.mark.parametrize("size", forms.TILES, ids=lambda s: "x".join(map(str, s[:4])) + str(s[4])[6:])
def test_many_rows(dev, size, zeros):
    m, n, k, group, dtype = size
    codes, scales, z, w = _weight(n, k, group, dtype, 1, zeros)
    x = randn((m, k), dtype, 2)
    b = None if zeros else randn((n,), dtype, 3)
    got, ran = _launches(lambda: quantized_linear(x.cuda(), w, bias=None if b is None else b.cuda()))
    split = int(forms.TILES[size].split()[1]) > 1
    assert ran == [0, 1, int(dtype is BF16), int(split)]
    _check(got, x, codes, scales, z, b)
    if m * n * k < 2 ** 33:
        assert_bit_exact(quantized_linear(x.cuda(), w, bias=None if b is None else b.cuda()).cpu(), got.cpu())


@pytest.mark.parametrize("dtype,other", [(BF16, FP16), (FP16, BF16)])
def test_many_rows_scales_of_the_other_type(dev, dtype, other):
    for m, n, k, group, dt in forms.KINDS:
        if dt is not dtype:
            continue
        codes, scales, z, w = _weight(n, k, group, other, 4)
        x = randn((m, k), dtype, 5)
        _check(quantized_linear(x.cuda(), w), x, codes, scales, z)


@pytest.mark.parametrize("size", forms.KINDS, ids=lambda s: "x".join(map(str, s[:4])))
def test_many_rows_strides_and_out(dev, size):
    """Rows of a wider tensor, an odd address, leading dimensions; rows of one stride in `out` at any
    alignment, what lies between them and around them as it was."""
    m, n, k, group, dtype = size
    _, _, _, w = _weight(n, k, group, dtype, 3)
    x, b = randn((m, k), dtype, 4).cuda(), randn((n,), dtype, 5).cuda()
    want = quantized_linear(x, w, bias=b)
    wide = torch.zeros((m, k + 24), dtype=dtype, device="cuda")
    wide[:, 8:8 + k] = x
    odd = torch.zeros((m, k + 1), dtype=dtype, device="cuda")
    odd[:, 1:] = x
    for y in (wide[:, 8:8 + k], odd[:, 1:], x.view(m, 1, k)):
        got = quantized_linear(y, w, bias=b)
        assert got.shape == (*y.shape[:-1], n)
        assert_bit_exact(got.reshape(m, n).cpu(), want.cpu())
    for first, more in ((3, 5), (8, 16), (0, 8)):
        target = torch.full((m + 2, n + first + more), 7.0, dtype=dtype, device="cuda")
        out = target[1:1 + m, first:first + n]
        assert quantized_linear(x, w, bias=b, out=out) is out
        assert_bit_exact(out.contiguous().cpu(), want.cpu())
        target[1:1 + m, first:first + n] = 7.0
        assert (target == 7.0).all()
    same = x[:1].expand(m, k)
    assert_bit_exact(quantized_linear(same, w).cpu(), quantized_linear(same.contiguous(), w).cpu())


@pytest.mark.parametrize("size", forms.KINDS, ids=lambda s: "x".join(map(str, s[:4])))
def test_many_rows_do_not_reach_each_other(dev, size):
    """A row with a NaN or an infinity is NaN or infinite; the others have the bits they have without it,
    and those of any other place."""
    m, n, k, group, dtype = size
    _, _, _, w = _weight(n, k, group, dtype, 7)
    x = randn((m, k), dtype, 8)
    clean = quantized_linear(x.cuda(), w).cpu()
    bad = x.clone()
    hit = {0: math.nan, m // 2: math.inf, m - 1: -math.inf, 130: math.nan}
    for i, v in hit.items():
        bad[i, (37 * i) % k] = v
    got = quantized_linear(bad.cuda(), w).cpu()
    rows = torch.ones(m, dtype=torch.bool)
    rows[list(hit)] = False
    assert not got[~rows].isfinite().any()
    assert_bit_exact(got[rows], clean[rows])
    turned = quantized_linear(x.flip(0).cuda(), w).cpu()
    assert_bit_exact(turned.flip(0), clean)


@pytest.mark.parametrize("size", [s for s in forms.KINDS if s[4] is BF16], ids=lambda s: "x".join(map(str, s[:4])))
def test_many_rows_large_values(dev, size):
    """Outliers a thousand times the rest, groups of scale zero, rows far up and down the range."""
    m, n, k, group, dtype = size
    codes, scales, z = ref.make(n, k, group, dtype, 8)
    scales[:, 1] = 0.0
    w = QuantizedLinear(codes.cuda(), scales.cuda(), z.cuda())
    x = randn((m, k), dtype, 9)
    x[:, 7] *= 1000.0
    for up in (2.0 ** 100, 2.0 ** -100):
        xs = (x.double() * up).to(dtype)
        _check(quantized_linear(xs.cuda(), w), xs, codes, scales, z)


@pytest.mark.parametrize("size", forms.KINDS, ids=lambda s: "x".join(map(str, s[:4])))
def test_many_rows_captured(dev, size):
    """Captured, replayed with new rows; two graphs of the same weight in turn."""
    m, n, k, group, dtype = size
    _, _, _, w = _weight(n, k, group, dtype, 3)
    xs = [torch.zeros((m, k), dtype=dtype, device="cuda") for _ in range(2)]
    quantized_linear(xs[0], w)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for x in xs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(quantized_linear(x, w))
    for seed in (1, 2, 3):
        for i, x in enumerate(xs):
            x.copy_(randn((m, k), dtype, 10 * seed + i))
        want = [quantized_linear(x, w) for x in xs]
        for o in outs:
            o.fill_(3.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert_bit_exact(a.cpu(), b.cpu())


def test_many_rows_on_two_streams(dev):
    """Calls of one weight at the same time on two streams, whole tiles and slices."""
    cases = []
    for m, n, k, group, dtype in forms.KINDS:
        w = _weight(n, k, group, dtype, 3)[3]
        x = randn((m, k), dtype, 4).cuda()
        cases.append((x, w, quantized_linear(x, w).cpu()))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(20):
        x, w, want = cases[i // 2 % len(cases)]
        with torch.cuda.stream(streams[i % 2]):
            got.append((quantized_linear(x, w), want))
    torch.cuda.synchronize()
    for y, want in got:
        assert_bit_exact(y.cpu(), want)
