"""Products with 4-bit weights against 64 bits (tests/quantized_reference.py)."""

from __future__ import annotations

import math

import pytest
import torch

from semblend_amd.quantized import QuantizedLinear, quantized_linear

from . import quantized_reference as ref
from .helpers import assert_bit_exact, randn

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def _case(m, n, k, group, dtype, zeros=True, bias=True, seed=0, scale_dtype=None):
    x, codes, scales, z = ref.inputs(m, n, k, group, dtype, seed, zeros, scale_dtype)
    b = randn((n,), dtype, seed + 2) if bias else None
    w = QuantizedLinear(*_cuda(codes, scales, z))
    got = quantized_linear(x.cuda(), w, bias=None if b is None else b.cuda()).cpu()
    ref.check(got, *ref.linear(x, codes, scales, z, b))
    return got


@pytest.mark.parametrize("m", [1, 2, 5, 16, 17, 31, 32, 33, 48, 64, 65, 100, 128, 129, 257])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_rows(dev, dtype, group, m):
    _case(m, 272, 640, group, dtype, seed=m)


@pytest.mark.parametrize("n", [1, 8, 15, 16, 17, 33, 100, 1000])
@pytest.mark.parametrize("m", [1, 19, 70, 150])
def test_features(dev, m, n):
    _case(m, n, 256, 128, BF16, bias=n % 2 == 0, seed=n)


@pytest.mark.parametrize("k,group", [(32, 32), (64, 64), (64, 32), (96, 32), (96, 96), (160, 32), (192, 64),
                                     (192, 96), (224, 224), (320, 64), (384, 384), (1056, 32), (1600, 64),
                                     (4736, 128), (4736, 4736), (18944, 64)])
@pytest.mark.parametrize("m", [1, 16, 40, 140])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_inputs_and_groups(dev, dtype, m, k, group):
    """Tiles of inputs that are not whole, groups smaller and larger than a tile, whole rows."""
    _case(m, 80, k, group, dtype, seed=k)


@pytest.mark.parametrize("m,n,k,group,dtype", [(1, 4608, 3584, 128, BF16), (8, 5000, 3584, 128, FP16),
                                               (64, 6144, 4096, 32, BF16), (614, 1152, 896, 64, FP16),
                                               (2458, 1040, 896, 128, BF16), (1, 40000, 512, 128, BF16)])
@pytest.mark.parametrize("zeros", [True, False])
def test_model_sizes(dev, m, n, k, group, dtype, zeros):
    _case(m, n, k, group, dtype, zeros=zeros, bias=not zeros)


@pytest.mark.parametrize("m", [3, 200])
def test_scales_of_the_other_type(dev, m):
    _case(m, 100, 256, 64, BF16, scale_dtype=FP16)
    _case(m, 100, 256, 64, FP16, scale_dtype=BF16)


@pytest.mark.parametrize("m", [1, 20, 130])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_weights_one_by_one(dev, dtype, m):
    """Rows of the unit matrix give the weights themselves: each rounded once, nothing from its
    neighbours; dequantize gives the same."""
    n, k = 48, 384
    codes, scales, z = ref.make(n, k, 64, dtype, 1)
    w = QuantizedLinear(*_cuda(codes, scales, z))
    want = ref.weight(codes, scales, z).to(dtype)
    eye = torch.eye(k, dtype=dtype, device="cuda")
    got = torch.cat([quantized_linear(eye[a:a + m], w) for a in range(0, k, m)]).t().contiguous()
    assert torch.equal(got.cpu(), want)
    assert torch.equal(w.dequantize(dtype).cpu(), want)
    assert torch.equal(w.dequantize(FP32).cpu().double(), ref.weight(codes, scales, z))


@pytest.mark.parametrize("m", [2, 33, 140])
def test_strides_shapes_and_out(dev, m):
    """Rows of a wider tensor, odd addresses, other strides, leading dimensions, rows of one stride in
    `out` (what lies between them as it was)."""
    n, k = 100, 256
    x, codes, scales, z = ref.inputs(m, n, k, 128, BF16, 3)
    b = randn((n,), BF16, 4).cuda()
    w = QuantizedLinear(*_cuda(codes, scales, z))
    x = x.cuda()
    want = quantized_linear(x, w, bias=b)
    wide = torch.zeros((m, k + 24), dtype=BF16, device="cuda")
    wide[:, 8:8 + k] = x
    odd = torch.zeros((m, k + 1), dtype=BF16, device="cuda")
    odd[:, 1:] = x
    for y in (wide[:, 8:8 + k], odd[:, 1:], x.t().contiguous().t(), x.view(m, 1, k), x[None]):
        got = quantized_linear(y, w, bias=b)
        assert got.shape == (*y.shape[:-1], n)
        assert_bit_exact(got.reshape(m, n).cpu(), want.cpu())
    target = torch.full((m, n + 5), 7.0, dtype=BF16, device="cuda")
    out = target[:, 3:3 + n]
    assert quantized_linear(x, w, bias=b, out=out) is out
    assert_bit_exact(out.contiguous().cpu(), want.cpu())
    assert (target[:, :3] == 7).all() and (target[:, 3 + n:] == 7).all()
    twice = torch.zeros(2 * n, dtype=BF16, device="cuda")
    twice[::2] = b
    assert_bit_exact(quantized_linear(x, w, bias=twice[::2]).cpu(), want.cpu())
    one = quantized_linear(x[0], w, bias=b)
    assert one.shape == (n,)
    assert_bit_exact(one.cpu(), quantized_linear(x[:1], w, bias=b)[0].cpu())
    assert quantized_linear(x[:0], w).shape == (0, n)
    same = x[:1].expand(m, k)
    assert_bit_exact(quantized_linear(same, w).cpu(), quantized_linear(same.contiguous(), w).cpu())


def test_packing_from_strided_inputs(dev):
    n, k = 40, 320
    codes, scales, z = ref.make(n, k, 32, FP16, 5)
    x = randn((7, k), FP16, 6).cuda()
    want = quantized_linear(x, QuantizedLinear(*_cuda(codes, scales, z)))
    wide = torch.cat([codes, codes], 1).cuda()[:, :k]
    got = quantized_linear(x, QuantizedLinear(wide, scales.t().contiguous().cuda().t(),
                                              z.t().contiguous().cuda().t()))
    assert_bit_exact(got.cpu(), want.cpu())
    got = quantized_linear(x, QuantizedLinear(codes.t().contiguous().cuda().t(), scales.cuda(), z.cuda()))
    assert_bit_exact(got.cpu(), want.cpu())


@pytest.mark.parametrize("m", [1, 16, 30, 64, 200])
def test_rows_do_not_reach_each_other(dev, m):
    """A row with a NaN or an infinity is NaN; the other rows have the bits they have without it. A
    row's result does not depend on its place or on the others."""
    n, k = 64, 512
    x, codes, scales, z = ref.inputs(m, n, k, 128, BF16, 7)
    w = QuantizedLinear(*_cuda(codes, scales, z))
    clean = quantized_linear(x.cuda(), w).cpu()
    bad = x.clone()
    bad[0, 5] = math.nan
    bad[m // 2, 300] = math.inf
    got = quantized_linear(bad.cuda(), w).cpu()
    rows = torch.ones(m, dtype=torch.bool)
    rows[0] = rows[m // 2] = False
    assert got[~rows].isnan().all()
    assert_bit_exact(got[rows], clean[rows])
    turned = quantized_linear(x.flip(0).cuda(), w).cpu()
    assert_bit_exact(turned.flip(0), clean)


@pytest.mark.parametrize("m", [1, 64, 150])
def test_large_values(dev, m):
    """Values and scales near the end of their ranges, outliers a thousand times the rest, groups of
    scale zero."""
    n, k = 32, 256
    x, codes, scales, z = ref.inputs(m, n, k, 32, BF16, 8)
    scales[:, 2] = 0.0
    x[:, 7] *= 1000.0
    for up in (1.0, 2.0 ** 100, 2.0 ** -100):
        xs = (x.double() * up).to(BF16)
        w = QuantizedLinear(*_cuda(codes, scales, z))
        got = quantized_linear(xs.cuda(), w).cpu()
        err = (got.double() - ref.linear(xs, codes, scales, z)[0]).abs()
        assert (err <= ref.linear(xs, codes, scales, z)[1]).all()
    x16, codes, scales, z = ref.inputs(m, n, k, 32, FP16, 9)
    got = quantized_linear((x16 * 30000).clamp(-65504, 65504).cuda(),
                           QuantizedLinear(*_cuda(codes, scales * 1000, z))).cpu()
    y = ref.linear((x16 * 30000).clamp(-65504, 65504), codes, scales * 1000, z)[0]
    assert (got.isinf() == (y.abs() >= 65520)).all()


@pytest.mark.parametrize("symmetric", [False, True])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_quantize(dev, dtype, symmetric):
    """Every weight within half a step of its own (plus the rounding of the zero point and scale)."""
    w = randn((24, 256), FP32, 1)
    w[3] = 0.0
    w[4] = w[4].abs()
    w = w.to(dtype)
    q = QuantizedLinear.quantize(w.cuda(), group=64, symmetric=symmetric)
    back = q.dequantize(FP32).cpu().double()
    g = w.double().unflatten(1, (-1, 64))
    if symmetric:
        step = g.abs().amax(-1) / 7.5
    else:
        step = (g.amax(-1).clamp(min=0) - g.amin(-1).clamp(max=0)) / 15
    err = (back - w.double()).abs().unflatten(1, (-1, 64))
    # half a step of the code and, at the ends of the range, half of one of the zero point; the
    # scale's own rounding (2^-8) moves an end by 15 * 2^-8 of a step
    assert (err <= step[..., None] * (1.0 + 16 * 2.0 ** -8) + 1e-30).all()
    assert (back[3] == 0).all()
    assert float(err.mean() / step.mean()) < 0.3         # (uniform in half a step: 0.25)


def test_captured(dev):
    """Captured once per kind of launch, replayed with new rows."""
    n, k = 208, 512
    _, codes, scales, z = ref.inputs(1, n, k, 64, BF16, 3)
    w = QuantizedLinear(*_cuda(codes, scales, z))
    for m in (1, 24, 150):
        x = torch.zeros((m, k), dtype=BF16, device="cuda")
        y = torch.empty((m, n), dtype=BF16, device="cuda")
        quantized_linear(x, w, out=y)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            quantized_linear(x, w, out=y)
            z2 = quantized_linear(x, w)
        for seed in (1, 2, 3):
            x.copy_(randn((m, k), BF16, seed))
            want = quantized_linear(x, w)
            y.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert_bit_exact(y.cpu(), want.cpu())
            assert_bit_exact(z2.cpu(), want.cpu())


def test_two_streams(dev):
    """Calls of one weight at the same time on two streams."""
    n, k = 512, 1024
    _, codes, scales, z = ref.inputs(1, n, k, 128, BF16, 3)
    w = QuantizedLinear(*_cuda(codes, scales, z))
    xs = [randn((m, k), BF16, m).cuda() for m in (1, 40, 300, 64)]
    want = [quantized_linear(x, w).cpu() for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(16):
        with torch.cuda.stream(streams[i % 2]):
            got.append((i % 4, quantized_linear(xs[i % 4], w)))
    torch.cuda.synchronize()
    for i, y in got:
        assert_bit_exact(y.cpu(), want[i])


def test_gradient_is_refused(dev):
    _, codes, scales, z = ref.inputs(1, 32, 64, 32, BF16, 3)
    w = QuantizedLinear(*_cuda(codes, scales, z))
    x = randn((3, 64), BF16, 1).cuda().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        quantized_linear(x, w).sum().backward()
    b = randn((32,), BF16, 1).cuda().requires_grad_()
    with pytest.raises(RuntimeError, match="no backward pass"):
        quantized_linear(x.detach(), w, bias=b).sum().backward()
    with torch.no_grad():
        assert not quantized_linear(x, w).requires_grad


def test_codes_out_of_range_are_refused(dev):
    codes = torch.full((16, 64), 3, dtype=torch.uint8, device="cuda")
    scales = torch.ones((16, 2), dtype=BF16, device="cuda")
    codes[3, 5] = 16
    with pytest.raises(ValueError, match="codes"):
        QuantizedLinear(codes, scales)
    codes[3, 5] = 15
    with pytest.raises(ValueError, match="zeros"):
        QuantizedLinear(codes, scales, codes[:, :2] + 13)
    with pytest.raises(ValueError, match="finite"):
        QuantizedLinear.quantize(torch.full((4, 64), math.inf, device="cuda"), group=32)
    with pytest.raises(ValueError, match="range"):
        QuantizedLinear.quantize(torch.full((4, 64), 1e30, device="cuda"), group=32, scale_dtype=FP16)


def test_more_rows_than_a_grid_of_the_few_rows_kernel(dev):
    """4.2 million rows of few features and inputs."""
    m = 65535 * 64 + 200
    codes, scales, zeros = ref.make(16, 32, 32, BF16, 1)
    w = QuantizedLinear(codes.cuda(), scales.cuda(), zeros.cuda())
    x = randn((1024, 32), BF16, 2)
    y = quantized_linear(x.cuda().repeat(m // 1024 + 1, 1)[:m], w)
    ref.check(y[:1024].cpu(), *ref.linear(x, codes, scales, zeros))
    last = m // 1024 * 1024
    assert torch.equal(y[:last].view(-1, 1024, 16), y[:1024].expand(last // 1024, 1024, 16))
    assert torch.equal(y[last:], y[:m - last])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n", [9000, 16300])
@pytest.mark.parametrize("m", [9, 20, 50, 70])
def test_features_of_a_workgroup(dev, m, n, group, dtype):
    """Feature counts at which a workgroup of few rows takes three and four tiles of them, the last
    workgroup not all of its own."""
    codes, scales, zeros = ref.make(n, 384, group, dtype, 1)
    x = randn((m, 384), dtype, 2)
    w = QuantizedLinear(codes.cuda(), scales.cuda(), zeros.cuda())
    ref.check(quantized_linear(x.cuda(), w).cpu(), *ref.linear(x, codes, scales, zeros))


@pytest.mark.parametrize("m,n,k", [(2, 131072, 4096), (16, 131072, 4096), (16, 9000, 45056)])
def test_weights_past_the_caches(dev, m, n, k):
    """Codes of 200 MB and more; some of the features against 64 bits."""
    codes, scales, zeros = ref.make(n, k, 128, FP16, 1)
    x = randn((m, k), FP16, 2)
    y = quantized_linear(x.cuda(), QuantizedLinear(codes.cuda(), scales.cuda(), zeros.cuda())).cpu()
    at = torch.cat([torch.arange(0, n, 97), torch.arange(n - 70, n)])
    ref.check(y[:, at], *ref.linear(x, codes[at], scales[at], zeros[at]))
