"""Products with 4-bit weights at the ends of the range that they are documented for: |x| below 2^116, scales
below 2^122, sums of |x| |scale| of an output below 2^120."""

from __future__ import annotations

import pytest
import torch

from semblend_amd.quantized import QuantizedLinear, quantized_linear

from . import quantized_forms as forms
from . import quantized_reference as ref
from .helpers import gen

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
SIZES = [(1, 17, 384, 128), (5, 17, 2176, 128), (2, 17, 448, 64), (2083, 34, 384, 128), (4461, 69, 384, 128),
         (1934, 1696, 2112, 64), (315, 248, 27264, 128), (306, 203, 25024, 32)]


def _run(x, codes, scales, z):
    got = quantized_linear(x.cuda(), QuantizedLinear(codes.cuda(), scales.cuda(), z.cuda())).cpu()
    assert got.isfinite().all()
    at = torch.arange(codes.shape[0])[:150]
    ref.check(got[:, at], *forms.linear(x, codes[at], scales[at], z[at]))


@pytest.mark.parametrize("m,n,k,group", SIZES)
def test_large_inputs(dev, m, n, k, group):
    """The largest inputs, all of one sign or of one a group, under the largest codes: the kernels' sums are of
    x (16 + c), up to 31 |x| each."""
    g = gen(1)
    codes = torch.randint(13, 16, (n, k), generator=g, dtype=torch.uint8)
    z = torch.randint(0, 16, (n, k // group), generator=g, dtype=torch.uint8)
    codes[0], z[0] = 15, 0
    x = (1.0 - torch.rand((m, k), generator=g) / 16).to(BF16).double().clamp(max=1 - 2.0 ** -8) * 2.0 ** 116
    sign = torch.randint(0, 2, (m, k // group), generator=g).double() * 2 - 1
    sign[0] = 1
    x = (x * sign.repeat_interleave(group, 1)).to(BF16)
    scales = torch.full(z.shape, 2.0 ** 4 / 2.0 ** (k - 1).bit_length(), dtype=BF16)
    assert float(x.double().abs().max()) < 2.0 ** 116
    assert float((x.double().abs() @ scales.double().repeat_interleave(group, 1).t()).max()) < 2.0 ** 120
    _run(x, codes, scales, z)


@pytest.mark.parametrize("m,n,k,group", SIZES)
def test_large_scales(dev, m, n, k, group):
    """The largest scales, on inputs that keep the sums in range."""
    codes, scales, z = ref.make(n, k, group, BF16, 2)
    scales = (scales.double() * 2.0 ** 126).clamp(max=(2 - 2.0 ** -7) * 2.0 ** 121).to(BF16)
    x = (torch.randn((m, k), generator=gen(3), dtype=torch.float64) * 2.0 ** -24).to(BF16)
    assert 2.0 ** 121 < float(scales.max()) < 2.0 ** 122
    _run(x, codes, scales, z)
