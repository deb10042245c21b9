"""Products with 4-bit weights in 64 bits, from the definition, with the bound the tests hold the
kernels to."""

from __future__ import annotations

import torch

from .helpers import gen, randn
from .paged_reference import half_step


def make(n: int, k: int, group: int, dtype: torch.dtype, seed: int, zeros: bool = True):
    """(codes, scales, zeros or None): every code and zero point, scales over a few powers of two."""
    g = gen(seed)
    codes = torch.randint(0, 16, (n, k), generator=g, dtype=torch.uint8)
    s = torch.rand((n, k // group), generator=g) + 0.5
    s = s * torch.exp2(torch.randint(-8, -4, s.shape, generator=g).float())
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    return codes, s.to(dtype), z


def weight(codes, scales, zeros) -> torch.Tensor:
    group = codes.shape[1] // scales.shape[1]
    z = torch.full(scales.shape, 8.0, dtype=torch.float64) if zeros is None else zeros.double()
    w = codes.double().unflatten(1, (-1, group)) - z[..., None]
    return (w * scales.double()[..., None]).flatten(1)


def linear(x, codes, scales, zeros, bias=None):
    """(y in 64 bits, the bound on a kernel's error). Its fp32 sums are of terms x (16 + c) and
    x (16 + zero), at most 31 |x| each before the scale: over a group, over the groups and over the
    parts of a split (16 of them at most), each addition off by 2^-23 of the terms added at most; the
    bias adds one. One rounding to the type."""
    w = weight(codes, scales, zeros)
    group = codes.shape[1] // scales.shape[1]
    x64 = x.double()
    size = 62 * x64.abs() @ scales.double().abs().repeat_interleave(group, 1).t()
    y = x64 @ w.t()
    if bias is not None:
        y, size = y + bias.double(), size + bias.double().abs()
    adds = min(group, 128) + -(-codes.shape[1] // min(group, 128)) + 16 + 2
    u = half_step(x.dtype)
    return y, u * y.abs() + (1 + u) * adds * 2.0 ** -23 * size + torch.finfo(x.dtype).tiny


def check(got: torch.Tensor, y: torch.Tensor, bound: torch.Tensor) -> None:
    err = (got.double() - y).abs()
    assert (err <= bound).all(), f"{float((err / bound).max()):.3f} of the bound"
    # The bound's sums are the worst ones; sums whose roundings are independent are off by about
    # sqrt(k) 2^-24 * 31 |x| s, under a thirtieth of an fp16 rounding of y: where there are enough
    # outputs, the whole error is that of the one rounding.
    if got.numel() >= 4096:
        rounding = (y.to(got.dtype).double() - y).pow(2).mean().sqrt()
        assert float(err.pow(2).mean().sqrt()) <= 1.05 * float(rounding)


def inputs(m, n, k, group, dtype, seed, zeros=True, scale_dtype=None):
    codes, scales, z = make(n, k, group, scale_dtype or dtype, seed, zeros)
    return randn((m, k), dtype, seed + 1), codes, scales, z
