"""Rotary positions in 64 bits on the CPU, from the definition, with the bound the tests hold the
kernels to."""

from __future__ import annotations

import torch

from .paged_reference import half_step


def pairs_of(n: int, layout: str):
    """(first, second) elements of the n / 2 pairs of the first n elements."""
    first = torch.arange(n // 2) * (2 if layout == "interleaved" else 1)
    return first, first + (1 if layout == "interleaved" else n // 2)


def turn(x: torch.Tensor, pos: torch.Tensor, freq: torch.Tensor, layout: str, factor: float = 1.0):
    """(x [T, H, D] turned by pos [T] in 64 bits, the norm of each element's pair (0: not turned))."""
    a, b = pairs_of(2 * freq.shape[0], layout)
    th = (pos.double()[:, None] * freq.double())[:, None]
    c, s = th.cos() * factor, th.sin() * factor
    out, norm = x.double().clone(), torch.zeros(x.shape, dtype=torch.float64)
    xa, xb = out[..., a].clone(), out[..., b].clone()
    out[..., a], out[..., b] = xa * c - xb * s, xa * s + xb * c
    norm[..., a] = norm[..., b] = torch.sqrt(xa ** 2 + xb ** 2) * factor
    return out, norm


def check(got: torch.Tensor, want: torch.Tensor, norm: torch.Tensor) -> None:
    """One rounding to the dtype; 16-bit rows are turned in fp32: cosine and sine, two products and a
    sum, each off by 2^-24 of the pair's norm at most (fp32 rows the same with 2^-53, kept loosely at
    2^-50). Elements that are not turned keep their bits."""
    dtype = got.dtype
    noise = 2.0 ** -50 if dtype == torch.float32 else 2.0 ** -22
    err = (got.double() - want).abs()
    tol = half_step(dtype) * want.abs() + noise * norm * (1 + half_step(dtype)) + \
        (norm > 0) * torch.finfo(dtype).tiny
    assert (err <= tol).all(), f"{float((err / tol.clamp_min(1e-300)).max()):.3f} of the bound"
