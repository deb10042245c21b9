"""The paged-cache operators in 64 bits on the CPU, from their definitions, with the bounds that
the tests hold the kernels to."""

from __future__ import annotations

import math

import torch

GRID = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def half_step(dtype: torch.dtype) -> float:
    """A rounding to dtype is off by at most this much of the value."""
    return torch.finfo(dtype).eps / 2


def rotate(x: torch.Tensor, pos: torch.Tensor, base: float) -> torch.Tensor:
    """x [T, H, D] rotated by pos [T]: interleaved pairs, fp32 frequencies, 64-bit angles."""
    d = x.shape[-1]
    f = 1.0 / (base ** (torch.arange(0, d, 2, dtype=torch.float32) / d))
    th = pos.double()[:, None, None] * f.double()
    e, o = x.double()[..., 0::2], x.double()[..., 1::2]
    return torch.stack([e * th.cos() - o * th.sin(), e * th.sin() + o * th.cos()], -1).flatten(-2)


def quantize(x: torch.Tensor):
    """(codes [..., D] 0..15, scale bytes [..., D / 32]) of x (64 bits), element by element from
    the definition: the smallest e >= -127 with max |x| <= 7 * 2^e, nearest grid value, ties to the
    even code."""
    b = x.double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    bad = ~b.isfinite().all(-1)
    e = torch.full(top.shape, -127.0, dtype=torch.float64)
    for _ in range(254):  # (a plain search: no logarithm to round)
        e = torch.where((top > 7.0 * torch.exp2(e)) & ~bad, e + 1, e)
    y = torch.where(bad[..., None], torch.zeros_like(b), b.abs() / torch.exp2(e)[..., None])
    gap = (y[..., None] - GRID).abs()
    near = gap.amin(-1, keepdim=True)
    # among the nearest (two in a tie) the even code
    rank = torch.arange(8) + 8 * (torch.arange(8) % 2)
    code = torch.where(gap == near, rank, torch.full_like(rank, 99)).argmin(-1)
    code = code + 8 * torch.signbit(b).long()
    code = torch.where(bad[..., None], torch.zeros_like(code), code)
    scale = torch.where(bad, torch.full_like(e, 255.0), e + 127)
    return code.flatten(-2), scale.long()


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Values [..., D] (64 bits) of packed bytes [..., D / 2] and scale bytes [..., D / 32]."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = torch.where(c >= 8, -GRID[c & 7], GRID[c & 7]).unflatten(-1, (-1, 32))
    s = torch.exp2(scales.double() - 127)
    s = torch.where(scales.long() == 255, torch.full_like(s, math.nan), s)
    return (v * s[..., None]).flatten(-2)


def visible(pos, keys: torch.Tensor, window, sinks: int) -> torch.Tensor:
    m = keys <= pos
    if window is not None:
        m &= (keys > pos - window) | (keys < sinks)
    return m


def attention(q, cache64, tables, positions, starts, window, sinks, scale):
    """q [R, Hq, D]; cache64 [NB, 2, Hkv, bs, D] (64 bits). Returns (out, weight, score_err) per
    row and head: the result (NaN where a padding row), sum_j w_j |v_j|, and the bound on the error of
    an fp32 score."""
    if torch.cuda.is_available():  # (64-bit elementwise operations and sums: the same there)
        q, cache64, tables = q.cuda(), cache64.cuda(), tables.cuda()
    r, hq, d = q.shape
    nb, _, hkv, bs, _ = cache64.shape
    out = torch.full((r, hq, d), math.nan, dtype=torch.float64, device=q.device)
    mass = torch.zeros((r, hq, d), dtype=torch.float64, device=q.device)
    serr = torch.zeros((r, hq, 1), dtype=torch.float64, device=q.device)
    positions = positions.tolist()
    for i in range(tables.shape[0]):
        lo, hi = (starts[i], starts[i + 1]) if starts is not None else (i, min(i + 1, r))
        for row in range(lo, hi):
            p = positions[row]
            if p < 0:
                continue
            keys = torch.arange(min(p + 1, tables.shape[1] * bs), device=q.device)
            page = tables[i].long()[keys // bs]
            seen = visible(p, keys, window, sinks) & (page >= 0) & (page < nb)
            keys, page = keys[seen], page[seen]
            if keys.numel() == 0:
                out[row] = 0.0
                continue
            kv = cache64[page, :, :, keys % bs].repeat_interleave(hq // hkv, 2)  # [n, 2, Hq, D]
            qq = q[row].double()
            s = (kv[:, 0] * qq).sum(-1) * scale                 # [n, Hq]
            w = torch.softmax(s, 0)[..., None]
            out[row] = (w * kv[:, 1]).sum(0)
            mass[row] = (w * kv[:, 1].abs()).sum(0)
            # d products and sums in fp32, the scale and exp2's argument
            serr[row, :, 0] = ((kv[:, 0] * qq).abs().sum(-1).amax(0) * abs(scale)
                               * (d + 4) * 2.0 ** -24)
    return out.cpu(), mass.cpu(), serr.cpu()


def attention_bound(out, mass, serr, dtype: torch.dtype, keys: int) -> torch.Tensor:
    """How far a kernel may be off: its fp32 scores move a weight by a relative serr each way and
    its sums of up to `keys` terms round n times (2^-24 each, with exp2's own 2^-22); 16-bit
    kernels round every weight once (the sum takes the rounded ones: each side by half a step),
    and the output once more."""
    out = out.abs()
    u = half_step(dtype)
    rel = 2 * serr + (keys + 8) * 2.0 ** -23
    bound = mass * rel + u * out
    if dtype != torch.float32:
        bound = bound + u * (mass + out) * (1 + 2 * u)
    return bound + torch.finfo(dtype).tiny
