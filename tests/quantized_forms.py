"""Sizes that reach every form of a product with 4-bit weights (semblend_amd/csrc/sb_w4_plan.h), each with
rows, features and inputs that the form's tiles do not divide. The CPU tests hold the sizes to their forms,
so that a change of the choice cannot leave a form without its test."""

from __future__ import annotations

import torch

from . import quantized_reference as ref
from .paged_reference import half_step

BF16, FP16 = torch.bfloat16, torch.float16

# (rows, features, inputs, group): few rows, form "R J groups of a tile, waves, codes read once".
ROWS = {
    (5, 17, 2176, 128): "16 1 1 16 0", (5, 17, 384, 128): "16 1 1 8 0", (22, 17, 2112, 64): "16 1 2 16 0",
    (5, 17, 448, 64): "16 1 2 8 0", (9, 17, 2112, 32): "16 1 4 16 0", (8, 17, 416, 32): "16 1 4 8 0",
    (1368, 36, 384, 128): "16 2 1 8 0", (1505, 33, 448, 64): "16 2 2 8 0", (1069, 51, 416, 32): "16 2 4 8 0",
    (1361, 85, 384, 128): "16 3 1 8 0", (1764, 65, 448, 64): "16 3 2 8 0", (1766, 66, 416, 32): "16 3 4 8 0",
    (397, 611, 384, 128): "16 4 1 8 0", (1353, 181, 448, 64): "16 4 2 8 0", (1345, 189, 448, 32): "16 4 4 8 0",
    (2083, 34, 384, 128): "32 1 1 8 0", (2135, 34, 448, 64): "32 1 2 8 0", (2054, 37, 416, 32): "32 1 4 8 0",
    (2090, 49, 384, 128): "32 2 1 8 0", (2839, 49, 448, 64): "32 2 2 8 0", (2213, 50, 416, 32): "32 2 4 8 0",
    (3064, 81, 384, 128): "32 3 1 8 0", (3404, 67, 448, 64): "32 3 2 8 0", (3340, 68, 448, 32): "32 3 4 8 0",
    (2731, 97, 384, 128): "32 4 1 8 0", (3028, 98, 448, 64): "32 4 2 8 0", (2916, 97, 416, 32): "32 4 4 8 0",
    (1, 17, 2176, 128): "4 1 1 16 0", (1, 17, 384, 128): "4 1 1 8 0", (3, 17, 2112, 64): "4 1 2 16 0",
    (2, 17, 448, 64): "4 1 2 8 0", (1, 17, 2080, 32): "4 1 4 16 0", (3, 17, 416, 32): "4 1 4 8 0",
    (2, 4114, 384, 128): "4 2 1 8 0", (1, 4104, 448, 64): "4 2 2 8 0", (3, 4134, 416, 32): "4 2 4 8 0",
    (4290, 34, 384, 128): "64 1 1 8 0", (4322, 33, 448, 64): "64 1 2 8 0", (4114, 34, 480, 32): "64 1 4 8 0",
    (4461, 69, 384, 128): "64 2 1 8 0", (4133, 65, 448, 64): "64 2 2 8 0", (4402, 68, 416, 32): "64 2 4 8 0",
    (5753, 66, 384, 128): "64 3 1 8 0", (5637, 66, 448, 64): "64 3 2 8 0", (4135, 99, 416, 32): "64 3 4 8 0",
    (5469, 97, 384, 128): "64 4 1 7 0", (5628, 97, 448, 64): "64 4 2 7 0", (4100, 146, 416, 32): "64 4 4 7 0",
}

# The same with codes of 192 MiB and more.
ROWS_ONCE = {
    (5, 56541, 7168, 128): "16 2 1 8 1", (9, 55384, 7232, 64): "16 2 2 8 1", (8, 37034, 10816, 32): "16 2 4 8 1",
    (5, 82851, 4864, 128): "16 3 1 8 1", (5, 17493, 22976, 64): "16 3 2 8 1", (8, 65735, 6112, 32): "16 3 4 8 1",
    (6, 95672, 4224, 128): "16 4 1 8 1", (5, 58659, 6848, 64): "16 4 2 8 1", (6, 131812, 2976, 32): "16 4 4 8 1",
    (1, 15882, 25344, 128): "4 2 1 8 1", (3, 82926, 4800, 64): "4 2 2 8 1", (2, 160533, 2464, 32): "4 2 4 8 1",
}

# Many rows, (..., type): form "groups of a tile, slices, steps of a slice, steps of sums". Features in
# whole vectors of 8 and not; slices that hold steps of codes and of sums, and sums alone.
TILES = {
    (315, 248, 27264, 128, BF16): "1 32 7 7", (460, 135, 24960, 128, BF16): "1 29 7 7",
    (355, 224, 28480, 64, BF16): "2 30 8 14", (419, 154, 25920, 64, BF16): "2 31 7 13",
    (275, 240, 26400, 32, BF16): "4 30 8 26", (306, 203, 25024, 32, BF16): "4 32 7 25",
    (3100, 968, 4352, 128, BF16): "1 1 36 2", (5043, 599, 4352, 128, BF16): "1 1 36 2",
    (1934, 1696, 2112, 64, BF16): "2 1 19 2", (5587, 533, 2368, 64, BF16): "2 1 21 2",
    (2826, 1216, 2016, 32, BF16): "4 1 18 2", (5782, 926, 1056, 32, BF16): "4 1 11 2",
    (154, 144, 18176, 128, FP16): "1 29 5 0", (140, 141, 16128, 128, FP16): "1 32 4 0",
    (158, 152, 17856, 64, FP16): "2 28 5 0", (137, 135, 21824, 64, FP16): "2 29 6 0",
    (152, 192, 18592, 32, FP16): "4 30 5 0", (147, 147, 15904, 32, FP16): "4 32 4 0",
    (5341, 392, 384, 128, FP16): "1 1 3 0", (4690, 413, 384, 128, FP16): "1 1 3 0",
    (3193, 816, 448, 64, FP16): "2 1 4 0", (4868, 438, 448, 64, FP16): "2 1 4 0",
    (3804, 752, 448, 32, FP16): "4 1 4 0", (4417, 502, 416, 32, FP16): "4 1 4 0",
    # prompts of the widths that the benchmark names
    (2458, 4608, 3584, 128, BF16): "1 1 29 1", (2458, 4608, 3584, 128, FP16): "1 1 28 0",
}

# One of each kind for what is asked of all of them (strides, NaN, captures, streams): whole with vectors of
# features, whole with packed differences, slices with single features and sums, slices without sums.
KINDS = [(1934, 1696, 2112, 64, BF16), (3193, 816, 448, 64, FP16), (306, 203, 25024, 32, BF16),
         (315, 248, 27264, 128, BF16), (140, 141, 16128, 128, FP16)]


def linear(x, codes, scales, zeros, bias=None):
    """(y in 64 bits, the bound on a kernel's error): fp32 sums of terms x (16 + c) and x (16 + zero) (fp16:
    128, at most 143 |x|), scaled. A term goes through the additions of its group (128 at most), of the
    groups, of sixteen waves or of 32 slices, the offset's and the bias's; each is off by half a step of the
    sums so far, which are the terms' magnitudes at most: 2^-24, and twice that where the matrix cores cut
    off instead of rounding. bf16's offsets as a product add 2^-24 of each (the part left out)."""
    y, _ = ref.linear(x, codes, scales, zeros, bias)
    group = codes.shape[1] // scales.shape[1]
    most = 2 * (143 if x.dtype == FP16 else 31)
    size = most * x.double().abs() @ scales.double().abs().repeat_interleave(group, 1).t()
    if bias is not None:
        size = size + bias.double().abs()
    step = min(group, 128)
    adds = step + -(-codes.shape[1] // step) + 32 + 4
    u = half_step(x.dtype)
    return y, u * y.abs() + (1 + u) * adds * 2.0 ** -23 * size + torch.finfo(x.dtype).tiny
