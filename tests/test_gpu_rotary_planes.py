"""Scatters whose workgroups take rows of K alone or of V alone (these evaluate no sines): 8192 pairs and more
with eight heads and more, where a workgroup takes eight rows of eight pairs."""

from __future__ import annotations

import pytest
import torch

from semblend_amd import rope_correction as rc
from semblend_amd.rotary import RotaryEmbedding

from . import rotary_reference as ref
from .helpers import assert_bit_exact, gen

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


@pytest.mark.parametrize("layers,heads,num", [(1, 8, 9000), (2, 16, 8200), (1, 24, 8192), (3, 12, 8193)])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
def test_planes_of_their_own(dev, dtype, layout, layers, heads, num):
    rot = RotaryEmbedding.from_config(64, 1e6, layout=layout)
    bs = 16
    need = -(-num // bs)
    table = torch.randperm(need + 3, generator=gen(1))[:need].to(torch.int32)
    dpos = torch.randperm(num, generator=gen(2)).to(torch.int32)
    tpos = torch.arange(num, dtype=torch.int32)
    donors = torch.randn((layers, 2, heads, num, 64), generator=torch.Generator("cuda").manual_seed(3),
                         device="cuda").to(dtype)
    caches = torch.zeros((layers, need + 3, 2, heads, bs, 64), dtype=dtype, device="cuda")
    # (what LDS holds before: rows turned by other angles)
    rc.rope_correct_scatter_paged_layers(list(caches), list(donors), table.cuda(), dpos.cuda(), tpos.cuda(),
                                         rotary=RotaryEmbedding.from_config(64, 1e2, layout=layout))
    rc.rope_correct_scatter_paged_layers(list(caches), list(donors), table.cuda(), dpos.cuda(), tpos.cuda(),
                                         rotary=rot)
    page, slot = table.long()[tpos.long() // bs], tpos.long() % bs
    got = caches.cpu()[:, page, :, :, slot]                            # [T, L, 2, H, D]
    src = donors.cpu()[:, :, :, dpos.long()].permute(3, 0, 1, 2, 4)    # [T, L, 2, H, D]
    assert_bit_exact(got[:, :, 1].contiguous(), src[:, :, 1].contiguous())
    want, norm = ref.turn(src[:, :, 0].flatten(1, 2), tpos - dpos, rot.inv_freq, layout)
    moved = (tpos != dpos)[:, None, None]
    ref.check(got[:, :, 0].flatten(1, 2), want, norm * moved)
