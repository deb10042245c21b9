"""Outputs of rotary rows in any order of tokens and heads, and their refusal where rows share elements."""

from __future__ import annotations

import pytest
import torch

from semblend_amd import paged_cache as pc
from semblend_amd.rotary import RotaryEmbedding, apply_rotary

from .helpers import assert_bit_exact, randn

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


@pytest.mark.parametrize("strides", [(256, 64), (64, 192), (300, 70), (128, 320), (256, 640), (64, 64 * 3 + 2)])
def test_orders_of_rows(dev, strides):
    """Heads within tokens, tokens within heads, and orders in which neither lies within the other."""
    tokens, heads, d = 3, 4, 64
    rot = RotaryEmbedding.from_config(d, 1e4)
    pos = torch.tensor([3, 700, -5], dtype=torch.int32).cuda()
    x = randn((tokens, heads, d), BF16, 1).cuda()
    want = apply_rotary(x, pos, rot)
    room = torch.full((4096,), 7.0, dtype=BF16, device="cuda")
    out, out_k = room.as_strided((tokens, heads, d), (*strides, 1), 8), torch.empty_like(x)
    assert apply_rotary(x, pos, rot, key=x, query_out=out, key_out=out_k)[0] is out
    assert_bit_exact(out.cpu().contiguous(), want.cpu())
    assert_bit_exact(out_k.cpu(), want.cpu())
    out.fill_(7.0)
    assert (room == 7.0).all()


@pytest.mark.parametrize("strides", [(64, 64), (64, 128), (200, 32), (0, 64), (256, 0)])
def test_rows_that_share_elements_are_refused(dev, strides):
    tokens, heads, d = 3, 4, 64
    rot = RotaryEmbedding.from_config(d, 1e4)
    pos = torch.arange(tokens, dtype=torch.int32).cuda()
    x = randn((tokens, heads, d), BF16, 1).cuda()
    out = torch.zeros(4096, dtype=BF16, device="cuda").as_strided((tokens, heads, d), (*strides, 1))
    cache = torch.zeros((4, 2, heads, 16, d), dtype=BF16, device="cuda")
    table = torch.arange(4, dtype=torch.int32).cuda()
    for call in (lambda: apply_rotary(x, pos, rot, query_out=out),
                 lambda: apply_rotary(x, pos, rot, key=x, key_out=out),
                 lambda: pc.append_kv_paged(cache, x, x, table, pos, rotary=rot, query=x, query_out=out),
                 lambda: pc.append_kv_paged(cache, x, x, table, pos, rope_base=1e4, query=x, query_out=out)):
        with pytest.raises(RuntimeError, match="overlap"):
            call()
    assert (out == 0).all() and (cache == 0).all()
