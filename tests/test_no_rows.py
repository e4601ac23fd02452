"""Calls without rows or sequences between an attention block's projections do nothing, whatever their buffers: an empty tensor has no address (CPU)."""
import pytest

import dramamoe as D
from test_attn_refusals import P


@pytest.mark.parametrize("name", ["dr_rope", "dr_rope_bf16"])
@pytest.mark.parametrize("rot", [0, 32])
def test_rope(name, rot):
    # x, ldx, hsx, nw, ldn, eps, pos, freq, mscale, layout, y, ldy, yb, ldb, rows, heads, d, rot, st
    f = D.lib().raw(name)
    assert f(None, 256, 64, None, 0, 1e-6, None, None, 1.0, 0, None, 256, None, 256, 0, 4, 64, rot, None) == 0
    assert f(None, 256, 64, P, 64, 1e-6, None, P, 1.0, 1, None, 256, None, 256, 0, 4, 64, rot, None) == 0
    # sizes and strides are looked at all the same
    assert f(None, 255, 64, None, 0, 1e-6, None, None, 1.0, 0, None, 256, None, 256, 0, 4, 64, rot, None) == -1
    assert f(None, 256, 64, None, 0, 1e-6, None, None, 1.0, 0, None, 256, None, 256, 0, 4, 64, 31, None) == -1


@pytest.mark.parametrize("rows,seqs", [(0, 2), (0, 0), (5, 0)])
def test_cache_and_attention(rows, seqs):
    lib = D.lib()
    cache = (None, 8, None, None, None, None, 9)
    for name in ("dr_kv8_append", "dr_kv8_append_bf16"):
        assert lib.raw(name)(None, 256, None, 256, None, None, *cache, rows, seqs, 2, 128, None) == 0
    assert lib.raw("dr_kv8_read")(None, None, *cache, None, 256, None, 256, rows, seqs, 2, 128, None) == 0
    assert lib.raw("dr_attn_kv8")(None, 512, None, None, *cache, 0.1, None, 0, 0, None, None, 512, rows, seqs, 4, 300, 4, 2, 128, None) == 0
