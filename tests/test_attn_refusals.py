"""Calls that the operators between an attention block's projections refuse with -1 before any launch (CPU)."""
import pytest

import dramamoe as D
from test_operator_refusals import P, expect

BAD_SIZE = [-1, (1 << 20) + 1]


@pytest.mark.parametrize("name", ["dr_rope", "dr_rope_bf16"])
def test_rope_refusals(name):
    # x, ldx, hsx, nw, ldn, eps, pos, freq, mscale, layout, y, ldy, yb, ldb, rows, heads, d, rot, st
    base = [P, 256, 64, P, 64, 1e-6, P, P, 1.0, 0, P, 256, P, 256, 3, 4, 64, 32, None]
    bad = [{14: -1}, {14: (1 << 23) + 1}, {15: 0}, {15: 4097, 1: 1 << 20, 11: 1 << 20, 13: 1 << 20}, {16: 0}, {16: 513, 2: 600, 1: 4096, 4: 600, 11: 4096, 13: 4096}, {17: 31}, {17: -2}, {17: 66},
           {9: 2}, {9: -1}, {0: None}, {10: None, 12: None}, {6: None}, {7: None}, {2: 63}, {2: -64}, {1: 255}, {11: 255}, {13: 255}, {4: 63}, {4: -1}]
    expect(name, base, bad)
    none = list(base)
    none[14] = 0
    assert D.lib().raw(name)(*none) == 0


@pytest.mark.parametrize("name", ["dr_kv8_append", "dr_kv8_append_bf16"])
def test_append_refusals(name):
    # k, ldk, v, ldv, start, len, table, maxp, kq, ks, vq, vs, pages, rows, seqs, hkv, d, st
    base = [P, 256, P, 256, P, P, P, 8, P, P, P, P, 9, 5, 2, 2, 128, None]
    bad = [{13: b} for b in BAD_SIZE] + [{14: b} for b in BAD_SIZE] + [{15: 0}, {15: 1025, 1: 1 << 20, 3: 1 << 20}, {16: 0}, {16: 8}, {16: 120}, {16: 272, 1: 1024, 3: 1024}, {7: 0},
           {7: 1 << 25}, {12: 0}, {1: 252}, {3: 252}, {1: 258}, {3: 258}, {1: -256}]
    bad += [{q: None} for q in (0, 2, 4, 5, 6, 8, 9, 10, 11)] + [{q: P + 8} for q in (0, 2, 8, 10)]
    expect(name, base, bad)
    for at in (13, 14):
        none = list(base)
        none[at] = 0
        assert D.lib().raw(name)(*none) == 0


def test_read_refusals():
    # start, len, table, maxp, kq, ks, vq, vs, pages, k, ldk, v, ldv, rows, seqs, hkv, d, st
    base = [P, P, P, 8, P, P, P, P, 9, P, 256, P, 256, 5, 2, 2, 128, None]
    bad = [{13: b} for b in BAD_SIZE] + [{14: b} for b in BAD_SIZE] + [{15: 0}, {16: 24}, {3: 0}, {8: 0}, {10: 252}, {12: 258}]
    bad += [{q: None} for q in (0, 1, 2, 4, 5, 6, 7, 9, 11)] + [{q: P + 8} for q in (4, 6, 9, 11)]
    expect("dr_kv8_read", base, bad)
    none = list(base)
    none[13] = 0
    assert D.lib().raw("dr_kv8_read")(*none) == 0


def test_attention_refusals():
    # q, ldq, start, len, table, maxp, kq, ks, vq, vs, pages, scale, gate, ldg, hsg, ws, y, ldy, rows, seqs, max_rows, max_len, hq, hkv, d, st
    base = [P, 512, P, P, P, 8, P, P, P, P, 9, 0.1, P, 512, 128, P, P, 512, 5, 2, 4, 300, 4, 2, 128, None]
    bad = [{18: b} for b in BAD_SIZE] + [{19: b} for b in BAD_SIZE] + [{20: -1}, {21: -1}, {22: 0}, {22: 3}, {22: 1026, 23: 1, 1: 1 << 20, 13: 1 << 20, 17: 1 << 20}, {23: 0}, {24: 100},
           {24: 272, 1: 2048, 13: 2048, 14: 272, 17: 2048}, {5: 0}, {5: 1 << 25}, {10: 0}, {1: 504}, {1: 516}, {17: 508}, {17: 514}, {13: 508}, {14: 124}, {14: 130, 13: 1024},
           {13: 514}, {11: float("inf")}, {11: float("-inf")}, {11: float("nan")}, {18: 1 << 20, 19: 1 << 20, 20: 1, 22: 8, 23: 8, 1: 1024, 13: 1024, 17: 1024}]
    bad += [{q: None} for q in (0, 2, 3, 4, 6, 7, 8, 9, 15, 16)] + [{q: P + 8} for q in (0, 6, 8, 12, 15)] + [{16: P + 4}]
    expect("dr_attn_kv8", base, bad)
    for at in (18, 19, 20):
        none = list(base)
        none[at] = 0
        assert D.lib().raw("dr_attn_kv8")(*none) == 0


def test_attention_ws():
    f = D.lib().cdll.dr_attn_kv8_ws
    assert f(1, 1, 1, 60000, 16, 2, 256) >= 2 * 16 * 258 * 4 and f(4096, 1, 4096, 4096, 16, 2, 128) > 0 and f(0, 0, 0, 0, 1, 1, 16) > 0
    for bad in ((-1, 1, 1, 1, 4, 2, 64), (1, -1, 1, 1, 4, 2, 64), (1, 1, -1, 1, 4, 2, 64), (1, 1, 1, -1, 4, 2, 64), (1, 1, 1, 1, 3, 2, 64), (1, 1, 1, 1, 4, 2, 72), (1 << 20, 1 << 20, 1, 1, 8, 8, 128)):
        assert f(*bad) == 0
