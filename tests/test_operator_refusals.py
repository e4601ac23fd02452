"""Calls that the operators around and of the MoE block refuse with -1 before any launch (CPU: shapes are
checked before any pointer is used)."""
import ctypes

import pytest

import dramamoe as D

P = 0x1000  # an aligned address that is never dereferenced


def expect(name, base, cases):
    f = D.lib().raw(name)
    for change in cases:
        args = list(base)
        for pos, bad in change.items():
            args[pos] = bad
        assert f(*args) == -1, (name, change)


# (x, ldx, pw, gate, gate_mode, ldg, cs, bscale, xscale, nw, eps, xo, ldo, hn, ldh, rows, h, st)
NORM_TAIL = [P, 64, P, P, 2, 64, P, 1.0, 1.0, P, 1e-6, P, 64, P, 64, 2, 64, None]


@pytest.mark.parametrize("name", ["dr_block_norm", "dr_block_norm_bf16"])
def test_block_norm_refusals(name):
    base = [P, 64] + NORM_TAIL
    expect(name, base, [
        {18: 0}, {18: 16385, 1: 20000, 3: 20000, 7: 20000, 14: 20000, 16: 20000}, {17: -1},
        {1: 63}, {3: 63}, {7: 63}, {14: 63}, {16: 63}, {1: -64},
        {6: 3}, {6: -1}, {5: None}, {5: None, 6: 1}, {11: None}, {13: None, 15: None}, {0: None, 2: None},
    ])


def test_block_norm_of_no_rows_does_nothing():
    for name, head in (("dr_block_norm", [P, 64]), ("dr_block_norm_bf16", [P, 64]), ("dr_moe_combine_norm", [P, P, P, P, P, 8])):
        args = head + NORM_TAIL
        args[-3] = 0
        assert D.lib().raw(name)(*args) == 0


def test_combine_norm_refusals():
    base = [P, P, P, P, P, 8] + NORM_TAIL
    expect("dr_moe_combine_norm", base, [
        {5: 0}, {5: 33}, {0: None}, {1: None}, {2: None}, {3: None}, {22: 0}, {22: 16385}, {21: -1}, {7: 63}, {18: 63},
        {10: 7}, {15: None}, {17: None, 19: None},
    ])


MOE = ["dr_moe_layer_rows", "dr_moe_layer_rows_bf16s", "dr_moe_layer_rows_fp8", "dr_moe_layer_rows_fp8_bf16s"]


@pytest.mark.parametrize("name", MOE)
def test_moe_layer_rows_refusals(name):
    # router, gu_q, gu_s, d_q, d_s, sgu_q, sgu_s, sd_q, sd_s, x, res, idx, wts, sgate, ws, y, rows, e, h, i, topk, st
    base = [P] * 16 + [4, 16, 2048, 512, 8, None]
    bad = [{16: 0}, {16: 65}, {17: 0}, {17: 257}, {17: 7}, {18: 0}, {18: 2050}, {18: 64}, {18: 8320}, {19: 0}, {19: 500}, {19: 64},
           {19: 8320}, {20: 0}, {20: 33, 17: 64}, {20: 17}]
    bad += [{q: None} for q in (0, 1, 2, 3, 4, 9, 11, 12, 13, 14, 15)] + [{q: None} for q in (5, 6, 7, 8)]
    bad += [{q: P + 8} for q in (0, 1, 2, 3, 4, 5, 7, 9, 10, 14, 15)]
    expect(name, base, bad)


def test_moe_layer_rows_ws():
    f = D.lib().cdll.dr_moe_layer_rows_ws
    assert f(1, 256, 2048, 512, 8) >= 1024 + 9 * (512 * 6 + 2048 * 4)
    assert f(64, 256, 2048, 512, 8) > f(1, 256, 2048, 512, 8)
    for bad in ((0, 256, 2048, 512, 8), (65, 256, 2048, 512, 8), (4, 256, 2050, 512, 8), (4, 4, 2048, 512, 8), (4, 256, 2048, 500, 8)):
        assert f(*bad) == 0


@pytest.mark.parametrize("name", ["dr_gemm_q8_lora", "dr_gemm_q8_lora_bf16s"])
def test_gemm_q8_lora_refusals(name):
    # w, s, x, ldx, adapter, la, lb, rank, lscale, adapters, rmax, ws, res, y, ldy, rows, n, k, st
    base = [P, P, P, 256, P, P, P, P, P, 4, 16, P, P, P, 100, 3, 100, 256, None]
    bad = [{15: -1}, {15: (1 << 20) + 1}, {16: 0}, {17: 0}, {17: 64}, {17: 200}, {17: 16512, 3: 16512}, {3: 248}, {3: 260}, {14: 99}, {10: 0},
           {10: 12}, {10: 136}, {9: -1}]
    bad += [{q: None} for q in (0, 1, 2, 5, 6, 7, 8, 11, 13)] + [{q: P + 8} for q in (0, 2, 5, 6, 11)]
    expect(name, base, bad)
    none = list(base)
    none[15] = 0
    assert D.lib().raw(name)(*none) == 0


def test_gemm_q8_lora_ws():
    f = D.lib().cdll.dr_gemm_q8_lora_ws
    assert f(5, 100, 256, 16) >= 256 + 5 * 16 * 4
    for bad in ((-1, 100, 256, 16), (5, 0, 256, 16), (5, 100, 200, 16), (5, 100, 256, 12)):
        assert f(*bad) == 0
