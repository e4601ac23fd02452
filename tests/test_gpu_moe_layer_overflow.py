"""dr_moe_layer_rows* where products or activations leave the range of fp32: a row's outputs are the infinities, the NaN and the
numbers that the definition gives, and the other rows keep their bits.

The definition in 64 bits, the activation rounded to fp32 (beyond 3.4e38 an infinity): an output is sum over picks and the
shared expert of w_k sum_j W[n, j] act[j], in IEEE arithmetic: infinity times a weight of zero is NaN, infinities of both signs add up
to NaN.  Outputs that are numbers: the bounds of test_gpu_moe_layer_rows.py."""
import numpy as np
import pytest

import synth
import test_gpu_moe_layer_rows as M
from helpers import host

pytestmark = pytest.mark.gpu


def nibble(L, name, n, k, q):
    """Nibble k of rows n of every expert."""
    b = L[name][:, n, k // 2]
    L[name][:, n, k // 2] = (b & 0xF0 | q) if k % 2 == 0 else (b & 0x0F | q << 4)


def pair(L, name, n, group, scale, low):
    """Scale and min of rows n of every expert."""
    for p, v in ((0, scale), (1, low)):
        L[name][:, n, group, p] = synth.enc(np.float32([v]), L["sc_kind"])


def only_unit(lay, unit, big):
    """Input `big` counts, with a weight of one, in gate and up of activation `unit` alone, and not for the router."""
    L, i, h = lay.L, lay.i, lay.h
    every, those = slice(None), [unit, i + unit]
    L["router"][:, big] = 0
    if lay.kind == "q4":
        nibble(L, "gu_q", every, big, 0)
        pair(L, "gu_s", every, big // 64, 2.0 ** -9, 0.0)
        pair(L, "gu_s", those, big // 64, 0.0, 1.0)
    else:
        L["gu_q"][:, :, big] = 0
        L["gu_q"][:, those, big] = 0x38  # one
        L["gu_s"][:, :, big // 128] = synth.enc(np.float32([1]), L["sc_kind"])
    if lay.shared:
        L["sgu_q"][:, big] = 0


def definition(lay, x, res, idx, w, sg):
    """y in 64 bits with fp32 activations, from the routing that the call reports."""
    xf = x.double().cpu().numpy()
    y = res.double().cpu().numpy().copy()

    def mlp(v, gu, dn):
        z = v @ gu.T
        with np.errstate(over="ignore", invalid="ignore"):
            act = z[:, :lay.i] / (1 + np.exp(-z[:, :lay.i])) * z[:, lay.i:]
            act = act.astype(np.float32).astype(np.float64)
            out = np.empty((len(v), lay.h))
            for r in range(len(v)):  # elementwise: a matrix product may reorder infinities
                out[r] = (dn * act[r]).sum(1)
        return out

    with np.errstate(invalid="ignore"):
        for j in sorted(set(idx.ravel().tolist())):
            rr, kk = np.nonzero(idx == j)
            y[rr] += w[rr, kk][:, None] * mlp(xf[rr], lay.weights("gu_q", "gu_s", j)[0], lay.weights("d_q", "d_s", j)[0])
        if lay.shared:
            s = 1 / (1 + np.exp(-sg.astype(np.float64)))
            y += s[:, None] * mlp(xf, lay.shared_weights("sgu_q", "sgu_s")[0], lay.shared_weights("sd_q", "sd_s")[0])
    return y


CASES = [  # kind, fmt, rows, e, h, i, topk, shared
    ("q4", "ref", 1, 4, 256, 128, 1, False), ("q4", "cfg", 1, 6, 384, 256, 3, True), ("q4", "ref", 2, 4, 256, 384, 1, True),
    ("q4", "cfg", 21, 5, 640, 256, 2, True), ("q4", "ref", 64, 3, 256, 2688, 1, False), ("q4", "cfg", 1, 4, 128, 8192, 3, False),
    ("fp8", "cfg", 1, 4, 256, 128, 1, True), ("fp8", "ref", 21, 5, 384, 256, 2, False),
]


@pytest.mark.parametrize("kind,fmt,rows,e,h,i,topk,shared", CASES)
def test_activation_beyond_fp32(kind, fmt, rows, e, h, i, topk, shared):
    """One activation of every third row is silu(1e22) 1e22, an infinity: each output takes its weight's sign, NaN for a weight of zero
    or for experts that disagree."""
    import torch

    lay = M.Layer(rows * 31 + h, kind, fmt, e, h, i, shared)
    unit, big = i - 3, h - 7
    only_unit(lay, unit, big)
    # outputs whose weight for that activation is zero
    if kind == "q4":
        nibble(lay.L, "d_q", slice(0, 40, 5), unit, 0)
        pair(lay.L, "d_s", slice(0, 40, 5), unit // 64, 2.0 ** -9, 0.0)
    else:
        lay.L["d_q"][:, 0:40:5, unit] = 0
    lay.put()
    torch.manual_seed(rows)
    x, res = torch.randn(rows, h, device="cuda").to(torch.bfloat16), torch.randn(rows, h, device="cuda")
    ws = M.workspace(rows, e, h, i, topk)
    x[:, big] = 0
    clean = lay.call(x, res, rows, topk, ws)
    hot = list(range(0, rows, 3))
    x[hot, big] = 1e22
    o = lay.call(x, res, rows, topk, ws)
    again = lay.call(x, res, rows, topk, ws)
    torch.cuda.synchronize()
    assert torch.equal(o["y"].view(torch.int32), again["y"].view(torch.int32))
    cold = [r for r in range(rows) if r not in hot]
    assert torch.equal(o["y"][cold], clean["y"][cold]) and torch.equal(o["idx"], clean["idx"])
    if cold:
        M.check(lay, x, res, o, rows, topk, skip=hot)
    want = definition(lay, x, res, host(o["idx"]), host(o["wts"]).astype(np.float64), host(o["sgate"]))[hot]
    got = host(o["y"])[hot].astype(np.float64)
    assert not np.isfinite(want).any() and np.isinf(want).sum() > want.size // 8 and np.isnan(want).any()
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("rows,e,h,i,topk,shared", [(1, 4, 256, 128, 2, True), (9, 4, 384, 256, 2, False), (40, 3, 256, 2688, 1, True),
                                                    (1, 4, 128, 8192, 3, False)])
def test_int4_products_beyond_fp32(rows, e, h, i, topk, shared):
    """An activation of 3.6e37: q scale + min times it is a number, 31 times it is not."""
    import torch

    lay = M.Layer(rows * 37 + h, "q4", "cfg", e, h, i, shared)
    unit, big = 5, 70
    only_unit(lay, unit, big)
    lay.put()
    torch.manual_seed(rows)
    x, res = torch.randn(rows, h, device="cuda").to(torch.bfloat16), torch.randn(rows, h, device="cuda")
    x[:, big] = 6e18
    o = lay.call(x, res, rows, topk, M.workspace(rows, e, h, i, topk))
    torch.cuda.synchronize()
    M.check(lay, x, res, o, rows, topk)


@pytest.mark.parametrize("rows", [1, 2, 20])
def test_int4_inputs_beyond_a_thirtieth_of_fp32(rows):
    """x of 3e38 under scales of 2e-38: gate and up are numbers of ordinary size."""
    import torch

    e, h, i, topk = 4, 512, 128, 2
    lay = M.Layer(rows + 41, "q4", "cfg", e, h, i, True)
    big = 200
    only_unit(lay, 0, big)
    pair(lay.L, "gu_s", slice(None), big // 64, 2e-38, 4e-38)
    lay.L["gu_q"][:, :, big // 2] = np.random.default_rng(rows).integers(0, 256, lay.L["gu_q"].shape[:2])
    lay.put()
    torch.manual_seed(rows)
    x = torch.randn(rows, h, device="cuda").to(torch.bfloat16)
    x[:, big] = 3e38
    x[:, big - big % 64:big] = 0
    x[:, big + 1:big - big % 64 + 64] = 0
    res = torch.randn(rows, h, device="cuda")
    o = lay.call(x, res, rows, topk, M.workspace(rows, e, h, i, topk))
    torch.cuda.synchronize()
    M.check(lay, x, res, o, rows, topk)
