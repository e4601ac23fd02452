"""dr_moe_layer_rows*: the activations between gate_up and down keep all 24 bits of an fp32 number.

x has one input, the weights let one activation count, and every scale is a power of two, so that there is nothing to sum:
q scale x and its int4 parts (16 + q) scale x and 16 scale x have at most 16 bits and are exact.  With u = 2^-24 the activation silu(g) u
is off by the exponential (2 ulp, 4 u), a sum, a division and a product (u each): 7 u.  Its three planes are exact and so is
each one's product; their two sums add 2 u.  The one pick's weight is 1, the shared gate's sigmoid(0) is 1/2: exact.  9 u in all.  An
activation cut to two planes (16 bits) would be off by up to 2^-15 = 512 u, half of them by more than 90."""
import numpy as np
import pytest

import synth
import test_gpu_moe_layer_rows as M
from helpers import host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def weights(rng, kind, n):
    """n stored values and what they are, before the scale."""
    if kind == "q4":
        q = rng.integers(1, 16, n).astype(np.uint8)
        return q, q.astype(np.float64)
    if kind == "fp8":
        q = rng.integers(0x28, 0x48, n).astype(np.uint8)  # 0.25 .. 3.75
        return q, synth.E4M3[q].astype(np.float64)
    q = rng.integers(1, 128, n).astype(np.int8)
    return q, q.astype(np.float64)


def put(L, kind, name, rows, k, q):
    """Stored values q in column k of rows, one per expert and row."""
    if kind == "q4":
        L[name][:, rows, k // 2] = q << 4 if k % 2 else q
    else:
        L[name][..., rows, k] = q


def silu(g):
    return g / (1 + np.exp(-g))


def cut(v):
    """v in two planes of 8 bits."""
    top = lambda a: (a.astype(np.float32).view(np.uint32) & np.uint32(0xffff0000)).view(np.float32)
    hi = top(v)
    return hi.astype(np.float64) + top(v.astype(np.float32) - hi)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("rows,h,i", [(1, 256, 128), (2, 384, 640), (11, 256, 384), (64, 128, 2688), (1, 128, 8192)])
@pytest.mark.parametrize("kind,fmt", sorted(M.NAMES))
def test_activation_bits(kind, fmt, rows, h, i, shared):
    import torch

    e, rng = 3, np.random.default_rng(rows + h + i)
    topk = 3 if i == 8192 else 1  # three picks of one row go through the kernels for several
    lay = M.Layer(5, kind, fmt, e, h, i, shared)
    L, at, unit = lay.L, h - 3, i - 6
    for k in ("gu_q", "d_q", "sgu_q", "sd_q", "router"):
        L[k][:] = 0
    L["router"][0] = synth.f32_to_bf16(np.float32([1.0]))  # expert 0 is picked wherever the input is positive
    for k in ("gu_s", "d_s"):
        L[k][:] = synth.enc(np.float32([0.125]), L["sc_kind"])
        if kind == "q4":
            L[k][..., 1] = 0
    for k in ("sgu_s", "sd_s"):
        L[k][:] = synth.enc(np.float32([2.0 ** -7]), L["sh_kind"])
    wk = "q8" if shared else kind
    q, gate = weights(rng, wk, 1)
    p, up = weights(rng, wk, 1)
    d, down = weights(rng, wk, h)
    names, sc = (("sgu_q", "sd_q"), 2.0 ** -7) if shared else (("gu_q", "d_q"), 0.125)
    if shared:
        L["sgu_q"][[unit, i + unit], at] = q[0], p[0]
        L["sd_q"][:, unit] = d
    else:
        only = {n: L[n].copy() for n in names}
        put(L, kind, "gu_q", [unit, i + unit], at, np.array([q[0], p[0]]))
        put(L, kind, "d_q", slice(None), unit, d)
        for n in names:  # the other experts add nothing
            L[n][1:] = only[n][1:]
    lay.put()
    ws, errs, planes = M.workspace(rows, e, h, i, topk), [], []
    for rep in range(max(1, 48 // rows)):
        v = (rng.uniform(0.2, 3, rows)).astype(np.float32)
        x = torch.zeros(rows, h, device="cuda")
        x[:, at] = torch.from_numpy(v).cuda()
        x = x.to(torch.bfloat16)
        o = lay.call(x, None, rows, topk, ws)
        torch.cuda.synchronize()
        xv = x[:, at].double().cpu().numpy()
        act = silu(gate[0] * sc * xv) * (up[0] * sc * xv)
        w = 0.5 if shared else host(o["wts"])[:, 0].astype(np.float64)
        if topk == 1 and not shared:
            assert (w == 1).all()
        share = np.broadcast_to(w, rows)[:, None] * sc * down[None, :]
        errs.append(np.abs(host(o["y"])[:rows] / (share * act[:, None]) - 1))
        planes.append(np.abs(cut(act) / act - 1))
    bound = (9 if topk == 1 or shared else 11) * U  # several picks: the weight's product and a sum
    assert np.concatenate(errs).max() <= bound
    assert np.median(np.concatenate(planes)) > 3 * bound  # what the bound tells apart
