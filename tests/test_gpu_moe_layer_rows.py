"""dr_moe_layer_rows* against the formulas in 64 bits, its routing against dr_gemm + dr_moe_topk bit for bit.

Tolerances, u = 2^-24.  A product row . x is summed in fp32: 64 terms of a scale group, the group's scale applied
with one fma each, at most 32 chunks of 4 groups and 8 waves added: each partial sum is at most M = sum of the terms'
magnitudes (int4: |(16 + q) s x| + |(m - 16 s) x|), so the error is at most (64 + 128 + 8 + 4) u M < 208 u M.  silu(g) u:
slope at most 1.1 in g, an exp (4 u), a sum, a division and a product: 8 u.  The activation's three bf16 planes are
exact.  The combine adds topk + 2 products; each weight has the softmax's error, (e / 64 + 16) u, the gate's exp as above."""
import ctypes

import numpy as np
import pytest

import dramamoe as D
import synth
from helpers import bits, dev, host

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NAMES = {("q4", "ref"): "dr_moe_layer_rows", ("q4", "cfg"): "dr_moe_layer_rows_bf16s", ("fp8", "ref"): "dr_moe_layer_rows_fp8",
         ("fp8", "cfg"): "dr_moe_layer_rows_fp8_bf16s"}


class Layer:
    def __init__(self, seed, kind, fmt, e, h, i, shared):
        L = self.L = synth.make_layer(seed, E=e, H=h, I=i, fmt=fmt, kind=kind, with_norm=False, quick=True)
        self.kind, self.fmt, self.e, self.h, self.i, self.shared = kind, fmt, e, h, i, shared
        if not shared:
            L["router"] = np.ascontiguousarray(L["router"][:e])
        self.put()

    def put(self):
        L = self.L
        keys = ("router", "gu_q", "gu_s", "d_q", "d_s") + (("sgu_q", "sgu_s", "sd_q", "sd_s") if self.shared else ())
        self.t = {k: dev(L[k]) for k in keys}

    def weights(self, q, s, j):
        """(w, magnitude bound of its terms per unit of x) of expert j in float64."""
        L = self.L
        if self.kind == "q4":
            b = L[q][j].astype(np.int64)
            v = np.stack([b & 15, b >> 4], -1).reshape(b.shape[0], -1)
            p = synth.dec(L[s][j], L["sc_kind"]).astype(np.float64).repeat(64, axis=1)
            sc, mn = p[..., 0], p[..., 1]
            return v * sc + mn, (16 + v) * np.abs(sc) + np.abs(mn - 16 * sc)
        sc = synth.dec(L[s][j], L["sc_kind"]).astype(np.float64).repeat(128, 0).repeat(128, 1)
        w = synth.E4M3[L[q][j]].astype(np.float64) * sc
        return w, np.abs(w)

    def shared_weights(self, q, s):
        L = self.L
        sc = synth.dec(L[s], L["sh_kind"]).astype(np.float64)
        sc = sc[:, None] if sc.ndim == 1 else sc.repeat(128, 1)
        w = L[q].astype(np.float64) * sc
        return w, np.abs(w)

    def call(self, x, res, rows, topk, ws, stream=None, out=None):
        import torch

        o = out or {"idx": torch.full((rows, topk), -7, dtype=torch.int32, device="cuda"), "wts": torch.full((rows, topk), -7.0, device="cuda"),
                    "sgate": torch.full((rows,), -7.0, device="cuda"), "y": torch.full((rows + 1, self.h), -7.0, device="cuda")}
        P, t = D.ptr, self.t
        getattr(D.lib(), NAMES[self.kind, self.fmt])(
            P(t["router"]), P(t["gu_q"]), P(t["gu_s"]), P(t["d_q"]), P(t["d_s"]), *(P(t.get(k)) for k in ("sgu_q", "sgu_s", "sd_q", "sd_s")),
            P(x), P(res), P(o["idx"]), P(o["wts"]), P(o["sgate"]) if self.shared else None, P(ws), P(o["y"]), rows, self.e, self.h, self.i,
            topk, stream or D.stream_ptr())
        return o


def workspace(rows, e, h, i, topk):
    import torch

    n = D.lib().dr_moe_layer_rows_ws(rows, e, h, i, topk)
    ws = torch.full((n + 256,), 0x5A, dtype=torch.uint8, device="cuda")  # only the first 1024 bytes need be zero
    ws[:1024] = 0
    return ws


def mlp(x, gu, dn, i):
    """(D silu(G x) U x, its error bound) of rows x, from (w, magnitude) pairs."""
    z, dz = x @ gu[0].T, 208 * U * (np.abs(x) @ gu[1].T)
    g, v, dg, dv = z[:, :i], z[:, i:], dz[:, :i], dz[:, i:]
    silu = g / (1 + np.exp(-g))
    act = silu * v
    dact = 1.1 * dg * (np.abs(v) + dv) + np.abs(silu) * dv + 8 * U * np.abs(act)
    return act @ dn[0].T, dact @ np.abs(dn[0]).T + 208 * U * ((np.abs(act) + dact) @ dn[1].T)


def check(lay, x, res, o, rows, topk, skip=()):
    """o against the definition on the picks that o itself reports (their choice is checked apart)."""
    e, i = lay.e, lay.i
    xf = x[:rows].double().cpu().numpy()
    idx = host(o["idx"])
    router = synth.bf16_to_f32(lay.L["router"]).astype(np.float64)
    logits = xf @ router.T
    y = res.double().cpu().numpy().copy() if res is not None else np.zeros((rows, lay.h))
    mag, dy = np.abs(y), 0 * y
    w = np.zeros((rows, topk))
    keep = [r for r in range(rows) if r not in skip]
    for r in keep:
        l = logits[r, :e]
        p = np.exp(l[idx[r]] - l.max())
        w[r] = p / p.sum()
    # the router's fp32 dot is within (h / 64 + 6) u of its terms' magnitudes, which shifts every weight by that much
    dl = (lay.h / 64 + 6) * U * (np.abs(xf) @ np.abs(router).T).max(-1, initial=0.0)
    dw = w * ((e / 64 + 16) * U + 4 * dl[:, None])
    got_w = host(o["wts"]).astype(np.float64)
    assert (np.abs(got_w - w) <= dw)[keep].all()
    for j in sorted(set(idx[keep].ravel().tolist())):
        rr, kk = np.nonzero(idx == j)
        sel = [q for q in range(len(rr)) if rr[q] in keep]
        rr, kk = rr[sel], kk[sel]
        out, d = mlp(xf[rr], lay.weights("gu_q", "gu_s", j), lay.weights("d_q", "d_s", j), i)
        ww = w[rr, kk][:, None]
        y[rr] += ww * out
        mag[rr] += np.abs(ww * out)
        dy[rr] += ww * d + dw[rr, kk][:, None] * np.abs(out)
    if lay.shared:
        out, d = mlp(xf[keep], lay.shared_weights("sgu_q", "sgu_s"), lay.shared_weights("sd_q", "sd_s"), i)
        s = 1 / (1 + np.exp(-logits[keep, e]))[:, None]
        y[keep] += s * out
        mag[keep] += np.abs(s * out)
        dy[keep] += s * d + np.abs(s * out) * (8 * U + dl[keep, None])
        assert (np.abs(host(o["sgate"]) - logits[:, e]) <= dl + U * np.abs(logits[:, e]))[keep].all()
    bound = dy + (topk + 4) * U * mag
    got = host(o["y"]).astype(np.float64)[:rows]
    bad = ~(np.abs(got - y) <= bound)[keep]
    assert not bad.any(), (int(bad.sum()), np.abs(got - y)[keep][bad][:4], bound[keep][bad][:4])
    assert np.abs(got - y)[keep].max() <= 2e-3 * max(1.0, np.abs(y[keep]).max())  # the bound itself stays tight enough to mean something
    assert (host(o["y"])[rows:] == -7).all()
    for r in keep:
        assert len(set(idx[r].tolist())) == topk and 0 <= idx[r].min() and idx[r].max() < e


def routing(lay, x, rows, topk):
    """idx, wts, sgate of dr_gemm + dr_moe_topk (h <= 4096); a router without a gate row gets a row of zeros."""
    import torch

    e, h, P, lib, st = lay.e, lay.h, D.ptr, D.lib(), D.stream_ptr()
    w = lay.t["router"].view(torch.bfloat16).reshape(-1, h)
    if not lay.shared:
        w = torch.cat([w, torch.zeros(1, h, dtype=torch.bfloat16, device="cuda")])
    logits = torch.empty(rows, e + 1, device="cuda")
    hd = ctypes.c_void_p()
    lib.dr_cublas_create(ctypes.byref(hd), st)
    lib.dr_gemm(hd, P(x), P(w), P(logits), rows, e + 1, h, 0.0)
    idx, wts, sg = torch.empty(rows, topk, dtype=torch.int32, device="cuda"), torch.empty(rows, topk, device="cuda"), torch.empty(rows, device="cuda")
    lib.dr_moe_topk(P(logits), rows, e, topk, e + 1, P(idx), P(wts), P(sg), st)
    torch.cuda.synchronize()
    lib.dr_cublas_destroy(hd)
    return idx, wts, sg


CASES = [
    # kind, fmt, rows, e, h, i, topk, shared
    ("q4", "ref", 1, 16, 2048, 512, 8, True), ("q4", "cfg", 1, 1, 128, 128, 1, False), ("fp8", "ref", 1, 9, 256, 128, 3, True),
    ("fp8", "cfg", 2, 8, 384, 256, 8, True), ("q4", "ref", 3, 12, 640, 384, 5, True), ("q4", "cfg", 8, 40, 1280, 896, 4, False),
    ("fp8", "cfg", 9, 33, 512, 1152, 2, True), ("q4", "ref", 16, 20, 2048, 512, 8, True), ("q4", "cfg", 17, 5, 384, 128, 5, True),
    ("fp8", "ref", 33, 24, 1024, 256, 6, False), ("q4", "ref", 64, 64, 512, 256, 8, True), ("q4", "cfg", 64, 3, 256, 384, 1, True),
    ("fp8", "cfg", 61, 4, 256, 128, 4, True), ("q4", "ref", 5, 64, 128, 128, 32, True), ("q4", "cfg", 2, 4, 8192, 128, 2, True),
    ("fp8", "ref", 3, 4, 4224, 128, 2, True), ("q4", "ref", 4, 4, 256, 2688, 2, True), ("fp8", "cfg", 64, 256, 256, 128, 8, True),
    ("q4", "cfg", 31, 256, 256, 128, 3, False), ("q4", "ref", 1, 64, 256, 128, 32, True), ("fp8", "cfg", 2, 64, 256, 128, 32, True),
    ("q4", "cfg", 1, 4, 128, 8192, 3, False), ("fp8", "ref", 2, 32, 2176, 640, 6, False), ("q4", "ref", 2, 3, 1152, 1024, 3, True),
]


@pytest.mark.parametrize("kind,fmt,rows,e,h,i,topk,shared", CASES)
def test_layer(kind, fmt, rows, e, h, i, topk, shared):
    import torch

    lay = Layer(rows * 1000 + h, kind, fmt, e, h, i, shared)
    torch.manual_seed(rows)
    x, res = torch.randn(rows, h, device="cuda").to(torch.bfloat16), torch.randn(rows, h, device="cuda")
    ws = workspace(rows, e, h, i, topk)
    o = lay.call(x, res, rows, topk, ws)
    torch.cuda.synchronize()
    check(lay, x, res, o, rows, topk)
    assert (ws[:1024] == 0).all() and (ws[-256:] == 0x5A).all()
    if h <= 4096:
        idx, wts, sg = routing(lay, x, rows, topk)
        assert torch.equal(o["idx"], idx)
        np.testing.assert_array_equal(bits(host(o["wts"])), bits(host(wts)))
        if shared:
            np.testing.assert_array_equal(bits(host(o["sgate"])), bits(host(sg)))
    # again on the same workspace: the same bits; and in place of res, without one
    o2 = lay.call(x, res, rows, topk, ws)
    assert torch.equal(o["y"], o2["y"])
    y = torch.cat([res, torch.full((1, h), -7.0, device="cuda")])
    o3 = lay.call(x, y[:rows], rows, topk, ws, out={**o, "y": y})
    assert torch.equal(o3["y"], o2["y"])
    o4 = lay.call(x, None, rows, topk, ws)
    torch.cuda.synchronize()
    check(lay, x, None, o4, rows, topk)


@pytest.mark.parametrize("kind", ["q4", "fp8"])
def test_hot_expert_and_ties(kind):
    """Rows that all pick the same experts (passes of 16 beyond the first), picks among equal logits (lowest index
    first), next to rows that go elsewhere."""
    import torch

    rows, e, h, i, topk = 64, 24, 512, 256, 3
    lay = Layer(77, kind, "ref", e, h, i, True)
    lay.L["router"][5:9] = lay.L["router"][4]
    lay.put()
    torch.manual_seed(1)
    x = torch.randn(rows, h, device="cuda").to(torch.bfloat16)
    up = torch.from_numpy(synth.bf16_to_f32(lay.L["router"][4])).cuda()
    x[:50] = (x[:50].float() + 60 * up).to(torch.bfloat16)
    ws = workspace(rows, e, h, i, topk)
    o = lay.call(x, None, rows, topk, ws)
    torch.cuda.synchronize()
    assert (o["idx"][:50] == torch.tensor([4, 5, 6], device="cuda")).all()
    check(lay, x, None, o, rows, topk)


def test_row_keeps_its_bits_in_any_company():
    """A row's routing and output do not depend on the rows beside it but for the place in a pass: rows in another
    order, and NaN and infinities in one row, leave the others' bits."""
    import torch

    rows, e, h, i, topk = 21, 32, 1024, 256, 4
    lay = Layer(78, "q4", "cfg", e, h, i, True)
    torch.manual_seed(2)
    x, res = torch.randn(rows, h, device="cuda").to(torch.bfloat16), torch.randn(rows, h, device="cuda")
    ws = workspace(rows, e, h, i, topk)
    o = lay.call(x, res, rows, topk, ws)
    perm = torch.randperm(rows, device="cuda")
    q = lay.call(x[perm].contiguous(), res[perm].contiguous(), rows, topk, ws)
    torch.cuda.synchronize()
    assert torch.equal(q["y"][:rows], o["y"][perm]) and torch.equal(q["idx"], o["idx"][perm])
    bad = x.clone()
    bad[3, 5], bad[7, 1] = float("nan"), float("inf")
    b = lay.call(bad, res, rows, topk, ws)
    torch.cuda.synchronize()
    keep = [r for r in range(rows) if r not in (3, 7)]
    assert torch.equal(b["y"][keep], o["y"][keep]) and torch.equal(b["idx"][keep], o["idx"][keep])
    assert torch.isnan(b["y"][3]).all()
    assert (b["idx"] >= 0).all() and (b["idx"] < e).all()


def test_one_workspace_for_calls_of_any_size():
    import torch

    ws = workspace(40, 64, 1024, 512, 8)
    for kind, fmt, rows, e, h, i, topk, shared in (("q4", "ref", 40, 64, 1024, 512, 8, True), ("fp8", "ref", 3, 8, 256, 128, 2, False),
                                                   ("q4", "cfg", 33, 16, 512, 256, 4, True), ("q4", "ref", 1, 64, 1024, 512, 8, True)):
        lay = Layer(rows, kind, fmt, e, h, i, shared)
        x = torch.randn(rows, h, device="cuda").to(torch.bfloat16)
        o = lay.call(x, None, rows, topk, ws)
        torch.cuda.synchronize()
        check(lay, x, None, o, rows, topk)


def test_graph_replays():
    """Captured once, replayed on new rows with eager calls of another size on the same workspace in between."""
    import torch

    lib, (rows, e, h, i, topk) = D.lib(), (12, 32, 1024, 256, 4)
    lay = Layer(80, "fp8", "cfg", e, h, i, True)
    x, res = torch.randn(rows, h, device="cuda").to(torch.bfloat16), torch.randn(rows, h, device="cuda")
    ws = workspace(rows, e, h, i, topk)
    st = torch.cuda.Stream()
    o = lay.call(x, res, rows, topk, ws)
    torch.cuda.synchronize()
    g = ctypes.c_void_p()
    lib.dr_graph_begin(st.cuda_stream)
    lay.call(x, res, rows, topk, ws, stream=st.cuda_stream, out=o)
    assert lib.dr_graph_end(st.cuda_stream, ctypes.byref(g)) == 0
    try:
        for _ in range(4):
            x.copy_(torch.randn(rows, h, device="cuda"))
            torch.cuda.synchronize()
            want = lay.call(x, res, rows, topk, ws)
            lay.call(x, res, 1, topk, ws)
            torch.cuda.synchronize()
            lib.dr_graph_launch(g, st.cuda_stream)
            st.synchronize()
            assert torch.equal(o["y"], want["y"]) and torch.equal(o["idx"], want["idx"]) and torch.equal(o["wts"], want["wts"])
    finally:
        lib.dr_graph_destroy(g)
