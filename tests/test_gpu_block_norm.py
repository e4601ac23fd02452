"""dr_block_norm, dr_block_norm_bf16 and dr_moe_combine_norm against the formulas in 64 bits.

Tolerances, u = 2^-24 (an fp32 rounding).  A row's sum of squares is a chain of at most 16 fmas per lane, 6
butterfly steps and 16 wave sums, all of non-negative terms: relative error <= 38 u, with the division and
eps 40 u, so rsqrt of it (itself within 2 ulp = 4 u) is within 24 u.  n has four more products, the gate an exp (2 ulp =
4 u), a sum and a division: 24 + 4 + 6 < 36 u of the block's term.  xo adds one product and one sum.  The
combined b is a sum of topk + 1 products, its first with a sigmoid: (topk + 8) u of the sum of its terms'
magnitudes, which also moves the norm by sum(|b| db) / sum(b^2).  hn: xo's error, its own norm's 24 u, two
products, xo's error within the norm, and one rounding to bf16, 2^-8 of the value."""
import ctypes

import numpy as np
import pytest

import dramamoe as D

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(b, db, x, pw, gate, cs, bscale, xscale, nw, eps):
    """(xo, its bound, hn, its bound) in float64; db: how far b itself may be off."""
    n, dn = b, db
    if pw is not None:
        ms = (b * b).mean(-1, keepdims=True) + eps
        inv = 1 / np.sqrt(ms)
        rel = (np.abs(b) * db).mean(-1, keepdims=True) / ms
        n = b * inv * pw
        dn = db * inv * np.abs(pw) + np.abs(n) * rel
    s = bscale * (cs if cs is not None else 1.0)
    if gate is not None:
        s = s / (1 + np.exp(-gate))
    term, dterm = s * n, np.abs(s) * dn + 36 * U * np.abs(s * n)
    xs = xscale * x if x is not None else 0 * term
    xo = xs + term
    dxo = dterm + U * np.abs(xs) + U * np.abs(xo)
    ms = (xo * xo).mean(-1, keepdims=True) + eps
    inv = 1 / np.sqrt(ms)
    hn = xo * inv * nw
    rel = (np.abs(xo) * dxo).mean(-1, keepdims=True) / ms
    dhn = dxo * inv * np.abs(nw) + np.abs(hn) * (rel + 28 * U)
    return xo, dxo, hn, dhn + 2.0 ** -8 * (np.abs(hn) + dhn)


def dev(a, dt=None, off=0, ld=None, fill=float("nan")):
    """A 2-D float64 array on the device: rows of stride ld, the first element `off` elements into the
    allocation, everything outside the rows `fill`.  Returns (tensor, pointer, view of the rows)."""
    import torch

    rows, h = a.shape
    ld = ld or h
    dt = dt or torch.float32
    flat = torch.full((off + rows * ld + 64,), fill, dtype=dt, device="cuda")
    view = flat[off:off + rows * ld].view(rows, ld)
    view[:, :h] = torch.from_numpy(a).to(dt).cuda()
    return flat, flat.data_ptr() + off * flat.element_size(), view


def check(got, want, bound, what):
    got = got.double().cpu().numpy()
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:3], want[bad][:3], bound[bad][:3])


CASES = [
    # rows, h, stride beyond h, offset, gate_mode, post norm, cs
    (1, 2048, 0, 0, 0, True, False), (1, 1, 0, 0, 1, True, True), (3, 7, 5, 1, 2, True, True), (5, 512, 0, 0, 2, False, True),
    (9, 513, 0, 0, 1, True, False), (4, 1000, 24, 4, 2, True, True), (2, 1024, 0, 2, 0, False, False), (3, 2050, 2, 0, 2, True, True),
    (6, 4096, 0, 0, 1, True, True), (2, 4100, 4, 0, 2, True, False), (2, 8192, 0, 0, 2, True, True), (2, 8191, 0, 1, 2, True, True),
    (2, 12288, 0, 0, 2, True, True), (1, 16384, 0, 0, 1, True, False), (1, 16383, 0, 3, 2, True, True), (1000, 64, 0, 0, 2, True, True),
]


def run_norm(lib, name, b_ptr, ldb, x_ptr, ldx, v, gate_mode, gate_ptr, ldg, xo_ptr, ldo, hn_ptr, ldh, rows, h, stream=None):
    getattr(lib, name)(b_ptr, ldb, x_ptr, ldx, v["pw"], gate_ptr, gate_mode, ldg, v["cs"], 0.75, 1.25, v["nw"], 1e-6, xo_ptr, ldo, hn_ptr,
                       ldh, rows, h, stream or D.stream_ptr())


@pytest.mark.parametrize("b16", [False, True])
@pytest.mark.parametrize("rows,h,pad,off,gm,post,cs", CASES)
def test_block_norm(rows, h, pad, off, gm, post, cs, b16):
    import torch

    rng = np.random.default_rng(rows * 20011 + h)
    f32 = lambda *s: rng.normal(0, 1, s).astype(np.float32).astype(np.float64)
    b, x, g = 3 * f32(rows, h), f32(rows, h), 4 * f32(rows, h if gm == 2 else 1)
    pw, csv, nw = 1 + 0.2 * f32(1, h), 1 + 0.2 * f32(1, h), 1 + 0.2 * f32(1, h)
    pw, csv, nw = (a.astype(np.float32).astype(np.float64) for a in (pw, csv, nw))
    b = 3 * torch.from_numpy(b).to(torch.bfloat16) if b16 else torch.from_numpy(b).float()
    b = b.double().numpy()
    x, g = x.astype(np.float32).astype(np.float64), g.astype(np.float32).astype(np.float64)
    ld = h + pad
    keep, v = [], {}
    for k, a in (("pw", pw if post else None), ("cs", csv if cs else None), ("nw", nw)):
        t = dev(a, off=off) if a is not None else (None, None, None)
        keep.append(t), v.update({k: t[1]})
    tb = dev(b, torch.bfloat16 if b16 else None, off=off, ld=ld)
    tx, tg = dev(x, off=off, ld=ld), dev(g, off=off, ld=ld if gm == 2 else 1)
    to, th = dev(0 * x, off=off, ld=ld, fill=7.0), dev(0 * x, torch.bfloat16, off=off, ld=ld, fill=7.0)
    run_norm(D.lib(), "dr_block_norm_bf16" if b16 else "dr_block_norm", tb[1], ld, tx[1], ld, v, gm, tg[1] if gm else None, ld, to[1], ld,
             th[1], ld, rows, h)
    torch.cuda.synchronize()
    xo, dxo, hn, dhn = reference(b, 0 * b, x, pw if post else None, g if gm else None, csv if cs else None, 0.75, 1.25, nw, 1e-6)
    check(to[2][:, :h], xo, dxo, "xo")
    check(th[2][:, :h], hn, dhn, "hn")
    # what lies between and behind the rows is left as it was
    for flat, _, view in (to, th):
        assert (view[:, h:] == 7).all() and (flat[off + rows * ld:] == 7).all() and (flat[:off] == 7).all()


def test_optional_operands_and_aliases():
    """No block output (the norm before the first block), no residual, one output only, xo in place of x and of b,
    hn in place of a bf16 b."""
    import torch

    lib, rng = D.lib(), np.random.default_rng(5)
    rows, h = 5, 1536
    f32 = lambda *s: rng.normal(0, 1, s).astype(np.float32).astype(np.float64)
    b, x, nw, pw = f32(rows, h), f32(rows, h), f32(1, h), f32(1, h)
    tn, tp = dev(nw), dev(pw)
    v = {"pw": None, "cs": None, "nw": tn[1]}
    tx, th, to = dev(x), dev(0 * x, torch.bfloat16), dev(0 * x)
    run_norm(lib, "dr_block_norm", None, 0, tx[1], h, v, 0, None, 0, None, 0, th[1], h, rows, h)
    xo, dxo, hn, dhn = reference(0 * x, 0 * x, x, None, None, None, 0.75, 1.25, nw, 1e-6)
    check(th[2], hn, dhn, "hn of x alone")
    v["pw"] = tp[1]
    tb = dev(b)
    run_norm(lib, "dr_block_norm", tb[1], h, None, 0, v, 0, None, 0, to[1], h, th[1], h, rows, h)
    xo, dxo, hn, dhn = reference(b, 0 * b, None, pw, None, None, 0.75, 1.25, nw, 1e-6)
    check(to[2], xo, dxo, "xo without residual"), check(th[2], hn, dhn, "hn without residual")
    xo, dxo, hn, dhn = reference(b, 0 * b, x, pw, None, None, 0.75, 1.25, nw, 1e-6)
    run_norm(lib, "dr_block_norm", tb[1], h, tx[1], h, {**v, "nw": None}, 0, None, 0, to[1], h, None, 0, rows, h)
    check(to[2], xo, dxo, "xo alone")
    run_norm(lib, "dr_block_norm", tb[1], h, tx[1], h, v, 0, None, 0, tb[1], h, th[1], h, rows, h)
    check(tb[2], xo, dxo, "xo over b"), check(th[2], hn, dhn, "hn beside")
    tb = dev(b, torch.bfloat16)
    bb = tb[2].double().cpu().numpy()
    xo, dxo, hn, dhn = reference(bb, 0 * b, x, pw, None, None, 0.75, 1.25, nw, 1e-6)
    run_norm(lib, "dr_block_norm_bf16", tb[1], h, tx[1], h, v, 0, None, 0, tx[1], h, tb[1], h, rows, h)
    check(tx[2], xo, dxo, "xo over x"), check(tb[2], hn, dhn, "hn over b")


def test_rows_keep_to_themselves():
    """A row of zeros, of huge and of tiny values, infinities and NaN: its neighbours have the bits they have alone,
    and gate logits of +-100 and +-inf pass or close the gate."""
    import torch

    lib, rng = D.lib(), np.random.default_rng(6)
    rows, h = 8, 2048
    b = rng.normal(0, 1, (rows, h))
    x = rng.normal(0, 1, (rows, h))
    clean = dev(b), dev(x)
    g = dev(rng.normal(0, 1, (rows, 1)))
    nw = dev(np.ones((1, h)))
    outs = []
    for bad in (False, True):
        tb, tx = dev(b), dev(x)
        if bad:
            tb[2][1], tx[2][1] = 0.0, 0.0
            tb[2][3], tb[2][4], tb[2][5, 7], tx[2][6, 9] = 1e17, 1e-30, float("inf"), float("nan")
        to, th = dev(0 * x), dev(0 * x, torch.bfloat16)
        run_norm(lib, "dr_block_norm", tb[1], h, tx[1], h, {"pw": nw[1], "cs": None, "nw": nw[1]}, 1, g[1], 0, to[1], h, th[1], h, rows, h)
        outs.append((to[2].clone(), th[2].clone()))
    torch.cuda.synchronize()
    for r in (0, 2, 7):
        assert torch.equal(outs[0][0][r], outs[1][0][r]) and torch.equal(outs[0][1][r], outs[1][1][r])
    assert (outs[1][0][1] == 0).all() and (outs[1][1][1] == 0).all()
    assert torch.isfinite(outs[1][0][3:5]).all()
    assert not torch.isfinite(outs[1][0][5]).all() and torch.isnan(outs[1][1][6]).all()
    gate = dev(np.array([[100.0], [-100.0], [np.inf], [-np.inf]] * 2))
    to = dev(0 * x)
    lib.dr_block_norm(clean[0][1], h, clean[1][1], h, None, gate[1], 1, 0, None, 1.0, 1.0, None, 1e-6, to[1], h, None, 0,
                      rows, h, D.stream_ptr())
    bb, xx = clean[0][2], clean[1][2]
    assert torch.equal(to[2][0::4], (xx + bb)[0::4]) and torch.equal(to[2][2::4], (xx + bb)[2::4])
    assert torch.equal(to[2][1::4], xx[1::4]) and torch.equal(to[2][3::4], xx[3::4])


@pytest.mark.parametrize("rows,h,topk,shared,post,gm", [
    (1, 2048, 8, True, False, 0), (300, 2048, 8, True, True, 1), (7, 1800, 3, False, True, 2), (3, 515, 32, True, True, 2),
    (2, 5120, 1, True, True, 0), (2, 8196, 5, True, False, 2), (40, 96, 2, True, True, 1)])
def test_combine_norm(rows, h, topk, shared, post, gm):
    import torch

    rng = np.random.default_rng(h + topk)
    f32 = lambda *s: rng.normal(0, 1, s).astype(np.float32).astype(np.float64)
    y, sh, x, nw, pw = f32(rows * topk, h), f32(rows, h), f32(rows, h), f32(1, h), f32(1, h)
    w, sg, g = np.abs(f32(rows, topk)), f32(rows, 1), f32(rows, h if gm == 2 else 1)
    slot = rng.permutation(rows * topk).astype(np.int32)
    ts = torch.from_numpy(slot).cuda()
    ty, tsh, tx, tn, tp, tw, tsg, tg = (dev(a) for a in (y, sh, x, nw, pw, w, sg, g))
    to, th = dev(0 * x), dev(0 * x, torch.bfloat16)
    D.lib().dr_moe_combine_norm(ty[1], ts.data_ptr(), tw[1], tsg[1] if shared else None, tsh[1] if shared else None, topk, tx[1], h,
                                tp[1] if post else None, tg[1] if gm else None, gm, h, None, 0.75, 1.25, tn[1], 1e-6, to[1], h, th[1], h,
                                rows, h, D.stream_ptr())
    torch.cuda.synchronize()
    terms = w[:, :, None] * y[slot.reshape(rows, topk)]
    b, mag = terms.sum(1), np.abs(terms).sum(1)
    if shared:
        s = sh / (1 + np.exp(-sg))
        b, mag = b + s, mag + np.abs(s)
    xo, dxo, hn, dhn = reference(b, (topk + 8) * U * mag, x, pw if post else None, g if gm else None, None, 0.75, 1.25, nw, 1e-6)
    check(to[2], xo, dxo, "xo"), check(th[2], hn, dhn, "hn")


def test_combine_norm_matches_combine():
    """Without norm behind the block, gate and scales the residual stream is dr_moe_combine's up to the order of one sum."""
    import torch

    torch.manual_seed(3)
    rows, h, topk = 37, 2048, 8
    c = dict(device="cuda")
    y, sh, x = torch.randn(rows * topk, h, **c), torch.randn(rows, h, **c), torch.randn(rows, h, **c)
    w, sg = torch.rand(rows, topk, **c), torch.randn(rows, **c)
    slot = torch.randperm(rows * topk, **c).to(torch.int32)
    P, st = D.ptr, D.stream_ptr()
    want, got = x.clone(), torch.empty_like(x)
    D.lib().dr_moe_combine(P(want), P(y), P(slot), P(w), P(sg), P(sh), rows, topk, h, st)
    D.lib().dr_moe_combine_norm(P(y), P(slot), P(w), P(sg), P(sh), topk, P(x), h, None, None, 0, 0, None, 1.0, 1.0, None, 1e-6, P(got), h,
                                None, 0, rows, h, st)
    mag = (w.abs()[:, :, None] * y[slot.long()].view(rows, topk, h).abs()).sum(1) + sh.abs() + x.abs()
    # both are sums of the same ten terms in fp32; the fast exponential of dr_moe_combine's gate is within 2^-21
    assert ((got - want).abs() <= (2 * (topk + 8) * U + 2.0 ** -21) * mag).all()


def test_graph_and_stream():
    """Captured on a stream of its own and replayed with new inputs and eager calls in between: the eager bits."""
    import torch

    lib, (rows, h) = D.lib(), (33, 2048)
    torch.manual_seed(4)
    b, x, nw = torch.randn(rows, h, device="cuda"), torch.randn(rows, h, device="cuda"), torch.randn(h, device="cuda")
    xo, hn = torch.empty_like(x), torch.empty(rows, h, dtype=torch.bfloat16, device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    P = D.ptr

    def call():
        lib.dr_block_norm(P(b), h, P(x), h, P(nw), None, 0, 0, None, 1.0, 1.0, P(nw), 1e-6, P(xo), h, P(hn), h, rows, h, st.cuda_stream)

    g = ctypes.c_void_p()
    lib.dr_graph_begin(st.cuda_stream)
    call()
    assert lib.dr_graph_end(st.cuda_stream, ctypes.byref(g)) == 0
    try:
        for _ in range(3):
            b.normal_()
            torch.cuda.synchronize()
            call()
            st.synchronize()
            want = xo.clone(), hn.clone()
            xo.zero_(), hn.zero_()
            torch.cuda.synchronize()
            lib.dr_graph_launch(g, st.cuda_stream)
            st.synchronize()
            assert torch.equal(xo, want[0]) and torch.equal(hn, want[1])
    finally:
        lib.dr_graph_destroy(g)
