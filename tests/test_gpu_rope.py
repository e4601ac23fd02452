"""dr_rope and dr_rope_bf16 against the formulas in 64 bits.

Tolerances, U = 2^-24 (an fp32 rounding).  The sum of squares: chains of at most 8 non-negative terms a lane and 6 butterfly steps,
with the division and eps 16 U; its rsqrt (2 ulp = 4 U) 12 U; two products: n is within 14 U.  Angle: fp32's rounding of at most half a turn in units of
half turns, pi 2^-25, and 64 bits' of the whole turns, 2 pi turns 2^-51; sine and cosine 2 ulp = 4 U, mscale's product U: within 7 U mscale + that
of their value.  Two products and a sum: 3 U of the terms.  In all (14 + 7 + 3) U mscale (|a| + |b|) and the angle's; bf16 adds 2^-8 of the value."""
import numpy as np
import pytest

import dramamoe as D

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def reference(x, nw, eps, pos, freq, ms, pairs, rot):
    """(y, bound) [rows, heads, d] in float64."""
    n = x
    if nw is not None:
        n = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * nw
    y, bound = n.copy(), 14 * U * np.abs(n) if nw is not None else np.zeros(n.shape)
    if rot:
        th = pos.astype(np.float64)[:, None, None] * freq.astype(np.float64)
        c, s = ms * np.cos(th), ms * np.sin(th)
        ia = np.arange(0, rot, 2) if pairs else np.arange(rot // 2)
        ib = ia + 1 if pairs else ia + rot // 2
        a, b = n[..., ia], n[..., ib]
        y[..., ia], y[..., ib] = a * c - b * s, b * c + a * s
        e = abs(ms) * (np.abs(a) + np.abs(b)) * ((24 if nw is not None else 10) * U + np.abs(th) * 2.0 ** -51)
        bound[..., ia], bound[..., ib] = e, e
    return y, bound


CASES = [
    # rows, heads, d, rot, pairs, norm, head stride beyond d, row stride beyond the heads, offset of x in elements
    (1, 20, 128, 128, False, True, 0, 0, 0), (3, 5, 64, 64, True, False, 0, 0, 0), (7, 16, 256, 64, False, True, 256, 0, 0),
    (2, 3, 80, 36, True, True, 0, 4, 0), (2, 3, 80, 40, False, True, 8, 4, 4), (5, 1, 1, 0, False, True, 0, 0, 0), (4, 2, 2, 2, False, False, 0, 0, 0),
    (4, 2, 3, 2, True, True, 1, 3, 1), (3, 7, 33, 20, False, True, 2, 5, 3), (2, 2, 512, 512, True, True, 0, 0, 0), (2, 1, 511, 510, False, True, 1, 1, 1),
    (300, 4, 96, 0, False, True, 0, 0, 0), (1000, 1, 8, 8, False, True, 0, 0, 0), (129, 3, 100, 24, True, True, 0, 0, 0), (64, 40, 64, 32, False, False, 0, 0, 2),
    (2, 130, 192, 192, False, True, 0, 0, 0),
    # few rows whose heads several blocks share, evenly and not
    (1, 40, 256, 256, False, True, 0, 0, 0), (3, 37, 128, 64, True, True, 4, 8, 0), (5, 39, 219, 108, True, True, 1, 3, 1), (2, 130, 33, 32, False, False, 0, 0, 0),
    (300, 30, 223, 160, False, True, 0, 0, 0),
    # pairs whose turned elements end inside a wide load's half
    (9, 5, 20, 4, True, True, 0, 0, 0), (4, 3, 76, 76, True, True, 4, 0, 4), (2, 2, 508, 500, True, False, 0, 4, 0), (3, 1, 4, 4, True, True, 0, 0, 0), (5, 2, 12, 0, True, True, 0, 0, 0),
]


def buffer(rows, ld, off, dt, fill):
    import torch

    flat = torch.full((off + rows * ld + 16,), fill, dtype=dt, device="cuda")
    return flat, flat[off:off + rows * ld].view(rows, ld)


@pytest.mark.parametrize("b16", [False, True])
@pytest.mark.parametrize("rows,heads,d,rot,pairs,norm,hpad,rpad,off", CASES)
def test_rope(rows, heads, d, rot, pairs, norm, hpad, rpad, off, b16):
    import torch

    rng = np.random.default_rng(rows * 7919 + d)
    hs, ld = d + hpad, heads * (d + hpad) + rpad
    dt = torch.bfloat16 if b16 else torch.float32
    flat, view = buffer(rows, ld, off, dt, float("nan"))
    x = torch.from_numpy(rng.normal(0, 2, (rows, heads, d)).astype(np.float32)).to(dt)
    for h in range(heads):
        view[:, h * hs:h * hs + d] = x[:, h].cuda()
    one = norm and heads % 2 == 1  # one weight for all heads, or a row each
    nw = torch.from_numpy((1 + 0.2 * rng.normal(0, 1, (1 if one else heads, d))).astype(np.float32)) if norm else None
    tn = nw.cuda() if norm else None
    pos = rng.integers(0, 100000, rows).astype(np.int32)
    freq = (10000.0 ** -(np.arange(rot // 2) / max(rot // 2, 1))).astype(np.float32)
    tp, tf = torch.from_numpy(pos).cuda(), torch.from_numpy(freq).cuda() if rot else None
    n, ldy, ldb = heads * d, heads * d + 4, heads * d + 12
    y, yv = buffer(rows, ldy, 4, torch.float32, 7.0)
    yb, ybv = buffer(rows, ldb, 4, torch.bfloat16, 7.0)
    f = D.lib().dr_rope_bf16 if b16 else D.lib().dr_rope
    es = flat.element_size()
    call = lambda py, pb: f(flat.data_ptr() + off * es, ld, hs, D.ptr(tn), 0 if one else d, 1e-6, D.ptr(tp), D.ptr(tf), 1.25, int(pairs), py, ldy, pb, ldb, rows,
                            heads, d, rot, D.stream_ptr())
    call(y.data_ptr() + 16, yb.data_ptr() + 8)
    torch.cuda.synchronize()
    want, bound = reference(x.double().numpy(), nw.double().numpy() if norm else None, 1e-6, pos, freq, 1.25, pairs, rot)
    want, bound = want.reshape(rows, n), bound.reshape(rows, n)
    got, gotb = yv.double().cpu().numpy(), ybv.double().cpu().numpy()
    assert (np.abs(got[:, :n] - want) <= bound).all(), float((np.abs(got[:, :n] - want) - bound).max())
    assert (np.abs(gotb[:, :n] - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()
    assert (got[:, n:] == 7).all() and (gotb[:, n:] == 7).all() and (y[:4] == 7).all() and (y[4 + rows * ldy:] == 7).all() and (yb[4 + rows * ldb:] == 7).all()
    # one output alone has the same bits
    y1, y1v = buffer(rows, ldy, 4, torch.float32, 3.0)
    call(y1.data_ptr() + 16, None)
    y2, y2v = buffer(rows, ldb, 4, torch.bfloat16, 3.0)
    call(None, y2.data_ptr() + 8)
    torch.cuda.synchronize()
    assert torch.equal(y1v[:, :n], yv[:, :n]) and torch.equal(y2v[:, :n], ybv[:, :n])


@pytest.mark.parametrize("d,rot,pairs", [(64, 64, False), (256, 64, True), (24, 12, False), (200, 200, True)])
def test_in_place(d, rot, pairs):
    """y over an f32 x, yb over a bf16 x: the bits of separate buffers."""
    import torch

    rows, heads = 37, 6
    n = heads * d
    pos, freq = torch.arange(rows, dtype=torch.int32, device="cuda"), torch.rand(rot // 2, device="cuda")
    nw = 1 + 0.1 * torch.randn(heads, d, device="cuda")
    for dt, f in ((torch.float32, D.lib().dr_rope), (torch.bfloat16, D.lib().dr_rope_bf16)):
        x = torch.randn(rows, n, device="cuda").to(dt)
        out = torch.zeros_like(x)
        b16 = dt == torch.bfloat16
        tail = (rows, heads, d, rot, D.stream_ptr())
        head = lambda t: (D.ptr(t), n, d, D.ptr(nw), d, 1e-6, D.ptr(pos), D.ptr(freq), 1.0, int(pairs))
        f(*head(x), *((None, 0, D.ptr(out), n) if b16 else (D.ptr(out), n, None, 0)), *tail)
        f(*head(x), *((None, 0, D.ptr(x), n) if b16 else (D.ptr(x), n, None, 0)), *tail)
        torch.cuda.synchronize()
        assert torch.equal(x, out)


def test_far_and_negative_positions():
    import torch

    pos = np.array([0, 1, -1, 1000003, -1000003, 2 ** 31 - 1, -2 ** 31, 4096], np.int32)
    rng = np.random.default_rng(8)
    d = rot = 64
    x = rng.normal(0, 1, (len(pos), 2, d)).astype(np.float32)
    freq = np.concatenate([[1.0, 3.0], 500000.0 ** -(np.arange(30) / 30)]).astype(np.float32)
    tx, tp, tf = (torch.from_numpy(a).cuda() for a in (x, pos, freq))
    y = torch.zeros(len(pos), 2 * d, device="cuda")
    D.lib().dr_rope(D.ptr(tx), 2 * d, d, None, 0, 0.0, D.ptr(tp), D.ptr(tf), 1.0, 0, D.ptr(y), 2 * d, None, 0, len(pos), 2, d, rot, D.stream_ptr())
    torch.cuda.synchronize()
    want, bound = reference(x.astype(np.float64), None, 0.0, pos, freq, 1.0, False, rot)
    got = y.double().cpu().numpy().reshape(want.shape)
    assert (np.abs(got - want) <= bound).all(), float((np.abs(got - want) - bound).max())


def test_rows_keep_to_themselves():
    """Zeros, infinities and NaN in one head: every other head has the bits it has without them."""
    import torch

    rows, heads, d = 6, 5, 128
    x = torch.randn(rows, heads * d, device="cuda")
    nw, pos, freq = torch.ones(d, device="cuda"), torch.arange(rows, dtype=torch.int32, device="cuda"), torch.rand(d // 2, device="cuda")
    outs = []
    for bad in (False, True):
        if bad:
            x[1, d:2 * d] = 0
            x[2, 3] = float("inf")
            x[4, 4 * d + 100] = float("nan")
        y = torch.zeros(rows, heads * d, device="cuda")
        D.lib().dr_rope(D.ptr(x), heads * d, d, D.ptr(nw), 0, 1e-6, D.ptr(pos), D.ptr(freq), 1.0, 0, D.ptr(y), heads * d, None, 0, rows, heads, d, d, D.stream_ptr())
        torch.cuda.synchronize()
        outs.append(y.view(rows, heads, d))
    a, b = outs
    touched = {(1, 1), (2, 0), (4, 4)}
    for r in range(rows):
        for h in range(heads):
            assert (r, h) in touched or torch.equal(a[r, h], b[r, h])
    assert (b[1, 1] == 0).all() and torch.isnan(b[4, 4]).any() and not torch.isfinite(b[2, 0]).all()
