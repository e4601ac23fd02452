"""dr_kv8_append, dr_kv8_append_bf16 and dr_kv8_read against the header's text in 64 bits: integers, scales and the values read back
have to be equal, since every rounding is defined (scales fl(A / 127) or doublings, integers from the exact quotient, one product on
reading)."""
import numpy as np
import pytest

import dramamoe as D
from kv8_helpers import BLOCK, Cache, DevCache, ints, sums

pytestmark = pytest.mark.gpu


def rows_dev(x, b16, ld, fill=9.0):
    """[rows, n] on the device in rows of ld elements, the rest `fill`."""
    import torch

    t = torch.full((x.shape[0], ld), fill, dtype=torch.bfloat16 if b16 else torch.float32, device="cuda")
    t[:, :x.shape[1]] = torch.from_numpy(x).to(t.dtype).cuda()
    return t


def make_rows(rng, rows, hkv, d, b16, spread=1.0):
    import torch

    x = rng.normal(0, 1, (rows, hkv, d)) * np.exp(rng.normal(0, spread, (rows, 1, 1)))
    t = torch.from_numpy(x.astype(np.float32))
    return (t.to(torch.bfloat16) if b16 else t).double().numpy()


def append(dc, k, v, b16, start, lens, pad=0, stream=None):
    """k, v [rows, hkv, d] through the library; the strides have `pad` elements more than the heads."""
    rows, n = k.shape[0], dc.c.hkv * dc.c.d
    ld = n + pad
    tk, tv = (rows_dev(x.reshape(rows, n), b16, ld) for x in (k, v))
    ts, tl = ints(start), ints(lens)
    f = D.lib().dr_kv8_append_bf16 if b16 else D.lib().dr_kv8_append
    f(D.ptr(tk), ld, D.ptr(tv), ld, D.ptr(ts), D.ptr(tl), *dc.args(), rows, dc.c.seqs, dc.c.hkv, dc.c.d, stream or D.stream_ptr())
    return tk, tv, ts, tl


def check_cache(dc, c):
    k, v, ks, vs = dc.host()
    assert np.array_equal(ks.view(np.uint32)[~np.isnan(ks)], c.ks.view(np.uint32)[~np.isnan(c.ks)]) and np.array_equal(np.isnan(ks), np.isnan(c.ks))
    assert np.array_equal(vs.view(np.uint32)[~np.isnan(vs)], c.vs.view(np.uint32)[~np.isnan(c.vs)]) and np.array_equal(np.isnan(vs), np.isnan(c.vs))
    return k, v


def check_tokens(c, k, v, start, lens):
    """Every place of a sequence up to its length; what lies behind is of no use."""
    for i in range(c.seqs):
        for b in range((max(lens[i], 0) + BLOCK - 1) // BLOCK):
            p = c.table[i, b] if b < c.maxp else -1
            if 0 <= p < c.pages:
                m = min(BLOCK, lens[i] - b * BLOCK)
                assert np.array_equal(k[p, :, :m], c.k[p, :, :m]) and np.array_equal(v[p, :, :m], c.v[p, :, :m]), (i, b)


def untouched(c, before, k, v, start, lens):
    """Pages that no appended token lies in keep every byte."""
    used = set()
    for i in range(c.seqs):
        n = start[i + 1] - start[i]
        if n:
            used |= {int(c.table[i, b]) for b in range(max(lens[i] - n, 0) // BLOCK, (lens[i] + BLOCK - 1) // BLOCK) if b < c.maxp}
    for p in set(range(c.pages)) - used:
        assert np.array_equal(k[p], before[0][p]) and np.array_equal(v[p], before[1][p]), p


CASES = [
    # rows of each sequence, tokens each has with them, hkv, d, rows of no sequence behind, spread of the rows' sizes
    ([1], [1], 1, 16, 0, 0.0), ([1], [64], 2, 64, 0, 1.0), ([1], [65], 2, 64, 0, 1.0), ([64], [64], 1, 128, 0, 0.0), ([63], [63], 3, 48, 0, 1.0),
    ([65], [65], 2, 80, 0, 1.0), ([200], [333], 2, 256, 0, 1.0), ([1] * 70, [1 + 7 * i for i in range(70)], 2, 32, 3, 2.0),
    ([3, 0, 5, 129, 0, 1], [3, 100, 64, 140, 0, 700], 4, 96, 2, 2.0), ([2, 4, 3], [0, 2, 3], 2, 64, 1, 1.0),
    ([9, 0, 0, 70, 0, 0] + [1] * 20, [9, 5, 0, 200, 1, 0] + [64 * i for i in range(1, 21)], 2, 128, 1, 2.0), ([13, 0, 0, 0], [50, 9, 0, 0], 3, 256, 0, 1.0),
    ([130], [130], 1, 240, 0, 3.0), ([17] * 9, [17 + 61 * i for i in range(9)], 5, 112, 0, 2.0),
]


@pytest.mark.parametrize("b16", [False, True])
@pytest.mark.parametrize("rows,lens,hkv,d,behind,spread", CASES)
def test_append_and_read(rows, lens, hkv, d, behind, spread, b16):
    import torch

    rng = np.random.default_rng(sum(rows) * 31 + d + hkv)
    c = Cache(rng, [(n + 63) // 64 for n in lens], hkv, d)
    dc, start, total = DevCache(c), sums(rows), sum(rows) + behind
    before = (c.k.copy(), c.v.copy())
    k, v = make_rows(rng, total, hkv, d, b16, spread), make_rows(rng, total, hkv, d, b16, spread)
    for again in range(2):  # a second time changes nothing
        append(dc, k, v, b16, start, lens, pad=8 if d % 32 else 0)
        torch.cuda.synchronize()
        if not again:
            c.append(k, v, start, lens)
        gk, gv = check_cache(dc, c)
        check_tokens(c, gk, gv, start, lens)
        untouched(c, before, gk, gv, start, lens)
    # back: these rows, 0 for those that are no token, the rows behind left alone
    n, ld = hkv * d, hkv * d + 4
    tk, tv = (torch.full((total, ld), 7.0, device="cuda") for _ in range(2))
    ts, tl = ints(start), ints(lens)
    D.lib().dr_kv8_read(D.ptr(ts), D.ptr(tl), *dc.args(), D.ptr(tk), ld, D.ptr(tv), ld, total, c.seqs, hkv, d, D.stream_ptr())
    torch.cuda.synchronize()
    for t, which in ((tk, 0), (tv, 1)):
        want = np.full((total, ld), 7.0, np.float32)
        for i in range(c.seqs):
            for h in range(hkv):
                tok = c.tokens(i, max(lens[i], 0), h)[which]
                for r in range(rows[i]):
                    p = lens[i] - rows[i] + r
                    want[start[i] + r, h * d:(h + 1) * d] = tok[p] if p >= 0 else 0
        assert np.array_equal(t.cpu().numpy(), want)


def test_single_tokens_one_by_one():
    """200 tokens appended alone: scales grow by doublings only, and no element ends a whole step off."""
    import torch

    rng = np.random.default_rng(3)
    c = Cache(rng, [4, 4], 2, 64, content="none")
    dc = DevCache(c)
    size = np.exp(rng.normal(0, 1.5, 200))
    all_k, all_v = [], []
    for t in range(200):
        k, v = (rng.normal(0, size[t], (2, 2, 64)).astype(np.float32).astype(np.float64) for _ in range(2))
        all_k.append(k), all_v.append(v)
        append(dc, k, v, False, [0, 1, 2], [t + 1, t + 1])
        c.append(k, v, [0, 1, 2], [t + 1, t + 1])
    torch.cuda.synchronize()
    gk, gv = check_cache(dc, c)
    check_tokens(c, gk, gv, [0, 1, 2], [200, 200])
    for i in range(2):
        for h in range(2):
            for x, which, sc in ((all_k, 0, c.ks), (all_v, 1, c.vs)):
                got = c.tokens(i, 200, h)[which]
                step = np.repeat([sc[p, h] for p in c.table[i]], 64)[:200, None]
                assert (np.abs(got - np.stack([a[i, h] for a in x])) < step).all()


def test_borders_ties_and_tiny_values():
    """Quotients on the borders between integers (halves, to even), scales that are subnormal or vanish, zeros, the largest floats."""
    import torch

    f = np.float32
    rows = []
    s = f(0.7310585975646973)
    half = np.concatenate([[127 * s], (np.arange(63) - 31.5) * np.float64(s)]).astype(f)  # halves of s: exact ties
    rows.append(half)
    rows.append(np.nextafter(half, f(np.inf)).astype(f)), rows.append(np.nextafter(half, f(-np.inf)).astype(f))
    rows.append(np.linspace(-3e38, 3e38, 64).astype(f)), rows.append(np.zeros(64, f))
    rows.append((np.arange(64) * 2.0 ** -149).astype(f)), rows.append((np.arange(64) * 3e-41).astype(f)), rows.append(np.full(64, -0.0, f))
    rows.append((np.linspace(-1, 1, 64) * 2e-28).astype(f)), rows.append((np.linspace(-1, 1, 64) * 127).astype(f))
    k = np.stack(rows).astype(np.float64)[:, None, :]
    n = len(rows)
    rng = np.random.default_rng(4)
    c = Cache(rng, [1] * n, 1, 64, content="none")
    dc = DevCache(c)
    append(dc, k, -k, False, list(range(n + 1)), [1] * n)
    c.append(k, -k, list(range(n + 1)), [1] * n)
    # a second token three times as large: doublings from each of those scales
    with np.errstate(over="ignore"):
        k2 = np.minimum(np.maximum(3 * k, -3.4e38), 3.4e38).astype(f).astype(np.float64)
    append(dc, k2, k, False, list(range(n + 1)), [2] * n)
    c.append(k2, k, list(range(n + 1)), [2] * n)
    torch.cuda.synchronize()
    gk, gv = check_cache(dc, c)
    check_tokens(c, gk, gv, list(range(n + 1)), [2] * n)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_no_numbers_stay_in_their_block(value):
    """An infinity or NaN: its block and head have scale NaN from then on, all others are as without it; a call that begins
    the block again starts anew."""
    import torch

    rng = np.random.default_rng(5)
    c = Cache(rng, [3], 2, 64)
    dc = DevCache(c)
    k, v = make_rows(rng, 150, 2, 64, False), make_rows(rng, 150, 2, 64, False)
    bad = k.copy()
    bad[70, 1, 5] = value
    append(dc, bad, v, False, [0, 150], [150])
    c.append(bad, v, [0, 150], [150])
    append(dc, k[:1], v[:1], False, [0, 1], [151])  # a later block
    c.append(k[:1], v[:1], [0, 1], [151])
    torch.cuda.synchronize()
    check_cache(dc, c)
    assert np.isnan(c.ks[c.table[0, 1], 1]) and np.isnan(c.ks).sum() == 1 and not np.isnan(c.vs).any()
    append(dc, k[:1], v[:1], False, [0, 1], [100])  # inside the block: it stays
    torch.cuda.synchronize()
    assert np.isnan(dc.host()[2][c.table[0, 1], 1])
    append(dc, k[:40], v[:40], False, [0, 40], [104])  # from its first token on
    c.append(k[:40], v[:40], [0, 40], [104])
    torch.cuda.synchronize()
    gk, gv = check_cache(dc, c)
    check_tokens(c, gk, gv, [0, 40], [104])


def test_blocks_that_are_not_there():
    """Table entries outside the pages, tokens past the table, start values outside the rows: nothing is written for them, 0 is read."""
    import torch

    rng = np.random.default_rng(6)
    c = Cache(rng, [2, 2, 2], 2, 48, maxp=2)
    c.table[0, 1], c.table[1, 0] = c.pages, -7
    dc = DevCache(c)
    before = dc.host()
    rows, lens = [100, 128, 150], [100, 128, 150]
    k, v = make_rows(rng, 378, 2, 48, False), make_rows(rng, 378, 2, 48, False)
    append(dc, k, v, False, sums(rows), lens)
    c.append(k, v, sums(rows), lens)
    torch.cuda.synchronize()
    gk, gv = check_cache(dc, c)
    check_tokens(c, gk, gv, sums(rows), lens)
    untouched(c, before, gk, gv, sums(rows), lens)
    out = [torch.full((378, 96), 5.0, device="cuda") for _ in range(2)]
    ts, tl = ints(sums(rows)), ints(lens)
    D.lib().dr_kv8_read(D.ptr(ts), D.ptr(tl), *dc.args(), D.ptr(out[0]), 96, D.ptr(out[1]), 96, 378, 3, 2, 48, D.stream_ptr())
    torch.cuda.synchronize()
    got = out[0].cpu().numpy()
    assert (got[64:100] == 0).all() and (got[100:164] == 0).all() and (got[228 + 128:] == 0).all() and (got[:64] != 0).any()
    # start beyond the rows, or falling: no row outside the call
    bad = ints([-5, 3, 2, 1 << 30])
    tl = ints([3, 5, 128])
    D.lib().dr_kv8_read(D.ptr(bad), D.ptr(tl), *dc.args(), D.ptr(out[0]), 96, D.ptr(out[1]), 96, 6, 3, 2, 48, D.stream_ptr())
    torch.cuda.synchronize()
    assert np.array_equal(out[0].cpu().numpy()[6:], got[6:])


def test_sizes_beyond_32_bits():
    """A cache whose last pages lie past 2^32 bytes: tokens go to and come from there."""
    import torch

    hkv, d = 8, 128
    pages = (1 << 32) // (hkv * 64 * d) + 3
    kq, vq = (torch.zeros(pages * hkv * 64 * d, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(pages, hkv, device="cuda") for _ in range(2))
    table = ints([[0, pages - 1, 1, pages - 2]])
    k, v = torch.randn(200, hkv * d, device="cuda"), torch.randn(200, hkv * d, device="cuda")
    out = [torch.zeros(200, hkv * d, device="cuda") for _ in range(2)]
    cache = (D.ptr(table), 4, D.ptr(kq), D.ptr(ks), D.ptr(vq), D.ptr(vs), pages)
    ts, tl = ints([0, 200]), ints([200])
    n = hkv * d
    D.lib().dr_kv8_append(D.ptr(k), n, D.ptr(v), n, D.ptr(ts), D.ptr(tl), *cache, 200, 1, hkv, d, D.stream_ptr())
    D.lib().dr_kv8_read(D.ptr(ts), D.ptr(tl), *cache, D.ptr(out[0]), n, D.ptr(out[1]), n, 200, 1, hkv, d, D.stream_ptr())
    torch.cuda.synchronize()
    blk = torch.tensor([0, pages - 1, 1, pages - 2], device="cuda")[torch.arange(200, device="cuda") // 64]
    for x, o, s in ((k, out[0], ks), (v, out[1], vs)):
        assert ((x - o).abs().view(200, hkv, d) <= 0.5001 * s[blk][:, :, None]).all()
    assert int((kq[:(pages - 2) * hkv * 64 * d].view(-1, hkv * 64 * d)[2:] != 0).sum()) == 0
