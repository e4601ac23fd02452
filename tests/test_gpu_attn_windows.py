"""dr_attn_kv8 where a wave (few columns) or a block of threads (tiles) walks over more cached blocks than it has pages and scales of at once (64), and cuts
that no other test takes.  max_len 1 keeps a long sequence in one piece; rows of no sequence behind a small one have the host cut
for a large one.  test_attn_cuts.py checks that each case takes the cut it is here for.  Tolerances: kv8_helpers.attention."""
import numpy as np
import pytest

from test_gpu_attn_kv8 import Call, cache

pytestmark = pytest.mark.gpu

# cut, blocks in a row, (rows, tokens, hq, hkv, d), gate, rows behind, max_len
WINDOWS = [
    ("few 16 d64", 67, ([1], [17000], 4, 2, 64), True, 0, 1), ("few 16 d128", 67, ([1, 1], [17011, 70], 8, 2, 128), False, 0, 1), ("few 16 d192", 65, ([1], [16500], 2, 1, 176), False, 0, 1),
    ("few 16 d256", 130, ([2], [33100], 4, 1, 256), False, 0, 1), ("few 32 d64", 130, ([5, 1], [33030, 1], 8, 2, 48), False, 1, 1), ("few 32 d128", 65, ([3], [16449], 8, 1, 80), True, 0, 1),
    ("tiles 4 d64 several", 66, ([530], [4200], 4, 1, 64), False, 0, 1), ("tiles 4 d64 several", 130, ([530, 3], [8300, 3], 4, 1, 32), True, 0, 1), ("tiles 4 d128 several", 130, ([530], [8260], 4, 1, 128), False, 0, 1),
    ("tiles 4 d192 several", 66, ([530], [4190], 4, 1, 160), False, 0, 1), ("tiles 4 d256 several", 130, ([530], [8300], 4, 1, 256), False, 0, 1),
    ("tiles 8 d64 several folded", 130, ([70, 9], [8300, 90], 16, 1, 64), False, 2900, 1), ("tiles 8 d128 several folded", 66, ([70], [4200], 16, 1, 128), True, 2900, 1),
    ("tiles 8 d128 several folded", 130, ([90], [8300], 16, 1, 96), False, 2900, 1), ("tiles 8 d64 several", 66, ([70, 9], [4200, 90], 16, 1, 48), False, 4300, 1),
    ("tiles 8 d128 several", 130, ([90, 20], [8300, 500], 16, 1, 128), False, 4300, 1), ("tiles 8 d128 several", 195, ([40], [12440], 16, 1, 112), True, 4300, 1),
]


def many(first, others, seqs, *rest):
    """One sequence of (rows, tokens) and others alike."""
    return ([first[0]] + [others[0]] * (seqs - 1), [first[1]] + [others[1]] * (seqs - 1), *rest)


# cuts that the other files' cases leave out
OTHERS = [
    ("few 16 d192 split", 1, ([1], [3000], 4, 1, 192), True, 0, None), ("few 16 d192 several split", 1, ([5], [2900], 8, 1, 144), False, 0, None), ("few 16 d256 split", 1, ([1], [1098], 1, 1, 240), False, 0, None),
    ("few 32 d128 split", 1, ([6], [1171], 4, 1, 80), True, 0, None), ("few 32 d64 split", 1, ([5], [1159], 4, 1, 32), False, 1, None),
    ("tiles 4 d128", 1, ([33], [35], 2, 1, 80), True, 1, None), ("tiles 4 d192", 1, many((5, 7), (1, 3), 40, 64, 4, 160), False, 0, None), ("tiles 4 d256", 1, many((39, 42), (13, 21), 200, 2, 1, 240), True, 1, None),
    ("tiles 4 d192 split", 3, many((71, 2183), (23, 1091), 9, 2, 2, 160), False, 0, None), ("tiles 4 d256 split", 4, many((56, 708), (18, 354), 40, 4, 2, 240), False, 0, None),
    ("tiles 8 d128", 1, many((5, 8), (1, 4), 200, 64, 2, 80), False, 1, None), ("tiles 8 d128 folded", 1, many((5, 6), (1, 3), 200, 32, 1, 80), True, 0, None),
    ("tiles 8 d64", 1, many((27, 37), (9, 18), 200, 16, 2, 32), False, 0, None), ("tiles 8 d64 folded", 1, many((22, 23), (7, 11), 200, 8, 1, 32), False, 0, None),
    ("tiles 8 d128 several", 5, ([70, 9], [300, 90], 16, 1, 128), True, 4300, 300), ("tiles 8 d128 several split", 40, ([3], [5025], 16, 1, 80), False, 2900, None),
    ("tiles 8 d64 several split", 71, ([9], [9000], 16, 1, 48), True, 2900, None),
]


def run(case, max_rows):
    cut, blocks, (rows, lens, hq, hkv, d), gate, behind, max_len = case
    import torch

    call = Call(cache(sum(lens) + d, lens, hkv, d), rows, lens, hq, gate=gate, behind=behind, max_len=max_len, max_rows=max_rows)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)


def most_rows(case):
    """What the host says of the rows of a sequence: as many as the call has where rows stand behind it."""
    rows, behind = case[2][0], case[4]
    return sum(rows) + behind if behind > 1 else None


@pytest.mark.parametrize("case", WINDOWS + OTHERS)
def test_windows(case):
    run(case, most_rows(case))


@pytest.mark.parametrize("case", [WINDOWS[0], WINDOWS[3], WINDOWS[7], WINDOWS[10], WINDOWS[12], WINDOWS[15]])
def test_pages_of_every_window_count(case):
    """One block of each window of 64, and of the last, has no number: the rows that see it have none, and with it gone from the table the reference's values."""
    import torch

    cut, blocks, (rows, lens, hq, hkv, d), gate, behind, max_len = case
    c = cache(sum(lens) + d, lens, hkv, d)
    call = Call(c, rows, lens, hq, gate=gate, behind=behind, max_len=max_len, max_rows=most_rows(case))
    nb, n = (lens[0] + 63) // 64, rows[0]
    y = call.run()
    for b in sorted({0, 5, 63, 64, 70, 127, 128, 200, 255, 256, 257, nb // 2, nb - 1}):
        if b >= nb:
            continue
        p = int(c.table[0, b])
        old = float(call.dc.ks[p, 0])
        call.dc.ks[p, 0] = float("nan")
        z = call.run()
        torch.cuda.synchronize()
        call.dc.ks[p, 0] = old
        seen, g = min(max(b * 64 - (lens[0] - n), 0), n), hq // hkv
        z3, y3 = (t[:, :hq * d].view(-1, hq, d) for t in (z, y))
        assert torch.isnan(z3[seen:n, :g]).all() and torch.equal(z3[:seen], y3[:seen]) and torch.equal(z3[n:], y3[n:]) and torch.equal(z3[:n, g:], y3[:n, g:]), b


@pytest.mark.parametrize("rows,lens,hq,hkv,d", [([1], [4000], 4, 1, 64), ([3], [2000], 16, 1, 256), ([2], [700], 16, 1, 128), ([5], [3000], 5, 1, 96)])
@pytest.mark.parametrize("octaves", [26.5, 29.5, 33.5])
def test_small_weights_with_few_columns(rows, lens, hq, hkv, d, octaves):
    """One token without a value of its own outweighs all others by far, which decide the result.  Few columns hold a weight as 2^15 times its ratio to
    the largest: what fp16's least step leaves out is 2^-25 of 2^15, in units of a power of two up to twice the largest v scale: 2^-39 of that scale and
    an integer (2^-29 in kv8_helpers.attention, which tiles need)."""
    import torch

    c = cache(25, lens, hkv, d)
    first = int(c.table[0, 0])
    c.k[:], c.v[:] = -60, np.minimum(np.abs(c.v) + 1, 127)
    c.k[first, :, 0], c.v[first, :, 0] = 60, 0
    c.ks[:], c.vs[:] = 2.0 ** -4, 0.02
    call = Call(c, rows, lens, hq, scale=octaves * np.log(2) / (120 * 2.0 ** -4 * d))
    call.q[:, :hq * d] = 1.0
    y = call.run()
    torch.cuda.synchronize()
    want, bound = call.reference()
    n = np.array([lens[0] - rows[0] + r + 1 for r in range(rows[0])])[:, None, None]
    v = np.abs(c.tokens(0, lens[0], 0)[1]).max()
    bound = bound - (1 + 2.0 ** -8) * n * v * (2.0 ** -29 - 2.0 ** -39)
    got = y[:, :hq * d].double().cpu().numpy().reshape(want.shape)
    assert (bound < 0.5 * np.abs(want)).all() and (np.abs(got - want) <= bound).all()
