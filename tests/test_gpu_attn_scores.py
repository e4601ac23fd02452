"""dr_attn_kv8 where scores are so large that fp32 rounds them to whole octaves.

Every key has one element that is not zero, an integer n, and every query one, so that a score is one product, rounded alike wherever two tokens
share n and their blocks a scale: the softmax is the mean of v over the tokens of the largest product that a row sees, all others vanish (two
neighbouring integers are 2^24 / 127 octaves apart or more).

Tolerance, U = 2^-24: a weight's exponent is the sum of two terms up to 16 and a logarithm (1 ulp), 2^-20 and 2 ulp of its power of two: 16 U; the weight is rounded to
fp16 by 2^-11; the sums over at most n tied tokens round 2 n U, the waves' and splits' joins 16 U, the division 2 U; then bf16, 2^-8."""
import numpy as np
import pytest

from test_gpu_attn_kv8 import Call, cache

pytestmark = pytest.mark.gpu
U = 2.0 ** -24

# rows of each sequence, tokens each has with them, hq, hkv, d: few columns in one block of threads, in several, split; tiles of four
# and of eight waves, whole, folded and split
SHAPES = [([1], [300], 4, 2, 64), ([3], [3000], 40, 2, 64), ([5, 2], [1300, 70], 20, 4, 256), ([30, 7], [330, 900], 8, 2, 128), ([100], [700], 8, 2, 192),
          ([300], [1000], 8, 2, 128), ([300], [2700], 8, 1, 256), ([600], [600], 8, 1, 64), ([700], [900], 64, 1, 128), ([1500], [1500], 32, 1, 32)]


def one_product_scores(rows, lens, hq, hkv, d, octaves, seed):
    """(call, n [seq][hkv, tokens], sign [rows, hq]): the largest score is `octaves` powers of two."""
    import torch

    rng = np.random.default_rng(seed)
    c = cache(seed, lens, hkv, d)
    c.k[:] = 0
    c.k[:, :, :, 3] = rng.integers(-126, 127, c.k.shape[:3])
    c.ks[:] = 2.0 ** -5
    call = Call(c, rows, lens, hq, scale=0.37, seed=seed)
    q = np.zeros((call.total, hq, d))
    # 100 2^-5 scale log2(e) |q| is about 2^octaves
    q[:, :, 3] = np.exp2(octaves) / (100 * 2.0 ** -5 * 0.37 * np.log2(np.e)) * rng.uniform(1, 2, (call.total, hq)) * rng.choice([-1, 1], (call.total, hq))
    call.q[:, :hq * d] = torch.from_numpy(q.reshape(call.total, -1)).to(torch.bfloat16).cuda()
    n = [np.stack([c.k[c.table[i, :(m + 63) // 64], h, :, 3].reshape(-1)[:m] for h in range(hkv)]) for i, m in enumerate(lens)]
    return call, n, np.sign(q[:, :, 3])


def means(call, n, sign):
    """(y, |y| summed, tied tokens) of the tokens with the largest product, float64."""
    c, hq = call.c, call.hq
    y, mag, ties = np.zeros((call.total, hq, c.d)), np.zeros((call.total, hq, c.d)), np.ones((call.total, hq, 1))
    for i, rows in enumerate(call.rows):
        for h in range(c.hkv):
            v = c.tokens(i, call.lens[i], h)[1]
            for s in (-1, 1):
                for r in range(rows):
                    p = call.lens[i] - rows + r
                    z = s * n[i][h, :p + 1]
                    top = np.flatnonzero(z == z.max())
                    g = [a for a in range(h * (hq // c.hkv), (h + 1) * (hq // c.hkv)) if sign[call.start[i] + r, a] == s]
                    row = call.start[i] + r
                    y[row, g], mag[row, g], ties[row, g] = v[top].mean(0), np.abs(v[top]).mean(0), len(top)
    return y, mag, ties


@pytest.mark.parametrize("octaves", [21, 25, 28, 36, 90])
@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
def test_scores_far_from_zero(rows, lens, hq, hkv, d, octaves):
    import torch

    call, n, sign = one_product_scores(rows, lens, hq, hkv, d, octaves, octaves + d)
    got = call.run()
    torch.cuda.synchronize()
    y, mag, ties = means(call, n, sign)
    got = got[:, :hq * d].double().cpu().numpy().reshape(y.shape)
    e = mag * (2.0 ** -11 + (34 + 2 * ties) * U)
    bad = ~(np.abs(got - y) <= e + 2.0 ** -8 * (np.abs(y) + e))
    assert not bad.any(), (int(bad.sum()), bad.size, got[bad][:4], y[bad][:4])


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
def test_far_columns_leave_the_others_alone(rows, lens, hq, hkv, d):
    """One row's scores far from zero: every other row keeps its bits."""
    import torch

    call = Call(cache(61, lens, hkv, d), rows, lens, hq)
    y = call.run()
    at = rows[0] - 1
    call.q[at] *= 2.0 ** 30
    z = call.run()
    torch.cuda.synchronize()
    z[at] = y[at]
    assert torch.equal(z, y)


def overflow(rows, lens, hq, hkv, d, blocks, sign):
    """A call in which every score of `blocks` of sequence 0 passes fp32 with the given sign, (row, query) alike, and others are of the common size."""
    c = cache(71, lens, hkv, d)
    call = Call(c, rows, lens, hq, scale=0.1)
    call.q[:, :hq * d] = call.q[:, :hq * d].abs() + 1
    import torch

    for b in blocks:
        p = int(c.table[0, b])
        call.dc.ks[p] = 1e38
        # all of a block's k of one sign, 3 or more (stored with 128 added)
        k = call.dc.kq[p].to(torch.int32) - 128
        call.dc.kq[p] = (sign * k.abs().clamp(min=3) + 128).to(torch.uint8)
    return c, call


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
def test_scores_past_fp32(rows, lens, hq, hkv, d):
    """A block of scores that are +infinity in fp32: NaN for the rows that see it.  Of -infinity: as if the block was not there.  Nothing but such scores: NaN.
    The others keep their bits."""
    import torch

    n = hq * d
    blocks = sorted({0, (lens[0] - 1) // 128, (lens[0] - 1) // 64})
    plain = overflow(rows, lens, hq, hkv, d, [], 1)[1].run()
    for b in blocks:
        c, call = overflow(rows, lens, hq, hkv, d, [b], 1)
        y = call.run()
        torch.cuda.synchronize()
        seen = min(max(b * 64 - (lens[0] - rows[0]), 0), rows[0])
        assert torch.isnan(y[seen:rows[0], :n]).all() and torch.equal(y[:seen], plain[:seen]) and torch.equal(y[rows[0]:], plain[rows[0]:])
        c, call = overflow(rows, lens, hq, hkv, d, [b], -1)
        y = call.run()
        torch.cuda.synchronize()
        assert torch.equal(y[:seen], plain[:seen]) and torch.equal(y[rows[0]:], plain[rows[0]:])
        alone = max(0, min(rows[0], 64 - (lens[0] - rows[0]))) if b == 0 else 0  # rows that see that block only
        assert torch.isnan(y[:alone, :n]).all()
        page, c.table[0, b] = int(c.table[0, b]), -1
        want, bound = call.reference()
        c.table[0, b] = page
        got = y[:, :n].double().cpu().numpy().reshape(want.shape)
        own = slice(alone, call.start[-1])
        assert (np.abs(got[own] - want[own]) <= bound[own]).all()
    c, call = overflow(rows, lens, hq, hkv, d, range((lens[0] + 63) // 64), -1)
    y = call.run()
    torch.cuda.synchronize()
    assert torch.isnan(y[:rows[0], :n]).all() and torch.equal(y[rows[0]:], plain[rows[0]:])


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
def test_products_of_nothing(rows, lens, hq, hkv, d):
    """Queries of zeros on k scales next to fp32's largest, and a scale for the scores that is: all weights alike."""
    import torch

    c = cache(73, lens, hkv, d)
    c.ks[::2] = 3.4e38
    for scale in (3.4e38, 1.0):
        call = Call(c, rows, lens, hq, scale=scale)
        call.q[:, :hq * d] = 0
        y = call.run()
        torch.cuda.synchronize()
        call.check(y)
