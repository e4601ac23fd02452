"""The cache in 8 bits and attention over it, restated in 64 bits from the header's text, and device buffers for them."""
import numpy as np

import dramamoe as D

BLOCK = 64
U = 2.0 ** -24


def v_place(t):
    """Byte of token t in a block's row of vq: token 16 a + 4 b + c at 16 b + 4 a + c."""
    return 16 * (t % 16 // 4) + 4 * (t // 16) + t % 4


class Cache:
    """Pages on the host as integers [pages, hkv, 64, d] in token order, with the sequences' tables."""

    def __init__(self, rng, blocks, hkv, d, spare=2, maxp=None, content="full"):
        """blocks: the pages of each sequence; content "full": every place holds a number, "none": zeros of scale 0."""
        self.hkv, self.d, self.seqs = hkv, d, len(blocks)
        self.pages = sum(blocks) + spare
        self.maxp = maxp or max(max(blocks), 1)
        order, at = rng.permutation(self.pages), 0
        self.table = np.full((self.seqs, self.maxp), -1, np.int32)
        for i, n in enumerate(blocks):
            self.table[i, :n] = order[at:at + n]
            at += n
        shape = (self.pages, hkv, BLOCK, d)
        if content == "full":
            self.k = np.clip(np.rint(rng.normal(0, 40, shape)), -127, 127)
            self.v = np.clip(np.rint(rng.normal(0, 40, shape)), -127, 127)
            self.ks = np.exp(rng.normal(-3, 0.5, shape[:2])).astype(np.float32)
            self.vs = np.exp(rng.normal(-3, 0.5, shape[:2])).astype(np.float32)
        else:
            self.k, self.v = np.zeros(shape), np.zeros(shape)
            self.ks, self.vs = np.zeros(shape[:2], np.float32), np.zeros(shape[:2], np.float32)

    def pack(self):
        k = (self.k + 128).astype(np.uint8).reshape(self.pages, self.hkv, BLOCK, self.d // 16, 16).transpose(0, 1, 3, 2, 4)
        v = np.empty((self.pages, self.hkv, self.d, BLOCK), np.uint8)
        for t in range(BLOCK):
            v[..., v_place(t)] = self.v[:, :, t] + 128
        return np.ascontiguousarray(k), v

    def unpack(self, kq, vq):
        k = kq.astype(np.int64).transpose(0, 1, 3, 2, 4).reshape(self.k.shape) - 128
        v = np.stack([vq[..., v_place(t)].astype(np.int64) for t in range(BLOCK)], 2) - 128
        return k, v

    def tokens(self, i, n, h):
        """(k, v, present) of the first n tokens of sequence i, head h, in float64."""
        k, v, here = np.zeros((n, self.d)), np.zeros((n, self.d)), np.zeros(n, bool)
        for b in range((n + BLOCK - 1) // BLOCK):
            p = self.table[i, b] if b < self.maxp else -1
            if not 0 <= p < self.pages:
                continue
            m = min(BLOCK, n - b * BLOCK)
            k[b * BLOCK:b * BLOCK + m] = self.k[p, h, :m] * np.float64(self.ks[p, h])
            v[b * BLOCK:b * BLOCK + m] = self.v[p, h, :m] * np.float64(self.vs[p, h])
            here[b * BLOCK:b * BLOCK + m] = True
        return k, v, here

    def append(self, k, v, start, lens):
        """k, v [rows, hkv, d] float64 into the cache, as the header says."""
        for x, ints, scale in ((k, self.k, self.ks), (v, self.v, self.vs)):
            for i in range(self.seqs):
                n = start[i + 1] - start[i]
                first = lens[i] - n
                for b in range(max(first, 0) // BLOCK, (lens[i] + BLOCK - 1) // BLOCK if n else 0):
                    p = self.table[i, b] if b < self.maxp else -1
                    if not 0 <= p < self.pages:
                        continue
                    t0, t1 = max(first - b * BLOCK, 0), min(lens[i] - b * BLOCK, BLOCK)
                    r = start[i] + b * BLOCK + t0 - first
                    for h in range(self.hkv):
                        x1 = x[r:r + t1 - t0, h]
                        top, s = np.abs(x1).max(), scale[p, h]
                        if not np.isfinite(x1).all() or (t0 and not np.isfinite(s)):
                            scale[p, h], ints[p, h, t0:t1] = np.nan, 0
                            continue
                        if t0 == 0 or s == 0:
                            s = np.float32(top / 127)
                        else:
                            old = ints[p, h, :t0]
                            while top > 127 * np.float64(s):
                                s, old = np.float32(s * 2), old / 2
                            ints[p, h, :t0] = np.rint(old)
                        scale[p, h] = s
                        ints[p, h, t0:t1] = np.clip(np.rint(x1 / np.float64(s)), -127, 127) if s > 0 else 0


class DevCache:
    """A Cache's buffers on the device; guard bytes behind each."""

    def __init__(self, c):
        import torch

        self.c = c
        kq, vq = c.pack()
        up = lambda a: torch.from_numpy(np.ascontiguousarray(a)).cuda()
        self.kq, self.vq, self.ks, self.vs, self.table = up(kq), up(vq), up(c.ks), up(c.vs), up(c.table)

    def args(self):
        P = D.ptr
        return P(self.table), self.c.maxp, P(self.kq), P(self.ks), P(self.vq), P(self.vs), self.c.pages

    def host(self):
        k, v = self.c.unpack(self.kq.cpu().numpy(), self.vq.cpu().numpy())
        return k, v, self.ks.cpu().numpy(), self.vs.cpu().numpy()


def ints(v):
    import torch

    return torch.tensor(v, dtype=torch.int32, device="cuda")


def sums(rows):
    return [0] + [int(x) for x in np.cumsum(rows)]


def attention(c, q, start, lens, scale, gate):
    """(y, bound) [rows, hq, d] in float64; rows of no sequence NaN.  q and gate [rows, hq, d] float64.

    Bound, U an fp32 rounding: a score is a sum of d exact products, in fp32 with a rounding (up to 2 U) a term, and two factors: (2 d + 4) U
    of the sum of the products' magnitudes Z.  Its distance to the maximum (and 15, and the v scale's logarithm) is at most 300 where
    the weight counts: 300 U, its power of two 2 U: rho = (2 d + 310) U max(Z, 1).  A weight is
    rounded to fp16 by 2^-11, or where small by half of fp16's least step, 2^-25, of a value that stands for at least 2^-4 of a reference not above
    the largest weight: 2^-29 of it, in units of the largest v scale.  Weights and their sum share rho; the sums over n tokens round 2 n U.  Then the
    division, the gate (exp, sum, division: 8 U), and one rounding to bf16, 2^-8."""
    rows, hq, d = q.shape
    y, bound = np.full(q.shape, np.nan), np.full(q.shape, np.nan)
    g = hq // c.hkv
    for i in range(c.seqs):
        n = start[i + 1] - start[i]
        for h in range(c.hkv if n else 0):
            k, v, here = c.tokens(i, max(lens[i], 0), h)
            unit = np.abs(v).max() if len(v) else 0
            for r in range(n):
                p = lens[i] - n + r
                on = here[:p + 1] if p >= 0 else here[:0]
                kk, vv = k[:len(on)][on], v[:len(on)][on]
                for a in range(h * g, (h + 1) * g):
                    row = start[i] + r
                    if not len(kk):
                        y[row, a], bound[row, a] = 0, 0
                        continue
                    qq = q[row, a]
                    z = scale * (kk @ qq)
                    w = np.exp(z - z.max())
                    w /= w.sum()
                    o, mag = w @ vv, w @ np.abs(vv)
                    rho = (2 * d + 310) * U * max(1, (abs(scale) * (np.abs(kk) @ np.abs(qq))).max())
                    e = mag * (2.0 ** -11 + 2 * rho + (2 * len(kk) + 20) * U) + len(kk) * 2.0 ** -29 * unit
                    if gate is not None:
                        s = 1 / (1 + np.exp(-gate[row, a]))
                        o, e = o * s, e * s
                    y[row, a], bound[row, a] = o, e + 2.0 ** -8 * (np.abs(o) + e)
    return y, bound
