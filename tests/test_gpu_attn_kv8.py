"""dr_attn_kv8 against softmax(scale q k) v in 64 bits over the values that the cache stands for (kv8_helpers.attention: the tolerances' derivation)."""
import ctypes

import numpy as np
import pytest

import dramamoe as D
from kv8_helpers import Cache, DevCache, attention, ints, sums

pytestmark = pytest.mark.gpu


class Call:
    """One call's inputs; strides with `pad` elements more than the heads, rows of no sequence behind."""

    def __init__(self, c, rows, lens, hq, gate=False, behind=0, seed=0, pad=0, scale=None, qsize=2.0, max_len=None, max_rows=None):
        import torch

        self.c, self.dc, self.rows, self.lens, self.hq = c, DevCache(c), rows, lens, hq
        self.start, self.total, d = sums(rows), sum(rows) + behind, c.d
        rng = np.random.default_rng(seed + 1000 * d + hq)
        self.scale = scale if scale is not None else d ** -0.5
        n = hq * d
        self.ldq, self.ldy, self.hsg, self.ldg = n + 8 * pad, n + 4 * pad, d + 4 * pad, hq * (d + 4 * pad) + 4 * pad
        self.q = torch.full((self.total, self.ldq), float("nan"), dtype=torch.bfloat16, device="cuda")
        self.q[:, :n] = torch.from_numpy(rng.normal(0, qsize, (self.total, n))).to(torch.bfloat16).cuda()
        self.gate = None
        if gate:
            self.gate = torch.full((self.total, self.ldg), float("nan"), device="cuda")
            g = torch.from_numpy(rng.normal(0, 3, (self.total, hq, d)).astype(np.float32)).cuda()
            for h in range(hq):
                self.gate[:, h * self.hsg:h * self.hsg + d] = g[:, h]
        self.max_rows = max(rows) if max_rows is None else max_rows
        self.max_len = max(max(lens), 0) if max_len is None else max_len
        size = D.lib().dr_attn_kv8_ws(self.total, c.seqs, self.max_rows, self.max_len, hq, c.hkv, d)
        assert size > 0
        # scratch holding anything: NaN patterns, and a guard behind it
        self.ws = torch.full((size + 64,), 255, dtype=torch.uint8, device="cuda")
        self.ts, self.tl = ints(self.start), ints(lens)

    def run(self, y=None, stream=None):
        import torch

        if y is None:
            y = torch.full((self.total, self.ldy), 7.0, dtype=torch.bfloat16, device="cuda")
        c = self.c
        D.lib().dr_attn_kv8(D.ptr(self.q), self.ldq, D.ptr(self.ts), D.ptr(self.tl), *self.dc.args(), self.scale, D.ptr(self.gate), self.ldg, self.hsg,
                            D.ptr(self.ws), D.ptr(y), self.ldy, self.total, c.seqs, self.max_rows, self.max_len, self.hq, c.hkv, c.d,
                            stream or D.stream_ptr())
        return y

    def reference(self):
        n, d = self.hq * self.c.d, self.c.d
        q = self.q[:, :n].double().cpu().numpy().reshape(self.total, self.hq, d)
        gate = None
        if self.gate is not None:
            g = self.gate.double().cpu().numpy()
            gate = np.stack([g[:, h * self.hsg:h * self.hsg + d] for h in range(self.hq)], 1)
        return attention(self.c, q, self.start, self.lens, self.scale, gate)

    def check(self, y):
        n = self.hq * self.c.d
        want, bound = self.reference()
        got = y.double().cpu().numpy()
        own = slice(self.start[0], self.start[-1])
        g, w, b = got[own, :n].reshape(-1, self.hq, self.c.d), want[own], bound[own]
        bad = ~(np.abs(g - w) <= b)
        assert not bad.any(), (int(bad.sum()), bad.size, np.argwhere(bad)[:3].tolist(), g[bad][:3], w[bad][:3], b[bad][:3])
        assert (got[self.start[-1]:] == 7).all() and (got[own, n:] == 7).all()
        assert (self.ws[-64:] == 255).all()


def cache(seed, lens, hkv, d, **kw):
    return Cache(np.random.default_rng(seed), [(max(n, 0) + 63) // 64 for n in lens], hkv, d, **kw)


CASES = [
    # rows of each sequence, tokens each has with them, hq, hkv, d, gate, rows of no sequence behind, pad
    ([1], [1], 1, 1, 16, False, 0, 0), ([1], [64], 4, 2, 64, True, 0, 1), ([1], [65], 8, 1, 128, False, 0, 0), ([1], [300], 16, 4, 128, False, 0, 0),
    ([1], [500], 16, 2, 256, True, 0, 1), ([1] * 5, [1, 63, 64, 129, 700], 6, 3, 80, False, 2, 0), ([1, 0, 1, 1], [0, 5, 200, 1], 4, 4, 48, True, 1, 1),
    ([3], [3], 4, 2, 32, False, 0, 0), ([5, 2, 4], [70, 200, 4], 10, 2, 112, True, 0, 0), ([4, 6], [2, 6], 4, 2, 64, False, 0, 0),
    ([33], [33], 3, 3, 64, False, 0, 0), ([100], [100], 8, 2, 128, True, 3, 1), ([70, 0, 1, 129], [150, 64, 300, 129], 5, 1, 96, False, 0, 0),
    ([65], [200], 4, 1, 256, False, 0, 0), ([40, 90], [40, 400], 6, 2, 192, True, 0, 0), ([200], [130], 2, 1, 16, False, 0, 0),
    ([2], [90], 71, 1, 64, False, 0, 0), ([17] * 6, [17 + 40 * i for i in range(6)], 2, 2, 160, False, 5, 0), ([1] * 130, list(range(130)), 2, 1, 64, False, 0, 0),
    ([9] * 70, [9 + 3 * i for i in range(70)], 2, 1, 32, False, 0, 0), ([1], [5000], 4, 2, 128, False, 0, 0), ([1, 1], [9000, 64], 2, 1, 64, True, 0, 0),
    ([20], [4000], 4, 2, 64, False, 0, 0), ([150], [2500], 4, 1, 128, False, 0, 0), ([3], [2100], 16, 1, 240, True, 0, 0),
]


@pytest.mark.parametrize("rows,lens,hq,hkv,d,gate,behind,pad", CASES)
def test_attention(rows, lens, hq, hkv, d, gate, behind, pad):
    import torch

    call = Call(cache(sum(lens) + d, lens, hkv, d), rows, lens, hq, gate=gate, behind=behind, pad=pad)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)
    # the same call gives the same bits, over q's buffer too
    again = call.run()
    torch.cuda.synchronize()
    assert torch.equal(y, again)
    if call.ldq == call.ldy:
        call.run(y=call.q)
        torch.cuda.synchronize()
        n = call.start[-1]
        assert torch.equal(call.q[:n], y[:n])


# every way to cut a call: few columns in one block of threads or several, whole or split, and tiles of four and eight waves, whole or split
CUTS = [
    ([3], [40], 40, 2, 64, True), ([3], [3000], 40, 2, 64, False), ([8], [1500], 12, 2, 128, True), ([5, 2], [1300, 70], 20, 4, 256, True), ([9], [9], 16, 4, 192, False),
    ([30, 7, 0, 12], [30, 7, 5, 900], 8, 2, 128, False), ([30, 7, 0, 12], [30, 7, 5, 900], 8, 2, 256, True), ([100], [100], 8, 2, 256, False), ([140], [700], 4, 1, 64, False),
    ([300], [1000], 8, 2, 64, True), ([300], [1000], 8, 2, 128, False), ([300], [700], 8, 1, 256, True), ([600], [600], 8, 1, 160, False), ([700, 20], [900, 20], 8, 1, 128, False),
    ([20] * 40, [20 + i for i in range(40)], 32, 8, 64, False), ([4] * 300, [1 + i % 9 for i in range(300)], 16, 1, 32, True),
    ([2100], [2100], 8, 1, 96, False), ([1500], [1600], 32, 1, 64, True), ([700, 300, 701], [1000, 300, 701], 32, 1, 128, False), ([1430], [1430], 32, 1, 32, False), ([64] * 9, [64 + 300 * i for i in range(9)], 8, 4, 128, False),
]


@pytest.mark.parametrize("rows,lens,hq,hkv,d,gate", CUTS)
def test_every_cut(rows, lens, hq, hkv, d, gate):
    import torch

    call = Call(cache(31, lens, hkv, d), rows, lens, hq, gate=gate, behind=1, seed=4)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)


@pytest.mark.parametrize("rows,lens,hq,hkv,d,gate", CUTS)
def test_output_in_the_queries_place(rows, lens, hq, hkv, d, gate):
    import torch

    call = Call(cache(51, lens, hkv, d), rows, lens, hq, gate=gate, seed=6)
    y = call.run()
    call.run(y=call.q)
    torch.cuda.synchronize()
    assert torch.equal(call.q, y)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", [([1], [900], 8, 2, 128), ([70], [300], 4, 2, 64), ([1, 3], [2000, 100], 4, 1, 256)])
@pytest.mark.parametrize("max_len", [0, 1, 100000])
def test_any_cut_is_right(rows, lens, hq, hkv, d, max_len):
    """The host's word for the lengths sets the cut only: too small, and as large as a graph's final one."""
    import torch

    call = Call(cache(7, lens, hkv, d), rows, lens, hq, max_len=max_len)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)


def test_scales_of_every_size():
    """Blocks whose scales differ by far more than fp16's range, vanish, or weigh nothing; a scale of zero and a negative one for the scores."""
    import torch

    for scale in (None, 0.0, -0.3):
        c = cache(9, [700, 64], 2, 64)
        for i in range(2):
            for b, p in enumerate(c.table[i]):
                if p >= 0:
                    c.vs[p] = 10.0 ** ((7 * b) % 30 - 15)
                    c.ks[p] = (0, 1e-30, 0.05, 0.02)[b % 4]
        call = Call(c, [1, 2], [700, 64], 4, scale=scale)
        y = call.run()
        torch.cuda.synchronize()
        call.check(y)


def test_peaked_and_flat_weights():
    """Queries so large that one token takes all, and so small that all tokens weigh the same."""
    import torch

    for qsize in (1e-30, 1e-3, 300.0, 1e30):
        call = Call(cache(11, [1500], 1, 64), [2], [1500], 2, qsize=qsize, scale=0.1 if qsize < 1e20 else 1e-29)
        y = call.run()
        torch.cuda.synchronize()
        call.check(y)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", [([1], [4000], 4, 1, 64), ([3], [2000], 16, 1, 256), ([300], [4000], 8, 1, 128), ([600], [2500], 8, 1, 64), ([400], [1500], 8, 1, 256)])
@pytest.mark.parametrize("octaves", [17.5, 21.5, 26.5])
def test_small_weights_add_up(rows, lens, hq, hkv, d, octaves):
    """One token without a value of its own outweighs all others together or nearly, which decide the result: fp16's subnormals count."""
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
    call.check(y)
    assert (y[:, :hq * d] != 0).all()


def test_what_is_not_seen_has_no_part():
    """Scales that are no numbers and full-size integers in places behind a row's position, in blocks of no sequence and behind the last token."""
    import torch

    lens, rows = [130, 70], [66, 1]
    c = cache(13, lens, 2, 64, maxp=4)
    free = sorted(set(range(c.pages)) - set(c.table.ravel().tolist()))
    c.table[0, 3], c.table[1, 2] = free  # whole blocks behind the sequences' ends
    for p in free:
        c.ks[p], c.vs[p], c.k[p], c.v[p] = np.nan, np.nan, 127, 127
    call = Call(c, rows, lens, 4)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)
    # the last block of sequence 0 (tokens 128, 129) has no numbers: rows before it are as they were, the rows that see it have none
    for which in ("ks", "vs"):
        t = getattr(call.dc, which)
        p, old = int(c.table[0, 2]), t.clone()
        t[p, 1] = float("nan")
        z = call.run()
        torch.cuda.synchronize()
        n = 4 * 64
        z4, y4 = z[:, :n].view(-1, 4, 64), y[:, :n].view(-1, 4, 64)
        seen = 64  # rows 64, 65 of the call have positions 128, 129
        assert torch.equal(z4[:seen], y4[:seen]) and torch.equal(z4[66:], y4[66:]) and torch.equal(z4[64:66, :2], y4[64:66, :2])
        assert torch.isnan(z4[64:66, 2:]).all()
        t.copy_(old)


@pytest.mark.parametrize("rows,lens,hq,d", [([3, 1], [257, 60], 4, 64), ([3], [257], 12, 128), ([2], [1025], 8, 256), ([300], [300], 4, 64), ([90], [257], 4, 128), ([130], [200], 4, 256)])
@pytest.mark.parametrize("far", [2.0 ** 60, 1e38])
def test_later_blocks_of_huge_scale(rows, lens, hq, d, far):
    """The rows of a call that see less keep their bits, however large the numbers are that only rows beside them see, and where a block is not there."""
    import torch

    c = cache(23, lens, 2, d)
    last = (lens[0] - 1) // 64
    call = Call(c, rows, lens, hq)
    y = call.run()
    first = lens[0] - rows[0]
    before = last * 64 - first  # rows of sequence 0 that do not see its last block
    assert 0 < before < rows[0]
    call.dc.vs[int(c.table[0, last])] = far
    z = call.run()
    torch.cuda.synchronize()
    assert torch.equal(z[:before], y[:before]) and torch.equal(z[rows[0]:], y[rows[0]:]) and not torch.equal(z[before:rows[0]], y[before:rows[0]])
    # the page that an entry outside the pages stands in for has no part either
    call.dc.table[0, last] = -1
    call.dc.vs[0] = far if 0 not in c.table[:, :last].ravel().tolist() else call.dc.vs[0]
    z = call.run()
    torch.cuda.synchronize()
    assert torch.equal(z[:before], y[:before])


def test_queries_that_are_no_numbers():
    import torch

    for value in (float("inf"), float("-inf"), float("nan")):
        call = Call(cache(15, [100, 30, 0], 2, 64), [3, 1, 1], [100, 30, 0], 4)
        y = call.run()
        call.q[1, 64 + 5] = value
        call.q[4, 3] = value  # a row that sees nothing
        z = call.run()
        torch.cuda.synchronize()
        z4, y4 = z.view(5, 4, 64), y.view(5, 4, 64)
        assert torch.isnan(z4[1, 1]).all() and (z4[4] == 0).all()
        z4[1, 1] = y4[1, 1]
        assert torch.equal(z4, y4)


def test_blocks_that_are_not_there():
    """Table entries outside the pages and tokens past the table: as if those tokens were none."""
    import torch

    lens, rows = [300, 128, 64], [2, 70, 1]  # the fifth block of the first lies past the table
    c = cache(17, [256, 128, 64], 2, 96, maxp=4)
    c.table[0, 1], c.table[1, 0], c.table[2, 0] = -3, c.pages + 5, -1
    call = Call(c, rows, lens, 2)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)
    assert (y[-1] == 0).all()


def test_start_outside_the_rows():
    """start values that are negative, fall, or pass the rows: no row outside the call is touched."""
    import torch

    call = Call(cache(19, [100, 100, 100], 1, 64), [2, 2, 2], [100, 100, 100], 2)
    call.ts = ints([-4, 3, 1, 1 << 30])
    y = torch.full((8, call.ldy), 7.0, dtype=torch.bfloat16, device="cuda")
    call.run(y=y)
    torch.cuda.synchronize()
    assert (y[6:] == 7).all() and torch.isfinite(y.float()).all()


def test_long_cache_beyond_32_bits():
    """Pages past 2^32 bytes of the cache: the output is that of the same blocks at the cache's start."""
    import torch

    hkv, d, n = 8, 128, 400
    page = hkv * 64 * d
    pages = (1 << 32) // page + 8
    kq, vq = (torch.full((pages * page,), 128, dtype=torch.uint8, device="cuda") for _ in range(2))
    ks, vs = (torch.full((pages, hkv), float("nan"), device="cuda") for _ in range(2))
    q, st = torch.randn(1, 16 * d, device="cuda").to(torch.bfloat16), ints([0, 1])
    far, near, ln = ints([[pages - 1 - i for i in range(7)]]), ints([list(range(7))]), ints([n])
    blocks = torch.randint(1, 256, (7, page), device="cuda", dtype=torch.uint8)
    out = []
    for table in (near, far):
        for b, p in enumerate(table[0].tolist()):
            kq[p * page:(p + 1) * page], vq[p * page:(p + 1) * page] = blocks[b], blocks[6 - b]
            ks[p], vs[p] = 0.01, 0.02
        y = torch.zeros(1, 16 * d, dtype=torch.bfloat16, device="cuda")
        ws = torch.zeros(D.lib().dr_attn_kv8_ws(1, 1, 1, n, 16, hkv, d), dtype=torch.uint8, device="cuda")
        D.lib().dr_attn_kv8(D.ptr(q), 16 * d, D.ptr(st), D.ptr(ln), D.ptr(table), 7, D.ptr(kq), D.ptr(ks), D.ptr(vq), D.ptr(vs), pages, 0.1, None, 0, 0,
                            D.ptr(ws), D.ptr(y), 16 * d, 1, 1, 1, n, 16, hkv, d, D.stream_ptr())
        torch.cuda.synchronize()
        out.append(y)
    assert torch.equal(*out) and torch.isfinite(out[0].float()).all() and (out[0] != 0).any()


def test_captured_call_follows_its_inputs():
    """A captured call replayed for growing sequences and other queries: each replay has the eager call's bits."""
    import torch

    c = cache(21, [1100, 1100, 1100], 2, 64)
    call = Call(c, [1, 1, 1], [1, 500, 1000], 8, max_len=1100)
    y = torch.zeros(call.total, call.ldy, dtype=torch.bfloat16, device="cuda")
    st, g, lib = torch.cuda.Stream(), ctypes.c_void_p(), D.lib()
    call.run(y=y, stream=st.cuda_stream)
    st.synchronize()
    lib.dr_graph_begin(st.cuda_stream)
    call.run(y=y, stream=st.cuda_stream)
    assert lib.dr_graph_end(st.cuda_stream, ctypes.byref(g)) == 0
    try:
        for k in range(5):
            call.q.copy_(torch.randn(call.q.shape, device="cuda"))
            call.tl.copy_(torch.tensor([1 + k * 40, 500 + k * 100, 1000 + k], dtype=torch.int32))
            torch.cuda.synchronize()
            lib.dr_graph_launch(g, st.cuda_stream)
            st.synchronize()
            got = y.clone()
            call.lens = call.tl.tolist()
            want = call.run()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            call.check(want)
    finally:
        lib.dr_graph_destroy(g)
