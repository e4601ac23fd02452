"""An attention block's operators one behind the other, as a caller has them: norm, the q, k, v (and gate) projection with each row's adapter,
positions, cache, attention, output projection, norm and residual.  Every step is checked against 64 bits on what the step before left
(tolerances: test_gpu_block_norm.py, test_gpu_gemm_q8_lora.py, test_gpu_rope.py, kv8_helpers.py); a captured run replays to
the eager bits, and two runs on two streams beside each other have the bits of each alone."""
import ctypes

import numpy as np
import pytest

import dramamoe as D
import kvcache as K
import test_gpu_block_norm as N
import test_gpu_gemm_q8_lora as G
import test_gpu_rope as R
from kv8_helpers import Cache, attention

pytestmark = pytest.mark.gpu
H, HQ, HKV, DH, ROT = 512, 8, 2, 64, 32
QW = 2 * HQ * DH  # each query beside its gate
KW = HKV * DH


class Block:
    """One layer of 3 sequences; a step's buffers belong to the rows it has."""

    def __init__(self, seed, pages=40, max_len=700):
        import torch

        torch.manual_seed(seed)
        self.seed = seed
        self.cache = K.KvCache(1, pages, 3, max_len, HQ, HKV, DH)
        self.nw = [1 + 0.1 * torch.randn(H, device="cuda") for _ in range(2)]
        self.qnw, self.knw = (1 + 0.1 * torch.randn(DH, device="cuda") for _ in range(2))
        f, self.ms = K.rope_freq(ROT, 10000.0, "yarn", 4.0, trained=256)
        self.freq = f.cuda()
        self.host = Cache(np.random.default_rng(seed), [0, 0, 0], HKV, DH, spare=pages, maxp=self.cache.maxp, content="none")
        self.history = 0

    def buffers(self, rows):
        import torch

        b = type("Buffers", (), {})()
        t = sum(rows)
        b.qkv = G.Case("ref", t, QW + 2 * KW, H, 3, 16, G.ids_each(t, 3), with_res=False, seed=self.seed)
        b.out = G.Case("ref", t, H, HQ * DH, 3, 16, G.ids_each(t, 3), with_res=False, seed=self.seed + 1)
        b.x, b.hn, b.x1 = torch.randn(t, H, device="cuda"), b.qkv.tx, torch.zeros(t, H, device="cuda")
        b.hn2 = torch.zeros(t, H, dtype=torch.bfloat16, device="cuda")
        b.p, b.o = torch.full((t + 1, QW + 2 * KW), 5.0, device="cuda"), torch.full((t + 1, H), 5.0, device="cuda")
        return b

    def run(self, b, batch, max_len=None):
        """On torch's current stream."""
        lib, P, t, st = D.lib(), D.ptr, batch.total, D.stream_ptr()
        lib.dr_block_norm(None, 0, P(b.x), H, None, None, 0, 0, None, 0.0, 1.0, P(self.nw[0]), 1e-6, None, 0, P(b.hn), H, t, H, st)
        b.qkv.call(y=b.p, stream=st)
        b.q = K.rope(b.p[:t], HQ, DH, batch.pos, self.freq, self.ms, nw=self.qnw, head_stride=2 * DH)
        b.k = K.rope(b.p[:t, QW:], HKV, DH, batch.pos, self.freq, self.ms, nw=self.knw, f32=True)
        self.cache.append(0, b.k, b.p[:t, QW + KW:], batch)
        # the gate beside each query
        lib.dr_attn_kv8(P(b.q), HQ * DH, P(batch.start), P(batch.len), *self.cache._cache(0), DH ** -0.5, b.p.data_ptr() + 4 * DH, QW + 2 * KW, 2 * DH,
                        P(self.ws(st, batch, max_len)), P(b.out.tx), HQ * DH, t, 3, batch.max_rows, max_len or batch.max_len, HQ, HKV, DH, st)
        b.out.call(y=b.o, stream=st)
        lib.dr_block_norm(P(b.o), H, P(b.x), H, None, None, 0, 0, None, 1.0, 1.0, P(self.nw[1]), 1e-6, P(b.x1), H, P(b.hn2), H, t, H, st)

    def ws(self, st, batch, max_len):
        import torch

        self.keep = getattr(self, "keep", {})
        n = D.lib().dr_attn_kv8_ws(batch.total, 3, batch.max_rows, max_len or batch.max_len, HQ, HKV, DH)
        if st not in self.keep or self.keep[st].numel() < n:
            self.keep[st] = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
        return self.keep[st]

    def outputs(self, b):
        return [t.clone() for t in (b.hn, b.p, b.q, b.k, b.out.tx, b.o, b.x1, b.hn2, self.cache.kq, self.cache.vq, self.cache.ks, self.cache.vs)]

    def check(self, b, batch):
        f64 = lambda t: t.double().cpu().numpy()
        t, start, lens = batch.total, batch.start.tolist(), batch.len.tolist()
        zero = np.zeros((t, H))
        *_, hn, dh = N.reference(zero, zero, f64(b.x), None, None, None, 0.0, 1.0, f64(self.nw[0]), 1e-6)
        N.check(b.hn, hn, dh, "first norm")
        b.qkv.check(b.p)
        p, pos, freq = f64(b.p[:t]), batch.pos.cpu().numpy(), self.freq.cpu().numpy()
        qg = p[:, :QW].reshape(t, HQ, 2, DH)
        want, bound = R.reference(qg[:, :, 0], f64(self.qnw), 1e-6, pos, freq, self.ms, False, ROT)
        assert (np.abs(f64(b.q).reshape(want.shape) - want) <= bound + 2.0 ** -8 * (np.abs(want) + bound)).all()
        want, bound = R.reference(p[:, QW:QW + KW].reshape(t, HKV, DH), f64(self.knw), 1e-6, pos, freq, self.ms, False, ROT)
        assert (np.abs(f64(b.k).reshape(want.shape) - want) <= bound).all()
        # the cache: the host's copy takes the same tokens
        self.host.table = self.cache.table.cpu().numpy()
        self.host.append(f64(b.k).reshape(t, HKV, DH), p[:, QW + KW:].reshape(t, HKV, DH), start, lens)
        gk, gv = self.host.unpack(self.cache.kq[0].cpu().numpy(), self.cache.vq[0].cpu().numpy())
        assert np.array_equal(self.cache.ks[0].cpu().numpy(), self.host.ks) and np.array_equal(self.cache.vs[0].cpu().numpy(), self.host.vs)
        for i in range(3):
            for n in range((lens[i] + 63) // 64):
                g, m = self.host.table[i, n], min(64, lens[i] - 64 * n)
                assert np.array_equal(gk[g, :, :m], self.host.k[g, :, :m]) and np.array_equal(gv[g, :, :m], self.host.v[g, :, :m])
        y, bound = attention(self.host, f64(b.q).reshape(t, HQ, DH), start, lens, DH ** -0.5, qg[:, :, 1])
        assert (np.abs(f64(b.out.tx).reshape(y.shape) - y) <= bound).all()
        b.out.check(b.o)
        o = f64(b.o[:t])
        xo, dx, hn, dh = N.reference(o, 0 * o, f64(b.x), None, None, None, 1.0, 1.0, f64(self.nw[1]), 1e-6)
        N.check(b.x1, xo, dx, "residual"), N.check(b.hn2, hn, dh, "second norm")


def test_prompts_then_single_tokens():
    """Ragged prompts, a second chunk of one, then decode steps with one sequence resting, drafted tokens and their refusal."""
    import torch

    blk = Block(1)
    for rows in ([70, 3, 130], [0, 66, 5], [1, 1, 1], [1, 0, 1], [4, 1, 3]):
        batch = blk.cache.step(rows)
        b = blk.buffers(rows)
        blk.run(b, batch)
        torch.cuda.synchronize()
        blk.check(b, batch)
    blk.cache.truncate(0, 73)
    blk.cache.truncate(2, 128)
    for rows in ([2, 1, 1], [1, 1, 1]):
        batch = blk.cache.step(rows)
        b = blk.buffers(rows)
        blk.run(b, batch)
        torch.cuda.synchronize()
        blk.check(b, batch)


def test_captured_decode_steps():
    """A decode step captured once and replayed for growing sequences, its batch updated in place; eager steps of a second cache beside it."""
    import torch

    a, e = Block(2), Block(2)
    prompt = [60, 5, 120]
    bufs = {}
    for blk in (a, e):
        torch.manual_seed(5)
        b = blk.buffers(prompt)
        blk.run(b, blk.cache.step(prompt))
        torch.manual_seed(6)
        bufs[blk] = blk.buffers([1, 1, 1])
    ba, be = bufs[a], bufs[e]
    torch.cuda.synchronize()
    st, g, lib = torch.cuda.Stream(), ctypes.c_void_p(), D.lib()
    batch = a.cache.step([1, 1, 1])
    with torch.cuda.stream(st):
        a.run(ba, batch, max_len=200)  # workspaces of the stream; the same tokens again change nothing
        st.synchronize()
        ba.keep = (ba.q, ba.k)
        lib.dr_graph_begin(st.cuda_stream)
        # buffers of the captured run are those that were made before it
        P = D.ptr
        t = 3
        lib.dr_block_norm(None, 0, P(ba.x), H, None, None, 0, 0, None, 0.0, 1.0, P(a.nw[0]), 1e-6, None, 0, P(ba.hn), H, t, H, st.cuda_stream)
        ba.qkv.call(y=ba.p, stream=st.cuda_stream)
        lib.dr_rope(ba.p.data_ptr(), QW + 2 * KW, 2 * DH, P(a.qnw), 0, 1e-6, P(batch.pos), P(a.freq), a.ms, 0, None, 0, P(ba.q), HQ * DH, t, HQ, DH, ROT, st.cuda_stream)
        lib.dr_rope(ba.p.data_ptr() + 4 * QW, QW + 2 * KW, DH, P(a.knw), 0, 1e-6, P(batch.pos), P(a.freq), a.ms, 0, P(ba.k), KW, None, 0, t, HKV, DH, ROT, st.cuda_stream)
        a.cache.append(0, ba.k, ba.p[:t, QW + KW:], batch)
        lib.dr_attn_kv8(P(ba.q), HQ * DH, P(batch.start), P(batch.len), *a.cache._cache(0), DH ** -0.5, ba.p.data_ptr() + 4 * DH, QW + 2 * KW, 2 * DH,
                        P(a.keep[st.cuda_stream]), P(ba.out.tx), HQ * DH, t, 3, 1, 200, HQ, HKV, DH, st.cuda_stream)
        ba.out.call(y=ba.o, stream=st.cuda_stream)
        lib.dr_block_norm(P(ba.o), H, P(ba.x), H, None, None, 0, 0, None, 1.0, 1.0, P(a.nw[1]), 1e-6, P(ba.x1), H, P(ba.hn2), H, t, H, st.cuda_stream)
        assert lib.dr_graph_end(st.cuda_stream, ctypes.byref(g)) == 0
    try:
        for n in range(6):
            x = torch.randn(3, H, device="cuda")
            if n:
                nxt = a.cache.step([1, 1, 1])
                batch.pos.copy_(nxt.pos), batch.len.copy_(nxt.len)
            ba.x.copy_(x), be.x.copy_(x)
            torch.cuda.synchronize()
            lib.dr_graph_launch(g, st.cuda_stream)
            st.synchronize()
            got = a.outputs(ba)
            eager = e.cache.step([1, 1, 1])
            e.run(be, eager, max_len=200)
            torch.cuda.synchronize()
            for p, q in zip(got, e.outputs(be)):
                assert torch.equal(p, q), n
    finally:
        lib.dr_graph_destroy(g)


def test_two_streams_every_run_counts():
    """Two blocks with caches and workspaces of their own on two streams beside each other: every run has the bits it has alone."""
    import torch

    steps = [[33, 2, 70], [1, 1, 1], [2, 5, 1], [1, 1, 1]]

    def inputs(seed):
        out = []
        for k, rows in enumerate(steps):
            torch.manual_seed(seed * 10 + k)
            out.append(torch.randn(sum(rows), H, device="cuda"))
        return out

    def go(blocks, streams, xs):
        got = [[] for _ in blocks]
        bufs = [[blk.buffers(rows) for rows in steps] for blk in blocks]
        batches = [[blk.cache.step(rows) for rows in steps] for blk in blocks]
        for i in range(len(blocks)):
            for b, x in zip(bufs[i], xs[i]):
                b.x.copy_(x)
        torch.cuda.synchronize()
        for k in range(len(steps)):
            for i, (blk, s) in enumerate(zip(blocks, streams)):
                with torch.cuda.stream(s):
                    blk.run(bufs[i][k], batches[i][k])
                    got[i].append(blk.outputs(bufs[i][k]))
        torch.cuda.synchronize()
        return got

    xs = [inputs(3), inputs(4)]
    main = torch.cuda.current_stream()
    want = [go([Block(7 + i)], [main], [xs[i]])[0] for i in range(2)]
    for _ in range(3):
        got = go([Block(7), Block(8)], [torch.cuda.Stream(), torch.cuda.Stream()], xs)
        for g, w in zip(got, want):
            for k in range(len(steps)):
                assert all(torch.equal(p, q) for p, q in zip(g[k], w[k])), k


def test_attend_and_read_of_the_cache_object():
    """KvCache.attend (with a gate, in place, on a stream of its own) and KvCache.read against the entry points' definitions."""
    import torch

    c = K.KvCache(2, 20, 2, 400, 4, 2, 48)
    host = Cache(np.random.default_rng(0), [0, 0], 2, 48, spare=20, maxp=c.maxp, content="none")
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for rows in ([100, 7], [1, 1], [30, 0]):
            b = c.step(rows)
            k, v = (torch.randn(b.total, 2 * 48, device="cuda").to(torch.bfloat16) for _ in range(2))
            c.append(1, k, v, b)
            q, gate = torch.randn(b.total, 4 * 48, device="cuda").to(torch.bfloat16), torch.randn(b.total, 4 * 48, device="cuda")
            q0 = q.clone()
            out = c.attend(1, q, b, gate=gate, out=q)
            rk, rv = c.read(1, b)
            s.synchronize()
            assert out.data_ptr() == q.data_ptr()
            f = lambda t, h: t.double().cpu().numpy().reshape(-1, h, 48)
            start, lens = b.start.tolist(), b.len.tolist()
            host.table = c.table.cpu().numpy()
            host.append(f(k, 2), f(v, 2), start, lens)
            y, bound = attention(host, f(q0, 4), start, lens, 48 ** -0.5, f(gate, 4))
            assert (np.abs(f(out, 4) - y) <= bound).all()
            for i in range(2):
                for h in range(2):
                    tk, tv, _ = host.tokens(i, lens[i], h)
                    n = rows[i]
                    assert np.array_equal(f(rk, 2)[start[i]:start[i + 1], h], tk[lens[i] - n:lens[i]].astype(np.float32))
                    assert np.array_equal(f(rv, 2)[start[i]:start[i + 1], h], tv[lens[i] - n:lens[i]].astype(np.float32))
    assert (c.kq[0] == 0).all() and (c.ks[0] == 0).all()  # the other layer
