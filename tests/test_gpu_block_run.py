"""A decode block's operators one behind the other, as a caller has them: norm, a projection with each row's adapter, norm
and gate and residual, the MoE layer, norm.  Every step is checked against 64 bits on what the step before left (tolerances:
test_gpu_block_norm.py, test_gpu_gemm_q8_lora.py, test_gpu_moe_layer_rows.py), and a captured run replays to the eager bits."""
import ctypes

import numpy as np
import pytest

import dramamoe as D
import test_gpu_block_norm as N
import test_gpu_gemm_q8_lora as G
import test_gpu_moe_layer_rows as M

pytestmark = pytest.mark.gpu


class Block:
    def __init__(self, rows, h, e, i, topk):
        import torch

        torch.manual_seed(rows)
        self.rows, self.h, self.topk = rows, h, topk
        self.proj = G.Case("ref", rows, h, h, 4, 16, G.ids_each(rows, 4), with_res=False)
        self.moe = M.Layer(rows + 5, "q4", "ref", e, h, i, True)
        self.ws = M.workspace(rows, e, h, i, topk)
        f = lambda *s: torch.randn(*s, device="cuda")
        self.x, self.gate, self.pw, self.cs = f(rows, h), f(rows, h), 1 + 0.1 * f(h), f(h)
        self.nw = [1 + 0.1 * f(h) for _ in range(3)]
        self.hn = [torch.zeros(rows, h, dtype=torch.bfloat16, device="cuda") for _ in range(3)]
        self.hn[0] = self.proj.tx  # the norm writes the projection's input
        self.p, self.x1 = torch.full((rows + 1, h), 5.0, device="cuda"), torch.zeros(rows, h, device="cuda")
        self.o = None

    def run(self, stream=None):
        lib, P, h, rows = D.lib(), D.ptr, self.h, self.rows
        st = stream or D.stream_ptr()
        tail = lambda x, xo, k: (1e-6, xo, h, P(self.hn[k]), h, rows, h, st)
        lib.dr_block_norm(None, 0, P(self.x), h, None, None, 0, 0, None, 0.0, 1.0, P(self.nw[0]), *tail(None, None, 0))
        self.proj.call(y=self.p, stream=st)
        lib.dr_block_norm(P(self.p), h, P(self.x), h, P(self.pw), P(self.gate), 2, h, P(self.cs), 0.5, 1.5, P(self.nw[1]),
                          *tail(None, P(self.x1), 1))
        self.o = self.moe.call(self.hn[1], self.x1, rows, self.topk, self.ws, stream=st, out=self.o)
        lib.dr_block_norm(None, 0, P(self.o["y"]), h, None, None, 0, 0, None, 0.0, 1.0, P(self.nw[2]), *tail(None, None, 2))

    def outputs(self):
        return [t.clone() for t in (*self.hn, self.p, self.x1, self.o["y"], self.o["idx"], self.o["wts"], self.o["sgate"])]

    def check(self):
        f64 = lambda t: t.double().cpu().numpy()
        rows, zero = self.rows, np.zeros((self.rows, self.h))
        one = lambda x, nw: N.reference(zero, zero, f64(x), None, None, None, 0.0, 1.0, f64(nw), 1e-6)
        *_, hn, dh = one(self.x, self.nw[0])
        N.check(self.hn[0], hn, dh, "first norm")
        self.proj.check(self.p)
        b = f64(self.p[:rows])
        xo, dx, _, _ = N.reference(b, 0 * b, f64(self.x), f64(self.pw), f64(self.gate), f64(self.cs), 0.5, 1.5, f64(self.nw[1]), 1e-6)
        N.check(self.x1, xo, dx, "gated residual")
        *_, hn, dh = N.reference(b, 0 * b, f64(self.x), f64(self.pw), f64(self.gate), f64(self.cs), 0.5, 1.5, f64(self.nw[1]), 1e-6)
        N.check(self.hn[1], hn, dh, "second norm")
        M.check(self.moe, self.hn[1], self.x1, self.o, rows, self.topk)
        *_, hn, dh = one(self.o["y"][:rows], self.nw[2])
        N.check(self.hn[2], hn, dh, "third norm")


@pytest.mark.parametrize("rows", [1, 2, 9, 40])
def test_block_run(rows):
    import torch

    blk = Block(rows, 512, 16, 256, 4)
    blk.run()
    torch.cuda.synchronize()
    blk.check()
    st, g, lib = torch.cuda.Stream(), ctypes.c_void_p(), D.lib()
    lib.dr_graph_begin(st.cuda_stream)
    blk.run(stream=st.cuda_stream)
    assert lib.dr_graph_end(st.cuda_stream, ctypes.byref(g)) == 0
    try:
        for k in range(4):
            blk.x.copy_(torch.randn(rows, 512, device="cuda"))
            blk.proj.tids.copy_(torch.from_numpy(G.ids_each(rows, 4, seed=k)).int())
            torch.cuda.synchronize()
            lib.dr_graph_launch(g, st.cuda_stream)
            st.synchronize()
            got = blk.outputs()
            blk.run()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, blk.outputs()))
    finally:
        lib.dr_graph_destroy(g)


def test_two_streams_at_once():
    """Two runs of different sizes, each with its workspaces, on two streams beside each other: the bits of each alone."""
    import torch

    blocks = [Block(3, 512, 16, 256, 4), Block(40, 1024, 24, 384, 6)]
    want = []
    for b in blocks:
        b.run()
        torch.cuda.synchronize()
        want.append(b.outputs())
    streams = [torch.cuda.Stream() for _ in blocks]
    for _ in range(10):
        for b, s in zip(blocks, streams):
            b.run(stream=s.cuda_stream)
    torch.cuda.synchronize()
    for b, w in zip(blocks, want):
        assert all(torch.equal(p, q) for p, q in zip(b.outputs(), w))


def test_two_streams_every_run_counts():
    """As above with every run's outputs seen: each run starts on outputs filled with other values and on inputs of its own, and
    its outputs are kept on its stream before the next one."""
    import torch

    blocks, runs = [Block(3, 512, 16, 256, 4), Block(40, 1024, 24, 384, 6)], 10
    inputs = [[torch.randn_like(b.x) for _ in range(runs)] for b in blocks]

    def start(b, x):
        b.x.copy_(x)
        for t in (*b.hn, b.p, b.x1, b.o["y"]):
            t.fill_(5.0)
        for k in ("idx", "wts", "sgate"):
            b.o[k].fill_(-3)

    want = []
    for b, xs in zip(blocks, inputs):
        b.run()  # makes its outputs
        want.append([])
        for x in xs:
            start(b, x)
            b.run()
            torch.cuda.synchronize()
            want[-1].append(b.outputs())
    streams, got = [torch.cuda.Stream() for _ in blocks], [[] for _ in blocks]
    torch.cuda.synchronize()
    for k in range(runs):
        for b, s, xs, g in zip(blocks, streams, inputs, got):
            with torch.cuda.stream(s):
                start(b, xs[k])
                b.run(stream=s.cuda_stream)
                g.append(b.outputs())
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for k in range(runs):
            assert all(torch.equal(p, q) for p, q in zip(g[k], w[k])), k
        assert not any(torch.equal(g[k][-4], g[k + 1][-4]) for k in range(runs - 1))
