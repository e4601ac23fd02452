"""dr_gemm_q8_lora and dr_gemm_q8_lora_bf16s against the formula in 64 bits.

Tolerances, u = 2^-24.  W x: the products are exact; at most 128 of them and the scale's product, then a chain of at most
k / 128 + 8 sums, each of at most the terms' magnitudes: (136 + k / 128) u.  A x: a chain of k products: (k + 8) u, its
scale one more; B t: (rank + 2) u of its terms and B's share of t's error (t may travel in pieces whose sum is the
fp32 value: up to three sums per term, 3 rank u).  The residual: two more sums."""
import ctypes

import numpy as np
import pytest

import dramamoe as D
import synth
from helpers import dev

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Case:
    def __init__(self, fmt, rows, n, k, adapters, rmax, ids, pad_x=0, pad_y=0, with_res=True, ranks=None, seed=0):
        import torch

        rng = np.random.default_rng(seed + rows * 7919 + n)
        self.fmt, self.rows, self.n, self.k, self.adapters, self.rmax = fmt, rows, n, k, adapters, rmax
        self.ldx, self.ldy = k + pad_x, n + pad_y
        q, s, kind, _ = synth.q8_dense(rng, n, k, fmt)
        sc = synth.dec(s, kind).astype(np.float64)
        self.w = q.astype(np.float64) * (sc[:, None] if sc.ndim == 1 else sc.repeat(128, 1))
        self.tw, self.ts = dev(q), dev(s)
        torch.manual_seed(seed + rows)
        nan = float("nan")
        self.tx = torch.full((rows, self.ldx), nan, device="cuda").to(torch.bfloat16)
        self.tx[:, :k] = torch.randn(rows, k, device="cuda").to(torch.bfloat16)
        self.tres = torch.full((rows + 1, self.ldy), 5.0, device="cuda")
        self.tres[:rows, :n] = torch.randn(rows, n, device="cuda")
        self.with_res = with_res
        a = max(adapters, 1)
        self.rank = np.array(ranks if ranks is not None else rng.integers(1, rmax + 1, a), np.int32)
        self.scale = (0.5 + rng.random(a)).astype(np.float32)
        self.tla = (torch.randn(a, rmax, k, device="cuda") / k ** 0.5).to(torch.bfloat16)
        self.tlb = (0.1 * torch.randn(a, n, rmax, device="cuda")).to(torch.bfloat16)
        for j in range(a):  # what lies past an adapter's rank must not be read into a result
            r = min(max(int(self.rank[j]), 0), rmax)
            self.tla[j, r:] = nan
            self.tlb[j, :, r:] = nan
        self.ids = np.asarray(ids, np.int32) if ids is not None else None
        self.tids = dev(self.ids) if ids is not None else None
        self.trank, self.tscale = dev(self.rank), dev(self.scale)
        nb = D.lib().dr_gemm_q8_lora_ws(rows, n, k, rmax)
        self.ws = torch.full((nb + 256,), 0xFF, dtype=torch.uint8, device="cuda")  # NaN where nothing is written

    def call(self, y=None, stream=None):
        import torch

        y = torch.full((self.rows + 1, self.ldy), 5.0, device="cuda") if y is None else y
        P = D.ptr
        f = D.lib().dr_gemm_q8_lora if self.fmt == "ref" else D.lib().dr_gemm_q8_lora_bf16s
        f(P(self.tw), P(self.ts), P(self.tx), self.ldx, P(self.tids), P(self.tla), P(self.tlb), P(self.trank), P(self.tscale), self.adapters,
          self.rmax, P(self.ws), P(self.tres) if self.with_res else None, P(y), self.ldy, self.rows, self.n, self.k, stream or D.stream_ptr())
        return y

    def reference(self):
        x = self.tx[:, :self.k].double().cpu().numpy()
        y = x @ self.w.T
        mag = np.abs(x) @ np.abs(self.w).T
        dy = (136 + self.k / 128) * U * mag
        la, lb = self.tla.double().cpu().numpy(), self.tlb.double().cpu().numpy()
        for r in range(self.rows):
            j = self.ids[r] if self.ids is not None else -1
            if not 0 <= j < self.adapters or self.rank[j] < 1:
                continue
            rk = min(int(self.rank[j]), self.rmax)
            A, B, s = la[j, :rk], lb[j, :, :rk], float(self.scale[j])
            t, dt = s * (A @ x[r]), s * (self.k + 9) * U * (np.abs(A) @ np.abs(x[r]))
            y[r] += B @ t
            mag[r] += np.abs(B) @ np.abs(t)
            dy[r] += np.abs(B) @ dt + (3 * rk + 2) * U * (np.abs(B) @ (np.abs(t) + dt))
        if self.with_res:
            res = self.tres[:self.rows, :self.n].double().cpu().numpy()
            y, mag = y + res, mag + np.abs(res)
        return y, dy + 3 * U * mag

    def check(self, y):
        want, bound = self.reference()
        got = y[:self.rows, :self.n].double().cpu().numpy()
        bad = ~(np.abs(got - want) <= bound)
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3], got[bad][:3], want[bad][:3], bound[bad][:3])
        assert np.abs(got - want).max() <= 1e-3 * np.abs(want).max()  # the bound stays tight enough to mean something
        assert (y[:self.rows, self.n:] == 5).all() and (y[self.rows:] == 5).all()
        assert (self.ws[-256:] == 0xFF).all()


def ids_each(rows, adapters, seed=1):
    return np.random.default_rng(seed).integers(-1, adapters, rows)


def ids_runs(rows, adapters, run, seed=2):
    return np.random.default_rng(seed).integers(-1, adapters, rows // run + 1).repeat(run)[:rows]


SIZES = [
    # rows, n, k, adapters, rmax, ids, pad_x, pad_y
    (1, 2048, 2048, 4, 16, [2], 0, 0), (1, 1, 128, 1, 8, [0], 0, 0), (2, 17, 256, 3, 24, [1, -1], 8, 3), (7, 100, 384, 7, 8, [3, 3, 1, 0, 6, 3, -1], 0, 4),
    (16, 64, 1024, 16, 64, range(16), 0, 0), (17, 1031, 640, 9, 40, "each", 16, 1), (48, 512, 2048, 40, 32, "each", 0, 0),
    (64, 33, 1152, 64, 128, "each", 0, 0), (65, 130, 256, 5, 16, "each", 0, 2), (100, 1000, 512, 3, 16, "runs", 8, 0),
    (129, 257, 384, 12, 48, "each", 0, 7), (300, 2048, 512, 6, 16, "runs", 0, 0), (513, 96, 128, 30, 8, "each", 0, 0),
    (700, 1031, 1024, 5, 16, "runs", 0, 0), (3, 8, 16384, 2, 16, [0, 1, 1], 0, 0), (1025, 384, 256, 20, 112, "runs", 0, 0),
    (4, 40, 384, 3, 16, [2, 2, -1, 0], 0, 0), (3, 300, 1152, 4, 16, [1, 0, 3], 8, 0), (2, 100, 512, 5, 32, [4, 1], 0, 1), (1, 333, 2048, 2, 64, [1], 0, 0),
    (2, 64, 128, 3, 8, [0, 0], 0, 0), (2000, 8200, 128, 9, 24, "each", 0, 0), (1025, 4100, 256, 7, 72, "runs", 0, 3),
]


@pytest.mark.parametrize("fmt", ["ref", "cfg"])
@pytest.mark.parametrize("rows,n,k,adapters,rmax,ids,pad_x,pad_y", SIZES)
def test_gemm_q8_lora(rows, n, k, adapters, rmax, ids, pad_x, pad_y, fmt):
    import torch

    if ids == "each":
        ids = ids_each(rows, adapters)
    elif ids == "runs":
        ids = ids_runs(rows, adapters, max(1, rows // 7))
    c = Case(fmt, rows, n, k, adapters, rmax, list(ids), pad_x, pad_y)
    y = c.call()
    torch.cuda.synchronize()
    c.check(y)
    # again on the same workspace: the same bits; then in place of the residual
    again = c.call()
    assert torch.equal(again, y)
    inplace = c.call(y=c.tres)
    torch.cuda.synchronize()
    assert torch.equal(inplace[:rows, :n], y[:rows, :n])


@pytest.mark.parametrize("rows", [1, 20, 200])
def test_rows_without_adapter(rows):
    """No adapters at all, a null id list, ids out of range and adapters without rank: the projection alone, the same bits
    each way; ranks above rmax are rmax."""
    import torch

    n, k = 300, 512
    plain = Case("ref", rows, n, k, 0, 8, None, with_res=False)
    y = plain.call()
    torch.cuda.synchronize()
    plain.check(y)
    bad = [-1, 4, 1000000, -2147483648, 2147483647, 1, 3]
    c = Case("ref", rows, n, k, 4, 8, [bad[r % 7] for r in range(rows)], with_res=False, ranks=[8, 0, 8, -3])
    y2 = c.call()
    torch.cuda.synchronize()
    c.check(y2)
    assert torch.equal(y, y2)
    c = Case("cfg", rows, n, k, 4, 8, [r % 4 for r in range(rows)], ranks=[8, 9, 2147483647, 1])
    y3 = c.call()
    torch.cuda.synchronize()
    c.check(y3)


def test_one_row_is_the_decode_projection():
    """Without an adapter, one row gives dr_gemv_q8's projection up to the order of the fp32 sums."""
    import torch

    n, k = 2048, 2048
    c = Case("ref", 1, n, k, 0, 8, None)
    y = c.call()
    x = c.tx.float().contiguous()
    want = torch.empty(n, device="cuda")
    D.lib().dr_gemv_q8(D.ptr(c.tw), D.ptr(c.ts), D.ptr(x), D.ptr(c.tres), D.ptr(want), n, k, None, 0.0, None, 0, D.stream_ptr())
    torch.cuda.synchronize()
    mag = (np.abs(x.double().cpu().numpy()) @ np.abs(c.w).T).ravel()
    # dr_gemv_q8 adds 128 to every value and takes 128 sum(x) off again: its terms are up to 255 / |q| larger
    big = 255 * np.abs(x.double().cpu().numpy()).sum() * (np.abs(c.w).max(1) / 1.0)
    diff = np.abs((y[0, :n] - want).double().cpu().numpy())
    assert (diff <= (136 + k / 128) * U * mag + 64 * U * big / 127 + U * 4).all()


@pytest.mark.parametrize("rows", [24, 150])
def test_rows_keep_to_themselves(rows):
    """NaN and infinities in one row, and in the adapter that only one other row uses, leave the others' bits."""
    import torch

    c = Case("cfg", rows, 200, 512, 6, 16, [r % 5 for r in range(rows - 1)] + [5])
    y = c.call()
    torch.cuda.synchronize()
    c.check(y)
    c.tx[3, 7], c.tx[9, 0] = float("nan"), float("inf")
    c.tla[5] = float("nan")
    z = c.call()
    torch.cuda.synchronize()
    keep = [r for r in range(rows) if r not in (3, 9, rows - 1)]
    assert torch.equal(y[keep], z[keep])
    assert torch.isnan(z[3, :200]).all() and torch.isnan(z[rows - 1, :200]).all()
    # the same of B: a product with another row's zero would be NaN
    c.tlb[5, :, 0], c.tlb[5, :, 1] = float("inf"), float("nan")
    z = c.call()
    torch.cuda.synchronize()
    assert torch.equal(y[keep], z[keep])


@pytest.mark.parametrize("rows", [1, 24, 150])
def test_overflow_stays_infinite(rows):
    """A_a x past the range of fp32 in one rank: the outputs are infinities with that rank's signs, not NaN."""
    import torch

    c = Case("cfg", rows, 200, 512, 2, 16, [0] * rows)
    c.tx[0, :512] = 1.0
    c.tla[0, 0], c.tla[0, 1:] = 3e38, 0.0
    c.tlb[0] = torch.where(torch.arange(200, device="cuda") % 3 == 0, -1.0, 1.0)[:, None].to(torch.bfloat16)
    c.tscale[0] = 1.0
    c.trank[0] = 16
    y = c.call()[0, :200]
    torch.cuda.synchronize()
    assert torch.isinf(y).all() and torch.equal(y < 0, torch.arange(200, device="cuda") % 3 == 0)


@pytest.mark.parametrize("rows,n", [(40, 512), (333, 640)])
def test_graph_replays(rows, n):
    """Captured once, replayed with new rows and new adapter ids, eager calls on the same workspace in between."""
    import torch

    lib = D.lib()
    c = Case("ref", rows, n, 768, 8, 32, ids_each(rows, 8))
    st = torch.cuda.Stream()
    y = c.call()
    torch.cuda.synchronize()
    g = ctypes.c_void_p()
    lib.dr_graph_begin(st.cuda_stream)
    c.call(y=y, stream=st.cuda_stream)
    assert lib.dr_graph_end(st.cuda_stream, ctypes.byref(g)) == 0
    try:
        for q in range(3):
            c.tx.copy_(torch.randn(rows, c.k, device="cuda"))
            c.ids = ids_each(rows, 8, seed=10 + q).astype(np.int32)
            c.tids.copy_(torch.from_numpy(c.ids))
            torch.cuda.synchronize()
            want = c.call()
            torch.cuda.synchronize()
            c.check(want)
            lib.dr_graph_launch(g, st.cuda_stream)
            st.synchronize()
            assert torch.equal(y, want)
    finally:
        lib.dr_graph_destroy(g)
