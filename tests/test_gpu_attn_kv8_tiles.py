"""dr_attn_kv8 with so many pairs (rows of a sequence times queries of a cached head) that its tiles take them: what rows do not see, scales of every
size, numbers that are none, blocks that are not there.  Tolerances: kv8_helpers.attention."""
import pytest

from kv8_helpers import ints
from test_gpu_attn_kv8 import Call, cache

pytestmark = pytest.mark.gpu

# tiles of four waves at heads up to 64, 128, 192 and 256 elements, of eight waves, and of eight with a sequence's halves folded
SHAPES = [([1100, 3], [1200, 3], 4, 2, 64), ([1100], [1100], 4, 2, 128), ([1100], [1150], 4, 2, 192), ([1100], [1100], 4, 2, 256), ([1500], [1600], 64, 2, 64), ([1500], [1500], 32, 2, 128)]
SMALL = [([1100, 3], [1200, 3], 2, 1, 48), ([1050], [1050], 2, 1, 128), ([1040], [1100], 2, 1, 176), ([1030], [1030], 2, 1, 256)]


def views(call, *ys):
    n = call.hq * call.c.d
    return [y[:, :n].view(-1, call.hq, call.c.d) for y in ys]


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
@pytest.mark.parametrize("far", [2.0 ** 60, 1e38])
def test_later_blocks_of_huge_scale(rows, lens, hq, hkv, d, far):
    import torch

    call = Call(cache(33, lens, hkv, d), rows, lens, hq)
    y = call.run()
    last = (lens[0] - 1) // 64
    for block in (last, last // 2):
        before = block * 64 - (lens[0] - rows[0])
        old = call.dc.vs.clone()
        call.dc.vs[int(call.c.table[0, block])] = far
        z = call.run()
        torch.cuda.synchronize()
        assert torch.equal(z[:before], y[:before]) and torch.equal(z[rows[0]:], y[rows[0]:]) and not torch.equal(z[before:rows[0]], y[before:rows[0]])
        call.dc.vs.copy_(old)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
@pytest.mark.parametrize("which", ["ks", "vs"])
def test_scales_that_are_no_numbers(rows, lens, hq, hkv, d, which):
    import torch

    call = Call(cache(35, lens, hkv, d), rows, lens, hq)
    y = call.run()
    t, block = getattr(call.dc, which), (lens[0] - 1) // 64 - 2
    for bad in (float("nan"), float("inf"), -1.0):
        p, old = int(call.c.table[0, block]), t.clone()
        t[p, 1] = bad
        z = call.run()
        torch.cuda.synchronize()
        seen, (y3, z3) = block * 64 - (lens[0] - rows[0]), views(call, y, z)
        assert torch.equal(z3[:seen], y3[:seen]) and torch.equal(z3[rows[0]:], y3[rows[0]:])
        assert torch.equal(z3[seen:rows[0], :hq // 2], y3[seen:rows[0], :hq // 2]) and torch.isnan(z3[seen:rows[0], hq // 2:]).all()
        t.copy_(old)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
def test_queries_that_are_no_numbers(rows, lens, hq, hkv, d):
    import torch

    call = Call(cache(37, lens, hkv, d), rows, lens, hq)
    y = call.run()
    where = [(0, 0), (rows[0] // 2, 1), (rows[0] - 1, hq - 1)]
    for (r, h), value in zip(where, (float("nan"), float("inf"), float("-inf"))):
        call.q[r, h * d + 7] = value
    z = call.run()
    torch.cuda.synchronize()
    y3, z3 = views(call, y, z)
    for r, h in where:
        assert torch.isnan(z3[r, h]).all()
        z3[r, h] = y3[r, h]
    assert torch.equal(z3, y3)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SMALL)
@pytest.mark.parametrize("scale", [None, 0.0, -0.3])
def test_scales_of_every_size(rows, lens, hq, hkv, d, scale):
    import torch

    c = cache(39, lens, hkv, d)
    for b, p in enumerate(c.table[0]):
        if p >= 0:
            c.vs[p] = 10.0 ** ((7 * b) % 30 - 15)
            c.ks[p] = (0, 1e-30, 0.05, 0.02)[b % 4]
    call = Call(c, rows, lens, hq, scale=scale, gate=True, behind=2, pad=1)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SMALL)
@pytest.mark.parametrize("qsize", [1e-30, 1e-3, 300.0, 1e30])
def test_peaked_and_flat_weights(rows, lens, hq, hkv, d, qsize):
    import torch

    call = Call(cache(41, lens, hkv, d), rows, lens, hq, qsize=qsize, scale=0.1 if qsize < 1e20 else 1e-29)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SMALL)
def test_blocks_that_are_not_there(rows, lens, hq, hkv, d):
    """Entries outside the pages, at the start, inside and at the end, rows before the first token, and tokens past the table."""
    import torch

    c = cache(43, lens, hkv, d)
    c.table[0, 0], c.table[0, 5], c.table[0, (lens[0] - 1) // 64 - 1] = -1, c.pages, -7
    call = Call(c, rows, lens, hq, behind=1)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)
    lens = [lens[0] - 400] + lens[1:]  # fewer tokens than rows
    call = Call(cache(45, [min(n, 512) for n in lens], hkv, d, maxp=8), rows, lens, hq)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)


@pytest.mark.parametrize("max_len", [0, 1, 1200, 100000])
@pytest.mark.parametrize("rows,lens,hq,hkv,d", SMALL)
def test_any_cut_is_right(rows, lens, hq, hkv, d, max_len):
    import torch

    call = Call(cache(47, lens, hkv, d), rows, lens, hq, max_len=max_len, gate=True)
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)


@pytest.mark.parametrize("rows,lens,hq,hkv,d", SHAPES)
def test_captured_and_in_place(rows, lens, hq, hkv, d):
    """Replays for other queries and shorter sequences have the eager bits; the output may take the queries' place."""
    import torch

    call = Call(cache(49, lens, hkv, d), rows, lens, hq)
    y = torch.zeros(call.total, call.ldy, dtype=torch.bfloat16, device="cuda")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            call.run(y=y, stream=st.cuda_stream)
    q0 = call.q.clone()
    for k in range(3):
        call.q.copy_(q0 * (k + 1))
        call.tl.copy_(ints([lens[0] - 70 * k] + lens[1:]))
        want = call.run()
        torch.cuda.synchronize()
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(want, y)
    q = call.q.clone()
    call.run(y=call.q)
    torch.cuda.synchronize()
    assert torch.equal(call.q, want) and not torch.equal(q, want)
