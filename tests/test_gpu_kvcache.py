"""KvCache and rope on torch tensors as the served model lays them out: a gate beside each query, outputs in buffers of the caller's, one step captured."""
import numpy as np
import pytest

import kvcache as K
from kv8_helpers import Cache, attention

pytestmark = pytest.mark.gpu
HQ, HKV, DH, ROT = 8, 2, 64, 32


def setup(seed, total):
    import torch

    torch.manual_seed(seed)
    c = K.KvCache(1, 30, 3, 500, HQ, HKV, DH)
    freq, ms = K.rope_freq(ROT, device="cuda")
    p = torch.randn(total, 2 * HQ * DH + 2 * HKV * DH, device="cuda")  # query, gate, query, gate .., k, v
    return c, freq, ms, p


def parts(p):
    q = 2 * HQ * DH
    return p[:, :q], p[:, DH:q], p[:, q:q + HKV * DH], p[:, q + HKV * DH:]


@pytest.mark.parametrize("rows,lens", [([1, 1, 1], [70, 300, 1]), ([40, 3, 129], [40, 3, 200])])
def test_gate_beside_each_query(rows, lens):
    """The bits of a gate copied out, and the values of the definition."""
    import torch

    c, freq, ms, p = setup(1, sum(lens))
    c.step([m - n for n, m in zip(rows, lens)])
    first = K.Batch([m - n for n, m in zip(rows, lens)], [m - n for n, m in zip(rows, lens)], "cuda")
    kv = torch.randn(2, first.total + 1, HKV * DH, device="cuda")
    c.append(0, kv[0], kv[1], first)
    b = c.step(rows)
    qx, gate, kx, vx = parts(p)
    q = K.rope(qx[:b.total], HQ, DH, b.pos, freq, ms, head_stride=2 * DH)
    k = K.rope(kx[:b.total], HKV, DH, b.pos, freq, ms, f32=True)
    c.append(0, k, vx[:b.total], b)
    y = c.attend(0, q, b, gate=gate, gate_stride=2 * DH)
    g = gate.as_strided((p.shape[0], HQ, DH), (p.stride(0), 2 * DH, 1), gate.storage_offset()).reshape(-1, HQ * DH).contiguous()
    z = c.attend(0, q, b, gate=g)
    torch.cuda.synchronize()
    assert torch.equal(y, z)
    host = Cache(np.random.default_rng(0), [0, 0, 0], HKV, DH, spare=30, maxp=c.maxp, content="none")
    host.table = c.table.cpu().numpy()
    host.k, host.v = host.unpack(c.kq[0].cpu().numpy(), c.vq[0].cpu().numpy())
    host.ks, host.vs = c.ks[0].cpu().numpy(), c.vs[0].cpu().numpy()
    f = lambda t: t[:b.total].double().cpu().numpy().reshape(b.total, HQ, DH)
    want, bound = attention(host, f(q), b.start.tolist(), b.len.tolist(), DH ** -0.5, f(g))
    assert (np.abs(f(y) - want) <= bound).all()


def test_rope_into_buffers():
    """f32 and bf16 buffers with strides of their own, and x itself: the bits of a new tensor; what lies beside is left alone."""
    import torch

    c, freq, ms, p = setup(2, 50)
    pos = torch.arange(50, dtype=torch.int32, device="cuda")
    for dt in (torch.float32, torch.bfloat16):
        want = K.rope(parts(p)[0], HQ, DH, pos, freq, ms, head_stride=2 * DH, f32=dt == torch.float32)
        buf = torch.full((52, HQ * DH + 16), 7.0, dtype=dt, device="cuda")
        out = K.rope(parts(p)[0], HQ, DH, pos, freq, ms, head_stride=2 * DH, out=buf[:50, 8:8 + HQ * DH])
        torch.cuda.synchronize()
        assert out.data_ptr() == buf.data_ptr() + 8 * buf.element_size() and torch.equal(out, want)
        assert (buf[:, :8] == 7).all() and (buf[:, 8 + HQ * DH:] == 7).all() and (buf[50:] == 7).all()
        x = parts(p)[2].to(dt).contiguous()
        want = K.rope(x, HKV, DH, pos, freq, ms, f32=dt == torch.float32)
        K.rope(x, HKV, DH, pos, freq, ms, out=x)
        torch.cuda.synchronize()
        assert torch.equal(x, want)


def test_captured_step_of_an_attention_layer():
    """rope, append and attend captured together on tensors: each replay has the eager bits, while the sequences grow."""
    import torch

    a, freq, ms, p = setup(3, 3)
    e = K.KvCache(1, 30, 3, 500, HQ, HKV, DH)
    k0 = torch.randn(2, 180, HKV * DH, device="cuda")
    for c in (a, e):
        c.append(0, k0[0], k0[1], c.step([60, 5, 115]))
    batch, eager = a.step([1, 1, 1]), e.step([1, 1, 1])
    q, k, y = (torch.zeros(3, n * DH, dtype=t, device="cuda") for n, t in ((HQ, torch.bfloat16), (HKV, torch.float32), (HQ, torch.bfloat16)))

    def layer(c, b):
        qx, gate, kx, vx = parts(p)
        K.rope(qx, HQ, DH, b.pos, freq, ms, head_stride=2 * DH, out=q)
        K.rope(kx, HKV, DH, b.pos, freq, ms, out=k)
        c.append(0, k, vx, b)
        return c.attend(0, q, b, gate=gate, gate_stride=2 * DH, out=y, max_len=500)

    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        layer(a, batch)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            layer(a, batch)
    torch.cuda.synchronize()
    layer(e, eager)  # the first tokens take the place of other ones in both, whose scales stay
    for n in range(5):
        p.copy_(torch.randn_like(p))
        if n:
            nxt, eager = a.step([1, 1, 1]), e.step([1, 1, 1])
            batch.pos.copy_(nxt.pos), batch.len.copy_(nxt.len)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (q, k, y, a.kq, a.vq, a.ks, a.vs)]
        layer(e, eager)
        torch.cuda.synchronize()
        for g, w in zip(got, (q, k, y, e.kq, e.vq, e.ks, e.vs)):
            assert torch.equal(g, w), n


def test_outgrown_workspaces_stay_small():
    """Captured calls may use them, so they are kept: all together they are smaller than the one in use, however slowly the calls grow."""
    import torch

    c = K.KvCache(1, 70, 64, 5000, 16, 1, 64)
    sizes = set()
    for n in range(1, 65):
        b = c.step([int(i < n) for i in range(64)])
        q = torch.randn(b.total, 16 * 64, device="cuda").to(torch.bfloat16)
        c.attend(0, q, b, max_len=5000)
        ws = c._ws[torch.cuda.current_stream().cuda_stream]
        sizes.add(ws.numel())
        assert sum(o.numel() for o in c._old) < ws.numel(), n
    assert len(c._old) >= 3 and len(sizes) == len(c._old) + 1
    torch.cuda.synchronize()
