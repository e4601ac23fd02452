"""MoeStack.rows, MoeStack.forward and prefill with the next layer's norm, on synthetic checkpoints: routing
bit for bit with the oracle on the same normalised rows, outputs within the layer tests' 1e-3 + 1e-3 |ref|.

The normalised rows against 64 bits: a row's sum of squares is within 38 u (u = 2^-24), rsqrt and two products add
6 u, and the rounding to bf16 2^-8 of the value: 2^-8 + 32 u in all."""
import numpy as np
import pytest

import checkpoint as C
import oracle as O
import synth
from ckpt_helpers import write_checkpoint, write_fp8_source
from helpers import assert_close, bits, dev, host

pytestmark = pytest.mark.gpu
E, H, I, K = 64, 2048, 512, 8


def norm_ok(hn, x, nw):
    import torch

    want = x.astype(np.float64)
    want = want / np.sqrt((want * want).mean(-1, keepdims=True) + 1e-6) * nw
    got = synth.bf16_to_f32(host(hn.view(torch.int16)).view(np.uint16)).astype(np.float64)
    assert (np.abs(got - want) <= (2.0 ** -8 + 32 * 2.0 ** -24) * np.abs(want)).all()
    return got.astype(np.float32)


def write_checkpoint_layers(path, n):
    return write_checkpoint(path, [60 + j for j in range(n)], E=E)


def make(tmp_path, kind, n):
    """(stack, oracle layers)"""
    if kind == "q4":
        layers = write_checkpoint_layers(tmp_path, n)
        return C.MoeStack(str(tmp_path)), layers
    conv, src = tmp_path / "conv", tmp_path / "fp8"
    conv.mkdir(), src.mkdir()
    layers = write_checkpoint_layers(conv, n)
    fp8 = [synth.make_layer(80 + j, E=E, fmt="ref", kind="fp8", quick=True) for j in range(n)]
    write_fp8_source(str(src), fp8, E)
    for L, F in zip(layers, fp8):
        L.update({k: F[k] for k in ("kind", "gu_q", "gu_s", "d_q", "d_s", "sc_kind")})
    return C.MoeStack(str(conv), fp8_dir=str(src), vram_layers=1), layers


@pytest.mark.parametrize("kind", ["q4", "fp8"])
def test_rows_and_forward(tmp_path, kind):
    """1, 2, 5 and 33 rows through two layers (fp8: the second's experts in pinned host memory), each layer against the
    oracle on the rows that went into it; forward gives the bits of the layers one after the other."""
    import torch

    st, layers = make(tmp_path, kind, 2)
    for rows in (33, 1, 5, 2):
        x0 = np.random.default_rng(rows).normal(0, 1, (rows, H)).astype(np.float32)
        x = dev(x0).view(rows, H)
        hn = torch.empty((rows, H), dtype=torch.bfloat16, device="cuda")
        for l, L in enumerate(layers):
            xin, kept = host(x).copy(), {}
            st.lib.dr_block_norm(None, 0, x.data_ptr(), H, None, None, 0, 0, None, 0.0, 1.0, st.layers[l]["nw"].data_ptr(), 1e-6, None, 0,
                                 hn.data_ptr(), H, rows, H, torch.cuda.current_stream().cuda_stream)
            st.rows(l, x, hn, keep=kept)
            torch.cuda.synchronize()
            xn = norm_ok(hn, xin, L["nw"])
            raw = host(hn.view(torch.int16)).view(np.uint16)
            ri, rw, rs = O.moe_topk(O.router_logits_rows(raw, L["router"], rows, E + 1, H), rows, E, K, E + 1)
            np.testing.assert_array_equal(host(kept["idx"]).ravel(), np.asarray(ri).ravel())
            np.testing.assert_array_equal(bits(host(kept["wts"])).ravel(), bits(rw).ravel())
            np.testing.assert_array_equal(bits(host(kept["sgate"])).ravel(), bits(rs).ravel())
            ri, rw = np.asarray(ri).reshape(rows, K), np.asarray(rw).reshape(rows, K)
            for r in range(0, rows, max(1, rows // 5)):
                _, ry = O.moe_decode(L, xn[r], ri[r], rw[r], np.asarray(rs).ravel()[r], xin[r], H, I, K)
                assert_close(host(x)[r], ry, what=f"{kind}, {rows} rows, layer {l}, row {r}")
        z = dev(x0).view(rows, H)
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s):
            st.forward(z)
        torch.cuda.synchronize()
        np.testing.assert_array_equal(bits(host(z)), bits(host(x)))


def test_forward_of_a_prefill(tmp_path):
    """100 rows: prefill's combine leaves the next layer's norm, also in place of this layer's and in chunks; x is the prefill's
    without it but for the order of the sums, and forward gives the bits of the layers one after the other."""
    import torch

    st, layers = make(tmp_path, "q4", 2)
    rows = 100
    x0 = np.random.default_rng(9).normal(0, 1, (rows, H)).astype(np.float32)
    x, a = dev(x0).view(rows, H), dev(x0).view(rows, H)
    hn = torch.empty((rows, H), dtype=torch.bfloat16, device="cuda")
    lib, sp = st.lib, torch.cuda.current_stream().cuda_stream
    lib.dr_block_norm(None, 0, x.data_ptr(), H, None, None, 0, 0, None, 0.0, 1.0, st.layers[0]["nw"].data_ptr(), 1e-6, None, 0, hn.data_ptr(), H,
                      rows, H, sp)
    h0 = hn.clone()
    st.prefill(0, a, h0)
    st.prefill(0, x, hn, chunk=48, nw_next=st.layers[1]["nw"], hn_next=hn)
    torch.cuda.synchronize()
    # the same 10 terms in another order: each sum is within 10 u of the terms' magnitudes, the two 1.2e-6 apart; terms that cancel may
    # be larger than what they leave, by up to eight times here
    d = np.abs(host(x).astype(np.float64) - host(a))
    assert (d <= 1e-5 * (np.abs(host(a)) + np.abs(host(a) - x0).max())).all()
    norm_ok(hn, host(x), layers[1]["nw"])
    st.prefill(1, x, hn)
    z = dev(x0).view(rows, H)
    st.forward(z, chunk=48)
    torch.cuda.synchronize()
    np.testing.assert_array_equal(bits(host(z)), bits(host(x)))
    with pytest.raises(ValueError, match="belong together"):
        st.prefill(0, x, hn, nw_next=st.layers[1]["nw"])
    with pytest.raises(ValueError, match="65 rows"):
        st.rows(0, torch.zeros(65, H, device="cuda"), hn)


def test_forward_captured(tmp_path):
    """forward captured for 3 rows and replayed on new rows, with eager calls of 1 and 40 rows on the same stream in between; a
    first call under capture is refused."""
    import ctypes

    import torch

    st, _ = make(tmp_path, "q4", 2)
    s, g = torch.cuda.Stream(), ctypes.c_void_p()
    x, z = torch.randn(3, H, device="cuda"), torch.randn(40, H, device="cuda")
    torch.cuda.synchronize()
    st.lib.dr_graph_begin(s.cuda_stream)
    try:
        with pytest.raises(RuntimeError, match="before capturing"):
            st.forward(x, stream=s.cuda_stream)
    finally:
        assert st.lib.dr_graph_end(s.cuda_stream, ctypes.byref(g)) == 0
    st.lib.dr_graph_destroy(g)
    one = x.clone()
    torch.cuda.synchronize()
    st.forward(one, stream=s.cuda_stream)
    s.synchronize()
    g = ctypes.c_void_p()
    st.lib.dr_graph_begin(s.cuda_stream)
    st.forward(x, stream=s.cuda_stream)
    assert st.lib.dr_graph_end(s.cuda_stream, ctypes.byref(g)) == 0
    try:
        for _ in range(4):
            x.copy_(torch.randn(3, H, device="cuda"))
            want, one, many = x.clone(), z[:1].clone(), z.clone()
            torch.cuda.synchronize()
            st.forward(want, stream=s.cuda_stream)
            st.forward(one, stream=s.cuda_stream)
            st.forward(many, stream=s.cuda_stream)
            st.lib.dr_graph_launch(g, s.cuda_stream)
            s.synchronize()
            assert torch.equal(x, want)
    finally:
        st.lib.dr_graph_destroy(g)
