"""rope_freq and the host side of KvCache (CPU)."""
import math

import pytest
import torch

import kvcache as K


def test_rope_freq_plain_and_linear():
    f, ms = K.rope_freq(64, 10000.0)
    want = torch.tensor([10000.0 ** (-2 * j / 64) for j in range(32)], dtype=torch.float64).float()
    assert torch.equal(f, want) and ms == 1
    g, ms = K.rope_freq(64, 10000.0, "linear", 8.0)
    assert torch.equal(g, (want.double() / 8).float()) or torch.allclose(g, f / 8, rtol=2 ** -23, atol=0)
    assert ms == 1 and K.rope_freq(0)[0].numel() == 0


def test_rope_freq_base_draws_out_the_slowest():
    f, _ = K.rope_freq(128, 10000.0)
    g, _ = K.rope_freq(128, 10000.0, "base", 4.0)
    assert g[0] == f[0] == 1 and math.isclose(float(f[-1] / g[-1]), 4.0, rel_tol=1e-5) and (g <= f).all()


def test_rope_freq_yarn():
    f, _ = K.rope_freq(128, 10000.0)
    g, ms = K.rope_freq(128, 10000.0, "yarn", 8.0, trained=4096)
    turns = f.double() * 4096 / (2 * math.pi)
    assert (g[turns > 40] == f[turns > 40]).all() and torch.allclose(g[turns < 0.8], f[turns < 0.8] / 8, rtol=1e-6)
    assert ((g <= f) & (g >= f / 8 * (1 - 1e-6))).all() and math.isclose(ms, 0.1 * math.log(8) + 1)


@pytest.mark.parametrize("bad", [dict(rot=3), dict(rot=-2), dict(rot=4, scaling="other"), dict(rot=4, factor=0.5), dict(rot=4, theta=1.0)])
def test_rope_freq_refusals(bad):
    with pytest.raises(ValueError):
        K.rope_freq(**bad)


def cache(**kw):
    a = dict(layers=2, pages=6, seqs=3, max_len=200, hq=4, hkv=2, d=32, device="cpu")
    return K.KvCache(**{**a, **kw})


@pytest.mark.parametrize("bad", [dict(layers=0), dict(pages=0), dict(seqs=0), dict(max_len=0), dict(hq=3), dict(hkv=0), dict(d=24), dict(d=272), dict(hq=1026)])
def test_cache_refusals(bad):
    with pytest.raises(ValueError):
        cache(**bad)


def test_pages_of_sequences():
    c = cache()
    b = c.step([65, 0, 1])
    assert b.start.tolist() == [0, 65, 65, 66] and b.len.tolist() == [65, 0, 1] and b.max_rows == 65 and b.max_len == 65 and b.total == 66
    assert b.pos.tolist() == list(range(65)) + [0]
    assert c.table.tolist() == [[0, 1, -1, -1], [-1] * 4, [2, -1, -1, -1]]
    b = c.step([1, 128, 63])
    assert b.pos.tolist() == [65] + list(range(128)) + list(range(1, 64)) and b.len.tolist() == [66, 128, 64]
    assert c.table.tolist() == [[0, 1, -1, -1], [3, 4, -1, -1], [2, -1, -1, -1]]
    before = (list(c.lens), c.table.clone(), list(c.free_pages))
    with pytest.raises(MemoryError):
        c.step([0, 1, 1])  # two pages, one is free
    with pytest.raises(ValueError):
        c.step([135, 0, 0])
    with pytest.raises(ValueError):
        c.step([1, 1])
    with pytest.raises(ValueError):
        c.step([1, -1, 0])
    assert c.lens == before[0] and torch.equal(c.table, before[1]) and c.free_pages == before[2]
    c.truncate(1, 64)
    assert c.table[1].tolist() == [3, -1, -1, -1] and c.lens[1] == 64
    c.truncate(0, 65)  # the last token of a page: the page stays
    assert c.table[0].tolist() == [0, 1, -1, -1] and c.lens[0] == 65
    with pytest.raises(ValueError):
        c.truncate(0, 66)
    c.truncate(0, 0)
    assert sorted(c.free_pages) == [0, 1, 4, 5]
    b = c.step([200, 0, 0])
    assert sorted(c.table[0].tolist()) == [0, 1, 4, 5] and b.pos.tolist() == list(range(200))


def test_tensors_that_do_not_fit():
    c = cache()
    b = c.step([2, 1, 0])
    ok = torch.zeros(3, 64)
    for k, v in ((torch.zeros(2, 64), ok), (ok, torch.zeros(3, 63)), (ok.half(), ok.half()), (ok, ok.bfloat16()), (torch.zeros(64, 3).t(), ok)):
        with pytest.raises(ValueError):
            c.append(0, k, v, b)
    q = torch.zeros(3, 128, dtype=torch.bfloat16)
    for args in ((q.float(),), (q[:2],), (q, None, torch.zeros(3, 64)), (q, None, None, torch.zeros(3, 128))):
        with pytest.raises(ValueError):
            c.attend(0, args[0], b, *args[1:])
    with pytest.raises(ValueError):
        K.rope(ok.half(), 2, 32, b.pos, torch.zeros(8))
    with pytest.raises(ValueError):
        K.rope(ok, 3, 32, b.pos, torch.zeros(8))
    with pytest.raises(ValueError):
        K.rope(ok, 2, 32, b.pos.long(), torch.zeros(8))
    with pytest.raises(ValueError):
        K.rope(ok, 2, 32, b.pos, torch.zeros(17))
    with pytest.raises(ValueError):
        K.rope(ok, 2, 32, b.pos, torch.zeros(8), nw=torch.zeros(33))
