"""Which cuts the tests of dr_attn_kv8 take: every kernel and every way to split it, and each case the one that it is there for (CPU)."""
import random
import shutil

import pytest

import attn_cut
import test_gpu_attn_cut as C
import test_gpu_attn_kv8 as A
import test_gpu_attn_kv8_tiles as T
import test_gpu_attn_scores as S
import test_gpu_attn_windows as W

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="no g++")


@pytest.mark.parametrize("case", W.WINDOWS + W.OTHERS)
def test_windows_take_their_cut(case):
    cut, blocks, (rows, lens, hq, hkv, d), gate, behind, max_len = case
    a = (rows, lens, hq, hkv, d, behind, max_len, W.most_rows(case))
    assert (attn_cut.name(*a), attn_cut.blocks_in_a_row(*a)) == (cut, blocks)


def cuts_that_are_checked():
    """Cuts of all cases whose values are checked."""
    out = [attn_cut.name(rows, lens, hq, hkv, d, behind) for rows, lens, hq, hkv, d, gate, behind, pad in A.CASES]
    out += [attn_cut.name(rows, lens, hq, hkv, d, 1) for rows, lens, hq, hkv, d, gate in A.CUTS]
    out += [attn_cut.name(rows, lens, hq, hkv, d) for rows, lens, hq, hkv, d in T.SHAPES + T.SMALL + S.SHAPES]
    out += [attn_cut.name(rows, lens, hq, hkv, d, behind) for rows, lens, hq, hkv, d, behind in C.PADDED]
    return set(out) | {case[0] for case in W.WINDOWS + W.OTHERS}


def test_every_cut_is_tested():
    """A sweep over sizes finds no cut that no GPU test takes."""
    rng, found = random.Random(1), set()
    size = lambda top: int(2 ** rng.uniform(0, top))
    for _ in range(60000):
        d, hkv, g, seqs, rows = rng.choice([32, 64, 80, 128, 160, 192, 240, 256]), rng.choice([1, 2, 4]), rng.choice([1, 2, 4, 8, 16, 32]), rng.choice([1, 2, 3, 9, 40, 200]), size(11)
        many = [rows] + [max(1, rows // 3)] * (seqs - 1)
        behind = rng.choice([0, 0, 1, 2900, 4300])
        found.add(attn_cut.name(many, [rows + size(12.5)] * seqs, g * hkv, hkv, d, behind, None, sum(many) + behind if behind > 1 else None))
    assert len(found) >= 30 and not sorted(found - cuts_that_are_checked())


def test_cuts_of_real_calls():
    """The cut's limits: as many splits as blocks at most, chunks that cover the longest sequence, tiles that cover all rows."""
    for d in (16, 64, 80, 128, 176, 256):
        for hq, hkv in ((1, 1), (8, 2), (16, 1), (32, 32), (64, 1)):
            for seqs, most in ((1, 1), (3, 5), (1, 70), (64, 1), (7, 400), (1, 4096), (300, 2)):
                for behind in (0, 5, 3000):
                    for n in (0, 1, 64, 65, 300, 5000, 100000):
                        p, g = attn_cut.plan(seqs * most + behind, seqs, most, n, hq, hkv, d), hq // hkv
                        nb = (n + 63) // 64
                        assert 1 <= p["splits"] <= 128 and p["chunk"] >= 1 and (p["splits"] == 1 or p["splits"] <= nb) and p["splits"] * p["chunk"] >= nb
                        if p["few"]:
                            assert p["tiles"] == seqs and p["cols"] * 16 * p["mt"] >= most * g and p["chunk"] % 4 == 0
                        else:
                            per = (most * g + 32 * p["nw"] - 1) // (32 * p["nw"])
                            assert p["tiles"] >= seqs * per and p["cols"] == 1 and (p["scan"] or per == 1) and (not p["fold"] or p["splits"] == 1)
