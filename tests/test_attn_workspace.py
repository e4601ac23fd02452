"""Sizes of dr_attn_kv8's workspace (CPU)."""
import dramamoe as D


def ws(*a):
    return D.lib().cdll.dr_attn_kv8_ws(*a)


def test_rows_of_no_sequence_need_no_parts():
    """rows, seqs, max_rows, max_len, hq, hkv, d: what lies behind the last sequence does not count, with few columns and with tiles."""
    for seqs, most, rest in ((1, 1, (60000, 32, 1, 256)), (8, 1, (60000, 32, 2, 256)), (3, 20, (9000, 4, 2, 64)), (1, 150, (20000, 4, 1, 128))):
        bare = ws(seqs * most, seqs, most, *rest)
        assert bare > 256
        for rows in (seqs * most + 1, 4096, 8192, 1 << 20):
            assert ws(rows, seqs, most, *rest) <= bare, (rows, seqs, most, rest)


def test_parts_of_real_calls_stay_small():
    """Any number of sequences of single rows, drafts or prompts on up to 100000 tokens: no more than a part of each row for each of a few thousand blocks of threads."""
    for d in (64, 128, 256):
        for hq, hkv in ((8, 8), (16, 2), (32, 8), (64, 1)):
            for seqs, most in ((1, 1), (7, 1), (64, 1), (500, 1), (3, 5), (40, 8), (1, 400), (9, 70)):
                assert ws(seqs * most, seqs, most, 100000, hq, hkv, d) <= 512 << 20, (seqs, most, hq, hkv, d)
