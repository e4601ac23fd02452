"""The cut that dr_attn_kv8 takes for given sizes: the library's own plan(), compiled for the host."""
import ctypes as C
import functools
import os
import subprocess
import tempfile

import dramamoe as D

SRC = """#include "attn_plan.hpp"
extern "C" void cut(int rows, int seqs, int max_rows, int max_len, int hq, int hkv, int d, int* o) {
  const drm::Plan p = drm::plan(rows, seqs, max_rows, max_len, hq, hkv, d);
  const int v[] = {p.few, p.scan, p.fold, p.mt, p.cols, p.nw, p.splits, p.chunk, (int)p.tiles};
  for (int i = 0; i < 9; ++i) o[i] = v[i];
}
"""


@functools.lru_cache(None)
def _lib():
    with tempfile.TemporaryDirectory() as t:
        src, lib = os.path.join(t, "cut.cpp"), os.path.join(t, "cut.so")
        with open(src, "w") as f:
            f.write(SRC)
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-I", os.path.join(D.HERE, "csrc"), src, "-o", lib], check=True)
        return C.CDLL(lib)


def plan(rows, seqs, max_rows, max_len, hq, hkv, d):
    o = (C.c_int * 9)()
    _lib().cut(rows, seqs, max_rows, max_len, hq, hkv, d, o)
    return dict(zip(("few", "scan", "fold", "mt", "cols", "nw", "splits", "chunk", "tiles"), o))


def name(rows, lens, hq, hkv, d, behind=0, max_len=None, max_rows=None):
    """What a call of those rows and tokens is: the kernel (heads rounded up to what it is built for), its columns, and how it is cut."""
    p = plan(sum(rows) + behind, len(rows), max(rows) if max_rows is None else max_rows, max(max(lens), 0) if max_len is None else max_len, hq, hkv, d)
    dc = 64 * ((d + 63) // 64)
    if p["few"]:
        return f"few {16 * p['mt']} d{dc}" + (" several" if p["cols"] > 1 else "") + (" split" if p["splits"] > 1 else "")
    return f"tiles {p['nw']} d{dc}" + (" several" if p["scan"] else "") + (" split" if p["splits"] > 1 else "") + (" folded" if p["fold"] else "")


def blocks_in_a_row(rows, lens, hq, hkv, d, behind=0, max_len=None, max_rows=None):
    """Cached blocks that one wave (few columns) or one block of threads (tiles) walks over in the longest sequence."""
    p = plan(sum(rows) + behind, len(rows), max(rows) if max_rows is None else max_rows, max(max(lens), 0) if max_len is None else max_len, hq, hkv, d)
    nb = (max(lens) + 63) // 64
    n = min(nb, max((nb + p["splits"] - 1) // p["splits"], p["chunk"]))
    return (n + 3) // 4 if p["few"] else n
