"""What dr_moe_combine_norm hands to its kernel, seen on the CPU: a library of our own in front of the HIP runtime keeps the
arguments of the launch instead of launching."""
import shutil
import subprocess
import sys

import pytest

import dramamoe as D

STUB = r"""
#include <string.h>
typedef struct { unsigned x, y, z; } dim3_t;
unsigned long seen[21];  /* the kernel's one argument, a structure of 168 bytes */
int launches;
int __hipPushCallConfiguration(dim3_t g, dim3_t b, unsigned long m, void* s) { return 0; }
int __hipPopCallConfiguration(dim3_t* g, dim3_t* b, unsigned long* m, void** s) {
  dim3_t one = {1, 1, 1};
  *g = *b = one, *m = 0, *s = 0;
  return 0;
}
int hipLaunchKernel(const void* f, dim3_t g, dim3_t b, void** args, unsigned long m, void* s) {
  memcpy(seen, args[0], sizeof seen);
  ++launches;
  return 0;
}
"""

CHILD = r"""
import ctypes, sys
stub = ctypes.CDLL(sys.argv[1], mode=ctypes.RTLD_GLOBAL)
sys.path.insert(0, sys.argv[2])
import dramamoe as D
shared = int(sys.argv[3]) or None
Y, SLOT, WTS, SGATE, X, NW, XO, HN = (0x10000 * k for k in range(1, 9))
rc = D.lib().raw("dr_moe_combine_norm")(Y, SLOT, WTS, SGATE, shared, 8, X, 64, None, None, 0, 0, None, 1.0, 1.0, NW, 1e-6,
                                        XO, 64, HN, 64, 5, 64, None)
seen = list((ctypes.c_ulong * 21).in_dll(stub, "seen"))
at = seen.index(SLOT)
assert rc == 0 and ctypes.c_int.in_dll(stub, "launches").value == 1 and seen[at + 1] == WTS and seen[at + 3] == (shared or 0), seen
print(seen[at + 2] == SGATE, seen[at + 2])
"""


@pytest.mark.skipif(shutil.which("gcc") is None, reason="no gcc")
def test_sgate_stays_out_without_shared(tmp_path):
    """The kernel reads the gate logits it is given: without a shared expert's rows it gets none, as they may be of any length
    then."""
    (tmp_path / "stub.c").write_text(STUB)
    so = str(tmp_path / "stub.so")
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", so, str(tmp_path / "stub.c")], check=True)

    def given(shared):
        r = subprocess.run([sys.executable, "-c", CHILD, so, D.HERE, str(shared)], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0, r.stdout + r.stderr
        return r.stdout.split()

    assert given(0x90000) == ["True", str(0x40000)]
    assert given(0) == ["False", "0"]


@pytest.mark.gpu
def test_sgate_without_shared():
    """One NaN for all rows in place of their gate logits: the bits of a call without."""
    import torch

    rows, h, topk = 37, 1024, 4
    torch.manual_seed(8)
    y, x = torch.randn(rows * topk, h, device="cuda"), torch.randn(rows, h, device="cuda")
    slot, w = torch.randperm(rows * topk, device="cuda").to(torch.int32), torch.rand(rows, topk, device="cuda")
    nw, nan = torch.randn(h, device="cuda"), torch.full((1,), float("nan"), device="cuda")
    outs = []
    for sg in (None, nan):
        xo, hn = torch.empty_like(x), torch.empty(rows, h, dtype=torch.bfloat16, device="cuda")
        D.lib().dr_moe_combine_norm(D.ptr(y), D.ptr(slot), D.ptr(w), D.ptr(sg), None, topk, D.ptr(x), h, None, None, 0, 0, None, 1.0, 1.0,
                                    D.ptr(nw), 1e-6, D.ptr(xo), h, D.ptr(hn), h, rows, h, D.stream_ptr())
        outs.append((xo, hn))
    torch.cuda.synchronize()
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    assert torch.isfinite(outs[0][0]).all()
