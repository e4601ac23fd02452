"""What KvCache refuses, and what it leaves as it was (CPU)."""
import pytest
import torch

import kvcache as K
from test_kvcache import cache


def test_batch_of_another_cache():
    """A call reads start, len and the table of as many sequences as its cache has: a batch of fewer or more is refused."""
    a, b = cache(), cache(seqs=8, pages=40)
    kv, q = torch.zeros(3, 64), torch.zeros(3, 128, dtype=torch.bfloat16)
    for c, other in ((a, b.step([1, 1, 1, 0, 0, 0, 0, 0])), (b, a.step([1, 1, 1]))):
        for call in (lambda: c.append(0, kv, kv, other), lambda: c.read(0, other), lambda: c.attend(0, q, other)):
            with pytest.raises(ValueError, match="batch"):
                call()


@pytest.mark.parametrize("fails", ["Batch", "table"])
def test_step_that_fails_leaves_the_cache_as_it_was(monkeypatch, fails):
    """No memory for what a step makes on the device: no token is counted and no page taken."""
    c = cache()
    c.step([65, 0, 1])
    before = (list(c.lens), c.table.clone(), list(c.free_pages), [list(h) for h in c.held])

    def full(*a, **k):
        raise MemoryError("no room")

    with monkeypatch.context() as m:
        if fails == "Batch":
            m.setattr(K, "Batch", full)
        else:
            m.setattr(torch, "tensor", full)
        with pytest.raises(MemoryError, match="no room"):
            c.step([10, 64, 70])
    assert (c.lens, c.free_pages, c.held) == (before[0], before[2], before[3]) and torch.equal(c.table, before[1])
    b = c.step([10, 64, 70])
    assert b.len.tolist() == [75, 64, 71] and c.table.tolist() == [[0, 1, -1, -1], [3, -1, -1, -1], [2, 4, -1, -1]]


def test_outputs_and_gates_that_do_not_fit():
    c = cache()
    b = c.step([2, 1, 0])
    q, x = torch.zeros(3, 128, dtype=torch.bfloat16), torch.zeros(3, 64)
    for gate, stride in ((torch.zeros(3, 256), 64), (torch.zeros(3, 223), 64), (torch.zeros(3, 224), None), (torch.zeros(2, 224), 64), (torch.zeros(3, 224).double(), 64), (torch.zeros(224, 3).t(), 64)):
        with pytest.raises(ValueError, match="gate"):
            c.attend(0, q, b, gate=gate, gate_stride=stride)
    for out in (torch.zeros(2, 64), torch.zeros(3, 63), torch.zeros(3, 64).half(), torch.zeros(64, 3).t(), torch.zeros(3, 1, 64)):
        with pytest.raises(ValueError, match="out"):
            K.rope(x, 2, 32, b.pos, torch.zeros(8), out=out)
