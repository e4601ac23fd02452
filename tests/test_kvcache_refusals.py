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
