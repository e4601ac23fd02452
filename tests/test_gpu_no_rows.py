"""A step in which no sequence has a new row, through torch tensors."""
import pytest

import kvcache as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("f32", [False, True])
def test_batch_without_rows(f32):
    import torch

    c = K.KvCache(1, 4, 2, 100, 4, 2, 32)
    b = c.step([0, 0])
    freq, ms = K.rope_freq(16, device="cuda")
    e = lambda n, dt=torch.float32: torch.empty(0, n, dtype=dt, device="cuda")
    q = K.rope(e(4 * 64), 4, 32, b.pos, freq, ms, head_stride=64, f32=f32)
    k = K.rope(e(64, torch.bfloat16), 2, 32, b.pos, freq, ms, nw=torch.ones(32, device="cuda"), f32=f32)
    assert q.shape == (0, 128) and k.shape == (0, 64) and q.dtype == k.dtype == (torch.float32 if f32 else torch.bfloat16)
    c.append(0, k, k, b)
    assert c.attend(0, q.to(torch.bfloat16), b).shape == (0, 128) and c.read(0, b)[0].shape == (0, 64)
    torch.cuda.synchronize()
