"""dr_attn_kv8 where what the host says of a call (its most rows, its rows of no sequence) and the call itself are far apart.  Tolerances:
kv8_helpers.attention."""
import numpy as np
import pytest

from test_gpu_attn_kv8 import Call, cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,lens,hq,hkv,d,most", [([20, 3, 9, 1], [300, 90, 9, 70], 4, 2, 64, 5), ([20, 3, 9], [3000, 900, 700], 8, 2, 128, 4), ([700, 40, 701, 130], [900, 40, 701, 200], 8, 1, 128, 150),
                                                     ([300, 40, 130], [300, 700, 200], 8, 2, 256, 100), ([100, 60, 130], [100, 60, 200], 2, 1, 64, 64),
                                                     # tiles that the first sequence's surplus would take from the others; a sequence folded at an end that is not the host's
                                                     ([600, 40], [700, 60], 32, 1, 64, 70), ([1700], [1700], 32, 1, 32, 1500)])
def test_more_rows_than_the_host_says(rows, lens, hq, hkv, d, most):
    """The rows past the limit are undefined; those before it, and the other sequences', are right."""
    import torch

    call = Call(cache(81, lens, hkv, d), rows, lens, hq, max_rows=most, behind=1)
    y = call.run()
    torch.cuda.synchronize()
    want, bound = call.reference()
    got = y.double().cpu().numpy()[:, :hq * d].reshape(want.shape)
    for i, n in enumerate(rows):
        own = slice(call.start[i], call.start[i] + min(n, most))
        assert (np.abs(got[own] - want[own]) <= bound[own]).all(), i
    assert (got[-1] == 7).all()


PADDED = [([1], [6000], 32, 1, 256, 500), ([1, 1, 0], [3000, 70, 9], 8, 2, 64, 77), ([3, 1, 2], [2000, 900, 1], 20, 4, 80, 9), ([20], [4000], 4, 2, 64, 130), ([150, 0], [2500, 5], 4, 1, 128, 400),
          ([40, 33], [2700, 60], 8, 1, 192, 90)]


@pytest.mark.parametrize("rows,lens,hq,hkv,d,behind", PADDED)
@pytest.mark.parametrize("gate", [False, True])
def test_rows_of_no_sequence(rows, lens, hq, hkv, d, behind, gate):
    """Split calls with more rows behind the last sequence than the sequences can have: the bits of the call without them, whose workspace is as large."""
    import torch

    c = cache(83, lens, hkv, d)
    call, bare = Call(c, rows, lens, hq, gate=gate, behind=behind, pad=1), Call(c, rows, lens, hq, gate=gate, pad=1)
    assert bare.ws.numel() <= call.ws.numel() <= len(rows) * max(rows) / sum(rows) * bare.ws.numel() + 512 and bare.ws.numel() > 4096
    y = call.run()
    torch.cuda.synchronize()
    call.check(y)
    n = sum(rows)
    bare.q.copy_(call.q[:n])
    if gate:
        bare.gate.copy_(call.gate[:n])
    z = bare.run()
    torch.cuda.synchronize()
    assert torch.equal(y[:n], z)
    # in the queries' place, and rows of none in front
    if call.ldq == call.ldy:
        call.run(y=call.q)
        torch.cuda.synchronize()
        assert torch.equal(call.q[:n], y[:n])
    k = behind // 2
    shift = torch.full_like(y, 7.0)
    call.ts += k
    call.q[k:k + n] = bare.q
    if gate:
        call.gate[k:k + n] = bare.gate
    call.run(y=shift)
    torch.cuda.synchronize()
    assert torch.equal(shift[k:k + n], z) and (shift[:k] == 7).all() and (shift[k + n:] == 7).all()
