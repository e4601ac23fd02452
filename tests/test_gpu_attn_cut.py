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
