"""dr_gemm_q8_lora*, more than 64 rows: t = s A x travels as three bf16 planes that sum to the fp32 number it is rounded to.

W is zero, x has one input, each adapter one rank with B = 1: A x is one product of two bf16 numbers, exact in fp32, and
y = fp32(s A x) to the bit, as for 64 rows or fewer."""
import numpy as np
import pytest

import dramamoe as D

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["ref", "cfg"])
@pytest.mark.parametrize("rows,n,k", [(16, 40, 256), (100, 40, 256), (700, 130, 128), (4096, 1030, 128), (2100, 4100, 128)])
def test_planes_sum_to_t(fmt, rows, n, k):
    import torch

    lib, P, rmax, adapters = D.lib(), D.ptr, 8, 37
    torch.manual_seed(rows)
    w = torch.zeros(n, k, dtype=torch.int8, device="cuda")
    s = torch.ones((n, k // 128) if fmt == "ref" else (n,), dtype=torch.float16 if fmt == "ref" else torch.bfloat16, device="cuda")
    x = torch.zeros(rows, k, dtype=torch.bfloat16, device="cuda")
    la = torch.zeros(adapters, rmax, k, dtype=torch.bfloat16, device="cuda")
    lb = torch.zeros(adapters, n, rmax, dtype=torch.bfloat16, device="cuda")
    x[:, 5] = torch.randn(rows, device="cuda").to(torch.bfloat16)
    la[:, 0, 5] = torch.randn(adapters, device="cuda").to(torch.bfloat16)
    lb[:, :, 0] = 1
    ids = torch.randint(0, adapters, (rows,), device="cuda").to(torch.int32).sort().values.contiguous()
    rank, scale = torch.ones(adapters, dtype=torch.int32, device="cuda"), torch.rand(adapters, device="cuda") + 0.5
    ws = torch.empty(lib.dr_gemm_q8_lora_ws(rows, n, k, rmax), dtype=torch.uint8, device="cuda")
    y = torch.empty(rows, n, device="cuda")
    f = lib.dr_gemm_q8_lora if fmt == "ref" else lib.dr_gemm_q8_lora_bf16s
    f(P(w), P(s), P(x), k, P(ids), P(la), P(lb), P(rank), P(scale), adapters, rmax, P(ws), None, P(y), n, rows, n, k, D.stream_ptr())
    torch.cuda.synchronize()
    i = ids.long()
    want = (scale[i].double() * (la[i, 0, 5].double() * x[:, 5].double())).float()  # one rounding, of a product of 40 bits
    np.testing.assert_array_equal(y.cpu().numpy(), want[:, None].expand(rows, n).cpu().numpy())
