"""Weights far below a row's largest one count in dense prefill: one key with a score well above
very many equal ones, whose values alone are not zero.

Bounds.  With u = eps / 2 of the type, a weight and the output are rounded by u of themselves.  FP16
weights are held 2^7 times as large as the row's reference has it, so that the smallest step, 2^-24,
is 2^-31 of the reference's weight, which no row's largest is below: rounding moves a weight by half
of that at most, and the output by 2^-32 for each of n keys.  The scores are exact here; the
exponential and the 32-bit sums are covered by 3e-4 as elsewhere."""
import math

import pytest
import torch

from deepseek_v4_kernel import cuda as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d_qk,d_v", [(64, 64), (128, 128), (192, 128)])
@pytest.mark.parametrize("first", [True, False])
@pytest.mark.parametrize("n_splits", [None, 1, 5])
@pytest.mark.parametrize("above", [0.0, 10.0, 14.0, 17.0, 18.0, 20.0])
def test_one_large_score_among_many(above, n_splits, first, d_qk, d_v, dtype):
    n, rows = 120000, 3
    q = torch.zeros(rows, 2, d_qk, dtype=dtype, device="cuda")
    k, v = torch.zeros(n, 1, d_qk, dtype=dtype, device="cuda"), torch.ones(n, 1, d_v, dtype=dtype, device="cuda")
    at = 0 if first else n - rows
    q[..., 3], k[at, 0, 3], v[at] = above, 1.0, 0.0
    cq, ck = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (rows, n))
    out, ml, lse = K.dense_prefill_fwd(q, k, v, cq, ck, 1.0, n_splits=n_splits)
    torch.cuda.synchronize()
    assert K.device_status() == 0
    u = torch.finfo(dtype).eps / 2
    for i in range(rows):
        seen = n - rows + i + 1                            # keys of this row, the large one among them
        rest = (seen - 1) * math.exp(-above)
        want = rest / (1.0 + rest)
        step = seen * 2.0 ** -32 / (1.0 + rest) if dtype == torch.float16 else 0.0
        assert float((out[i].double() - want).abs().max()) <= (2 * u + 3e-4) * want + step
        assert float((lse[i].double() - (above + math.log1p(rest))).abs().max()) <= 3e-4
    assert (ml == above).all()
