"""Calls of the serving operators that their documentation allows and the tests beside them do not
make: outputs whose rows start between sectors, and a first call that is captured."""
import os
import subprocess
import sys

import pytest
import torch

from deepseek_v4_kernel import cuda as K
from test_gpu_dense_prefill import BF16, DIMS, FP16, check, cu_of, definition, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n_splits", [1, 3])
@pytest.mark.parametrize("pad,at", [(8, 0), (8, 8), (24, 8), (16, 8)])
def test_outputs_whose_rows_start_anywhere_on_16_bytes(pad, at, n_splits, dtype, d_qk, d_v):
    lq, lk = [70, 1, 130], [90, 333, 130]
    q, k, v = make(lq, lk, 4, 2, d_qk, d_v, dtype, seed=pad + at)
    hold = torch.full((sum(lq), 4, d_v + pad), 3.0, dtype=dtype, device="cuda")
    out = hold[..., at:at + d_v]
    got = K.dense_prefill_fwd(q, k, v, cu_of(lq), cu_of(lk), 0.1, True, None, out, n_splits=n_splits)
    check(got, definition(q, k, v, lq, lk, 0.1, True, None), dtype)
    keep = torch.ones_like(hold, dtype=torch.bool)
    keep[..., at:at + d_v] = False
    assert (hold[keep] == 3.0).all()


SETUP = """
import torch
from deepseek_v4_kernel import ops
g = torch.Generator(device='cuda').manual_seed(0)
ints = lambda *v: torch.tensor(v, dtype=torch.int32, device='cuda')
q = torch.randn(40, 8, 128, device='cuda', generator=g).bfloat16()
k = torch.randn(3000, 2, 128, device='cuda', generator=g).bfloat16()
kv = torch.zeros(80, 64, 1, 644, dtype=torch.uint8, device='cuda')
row = torch.randn(2, 1, 64, 576, device='cuda', generator=g).bfloat16()
table, pages, prompt, single = ints(5, -1, 6, -1).view(2, 2), torch.arange(80, dtype=torch.int32, device='cuda'), ints(0, 40), ints(0, 1)
lens, pos = ints(3, 64), ints(1, 2, 3, 4).view(2, 1, 2)
n, many, ck = ints(4500), ints(0, 3000), ints(0, 40)
calls = dict(
    slots=lambda: ops.build_slot_maps(table, lens, ints_new, pages, 64, 8),
    indices=lambda: (ops.page_indices(table, pos, 64),),
    prompt=lambda: ops.dense_prefill_fwd(q, k[:40], k[:40], prompt, ck, 0.1),
    single=lambda: ops.dense_prefill_fwd(q[:1], k, k, single, many, 0.1),
    shared=lambda: ops.shared_prefix_decode_fwd(row, kv, pages, n, table, lens, None, 512, 0.04))
ints_new = ints(1, 1)
call = calls[NAME]
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    got = call()
graph.replay()
torch.cuda.synchronize()
want = call()
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(got, want))
print('same')
"""


@pytest.mark.parametrize("name", ["slots", "indices", "prompt", "single", "shared"])
def test_a_first_call_that_is_captured(name):
    env = dict(os.environ, PYTHONPATH=os.pathsep.join(p for p in sys.path if p))
    res = subprocess.run([sys.executable, "-c", f"NAME = {name!r}\n" + SETUP], env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "same" in res.stdout, res.stderr[-2000:]
