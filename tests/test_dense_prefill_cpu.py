"""Refusals of the dense-prefill entry and its split plan, without a GPU (no kernel runs)."""
import ctypes as C

import pytest
import torch

from deepseek_v4_kernel import _native as N
from deepseek_v4_kernel import ops


def dense_args(**kw):
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 15) & ~15
    a = N.DensePrefillArgs()
    a.b, a.t_q, a.t_k, a.h_q, a.h_kv, a.d_qk, a.d_v = 2, 8, 9, 8, 2, 128, 128
    a.n_splits, a.sm_scale = 1, 0.1
    for f in ("q", "k", "v", "cu_seqlens_q", "cu_seqlens_k", "out", "max_logits", "lse"):
        setattr(a, f, p)
    for f in ("stride_q_t", "stride_k_t", "stride_v_t", "stride_o_t"):
        setattr(a, f, 1024)
    for f in ("stride_q_h", "stride_k_h", "stride_v_h", "stride_o_h"):
        setattr(a, f, 128)
    for k, v in kw.items():
        setattr(a, k, p + v if isinstance(v, int) and v and k in ("q", "k", "v", "out", "o_accum") else v)
    a._keep = buf
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(cu_seqlens_q=None), 1), (dict(cu_seqlens_k=None), 1),
    (dict(out=None), 1), (dict(max_logits=None), 1), (dict(lse=None), 1), (dict(b=-1), 2), (dict(t_q=-1), 2),
    (dict(t_k=-1), 2), (dict(h_q=0), 2), (dict(h_kv=0), 2), (dict(h_kv=3), 2), (dict(n_splits=0), 2), (dict(n_splits=65), 2),
    (dict(sm_scale=0.0), 2), (dict(sm_scale=-1.0), 2), (dict(sm_scale=float("nan")), 2), (dict(sm_scale=float("inf")), 2),
    (dict(d_qk=64), 3), (dict(d_v=64), 3), (dict(d_qk=576, d_v=512), 3), (dict(dtype=2), 8), (dict(q=8), 4), (dict(k=2), 4),
    (dict(v=4), 4), (dict(out=8), 4), (dict(stride_q_t=1020), 4), (dict(stride_k_t=0), 4), (dict(stride_k_h=0), 4),
    (dict(stride_v_h=-128), 4), (dict(stride_o_h=4), 4), (dict(stride_v_t=1 << 40), 4), (dict(n_splits=2), 7),
    (dict(b=0), 0), (dict(t_q=0), 0)])
def test_entry_refuses(kw, code):
    assert N.lib.dsv4_dense_prefill(C.byref(dense_args(**kw)), None) == code


def test_entry_refuses_no_arguments_and_the_layout_of_the_block():
    assert N.lib.dsv4_dense_prefill(None, None) == 1
    assert C.sizeof(N.DensePrefillArgs) == 12 * 4 + 11 * 8 + 10 * 8


def test_split_plan():
    plan = N.lib.dsv4_plan_dense_splits
    assert plan(8192, 8192, 1, 16, 16, 148) == 1                 # the rows fill the GPU
    assert 1 < plan(8, 8 * 8192, 8, 32, 8, 148) <= 148 // 8      # 8 chunks of heads
    assert plan(1, 100000, 1, 8, 8, 148) > 8                     # one token over a long context
    assert plan(1, 200, 1, 8, 8, 148) == 1                       # too short to cut
    for bad in ((0, 1, 1, 1, 1, 148), (1, 0, 1, 1, 1, 148), (1, 1, 0, 1, 1, 148), (1, 1, 1, 3, 2, 148), (1, 1, 1, 1, 1, 0)):
        assert plan(*bad) == 1
    for args in ((3, 70000, 3, 64, 1, 148), (5, 1 << 24, 5, 1, 1, 148)):
        assert 1 <= plan(*args) <= 64


def test_operator_refuses_host_tensors():
    q, cu = torch.zeros(2, 4, 128, dtype=torch.bfloat16), torch.tensor([0, 2], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.dense_prefill_fwd(q, q, q, cu, cu, 0.1)
