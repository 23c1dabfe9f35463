"""Sizes that do not fit the kernels' 32-bit counters are refused, by the C entries and, before they
are cut to 32 bits, by the operators (on tensors that have no memory)."""
import ctypes as C

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from deepseek_v4_kernel import _native as N
from deepseek_v4_kernel import ops
from test_dense_prefill_cpu import dense_args
from test_shared_prefix_cpu import shared_args

TOP = 2 ** 31 - 1


@pytest.mark.parametrize("kw", [dict(t_q=TOP), dict(t_k=TOP), dict(t_k=2 ** 31 - 100)])
def test_dense_prefill_entry(kw):
    assert N.lib.dsv4_dense_prefill(C.byref(dense_args(**kw)), None) == 2


@pytest.mark.parametrize("kw", [dict(prefix_pages=(1 << 25) - 5, max_pages=4), dict(prefix_pages=1, max_pages=(1 << 25) - 2),
                                dict(num_blocks=(1 << 25) - 1), dict(b=1, s_q=1, h_q=65536), dict(b=512, s_q=2, h_q=128, flags=N.FLAG_IMPL_SIMPLE)])
def test_shared_prefix_entries(kw):
    a = shared_args(**kw)
    sets, nbytes = C.c_int32(0), C.c_int64(0)
    assert N.lib.dsv4_shared_prefix_scratch(C.byref(a), 148, C.byref(sets), C.byref(nbytes)) == 2
    assert N.lib.dsv4_shared_prefix_decode(C.byref(a), None) == 2


@pytest.mark.parametrize("kw", [dict(n_rows=TOP), dict(n_rows=2 ** 31 - 200), dict(topk=TOP)])
def test_page_indices_entry(kw):
    buf = (C.c_char * 64)()
    a = N.PageIndicesArgs()
    a.n_rows, a.topk, a.b, a.s_q, a.max_pages, a.page_block_size = 2, 4, 2, 1, 4, 64
    a.stride_table = a.stride_positions = 4
    a.block_table = a.positions = a.indices = C.addressof(buf)
    for k, v in kw.items():
        setattr(a, k, v)
    assert N.lib.dsv4_page_indices(C.byref(a), None) == 2


def ints(*shape):
    return torch.empty(*shape, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("call", [
    lambda: ops.build_slot_maps(ints(2, 4), ints(2), ints(2), ints(2 ** 32 + 1), 64, 8),
    lambda: ops.build_slot_maps(ints(1, 2 ** 32 + 4), ints(1), ints(1), ints(8), 64, 8),
    lambda: ops.page_indices(ints(1, 4), ints(1, 2 ** 32 + 1, 1), 64),
    lambda: ops.page_indices(ints(1, 4), ints(1, 1, 2 ** 32 + 4), 64),
    lambda: ops.page_indices(ints(1, 2 ** 32 + 4), ints(1, 1, 4), 64),
    lambda: ops.page_indices(ints(2, 4), ints(2 ** 32 + 3, 1), 64, ints(3)),
    lambda: ops.dense_prefill_fwd(*(torch.empty(n, 1, 64, dtype=torch.bfloat16, device="cuda") for n in (3, 2 ** 32 + 1, 2 ** 32 + 1)),
                                  ints(2), ints(2), 0.1),
    lambda: ops.shared_prefix_decode_fwd(torch.empty(1, 1, 16, 576, dtype=torch.bfloat16, device="cuda"),
                                         torch.empty(4, 64, 1, 644, dtype=torch.uint8, device="cuda"), ints(2 ** 32 + 1), ints(1),
                                         ints(1, 4), ints(1), None, 512, 0.04)])
def test_operators(call):
    with FakeTensorMode():
        with pytest.raises(RuntimeError, match="2\\^31"):
            call()
