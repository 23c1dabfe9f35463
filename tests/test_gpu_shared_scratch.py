"""The C entry of the shared-prefix decode keeps to the scratch that it was told to need."""
import ctypes as C

import pytest
import torch

from deepseek_v4_kernel import _native as N
from test_gpu_shared_prefix import Batch

pytestmark = pytest.mark.gpu
GUARD = 1 << 16


def guarded(nbytes):
    buf = torch.full((nbytes + 2 * GUARD,), 0xa5, dtype=torch.uint8, device="cuda")
    return buf, buf.data_ptr() + GUARD


def untouched(buf):
    return bool((buf[:GUARD] == 0xa5).all()) and bool((buf[-GUARD:] == 0xa5).all())


@pytest.mark.parametrize("num_sms", [2, 20, 148, 400])
@pytest.mark.parametrize("b,s_q,h_q,prefix,more,flags,splits", [
    (5, 1, 16, 700, 0, 0, (0, 0)), (12, 1, 64, 6000, 0, N.FLAG_SHARED_DENSE, (0, 0)), (12, 1, 64, 6000, 600, N.FLAG_SHARED_DENSE, (0, 0)),
    (3, 2, 64, 2000, 0, N.FLAG_SHARED_JOINED, (0, 0)), (2, 1, 20, 9000, 0, N.FLAG_SHARED_LISTS, (0, 0)), (2, 1, 20, 900, 0, 0, (7, 3)),
    (1, 1, 16, 5000, 0, N.FLAG_SHARED_DENSE, (0, 0))])
def test_scratch_is_enough(b, s_q, h_q, prefix, more, flags, splits, num_sms):
    x = Batch("V32", b, s_q, h_q, prefix, [(91 * r) % 500 for r in range(b)], 64, seed=1)
    if more:
        x.table = torch.cat([x.table, torch.full((b, more), -1, dtype=torch.int32, device="cuda")], 1)
    a = N.SharedPrefixArgs()
    a.b, a.s_q, a.h_q, a.d_qk, a.d_v, a.kv_format = b, s_q, h_q, 576, 512, N.KV_V32
    a.num_blocks, a.page_block_size = x.kv.size(0), 64
    a.prefix_pages, a.max_pages, a.sm_scale = x.prefix_table.numel(), x.table.size(1), x.scale
    a.flags, a.prefix_splits, a.suffix_splits = flags, *splits
    sets, nbytes = C.c_int32(0), C.c_int64(0)
    assert N.lib.dsv4_shared_prefix_scratch(C.byref(a), num_sms, C.byref(sets), C.byref(nbytes)) == 0
    rows = b * s_q * h_q
    (o, a.o_accum), (e, a.lse_accum), (w, a.workspace) = (guarded(n) for n in (sets.value * rows * 2048, sets.value * rows * 4, nbytes.value))
    (o2, a.out), (e2, a.lse) = guarded(rows * 1024), guarded(rows * 4)
    a.q, a.kv = x.q.data_ptr(), x.kv.data_ptr()
    a.prefix_table, a.prefix_length = x.prefix_table.data_ptr(), x.prefix_length.data_ptr()
    a.block_table, a.suffix_length, a.stride_table = x.table.data_ptr(), x.suffix_length.data_ptr(), x.table.stride(0)
    a.stride_kv_block = x.kv.stride(0)
    a.stride_o_b, a.stride_o_s, a.stride_o_h = s_q * h_q * 512, h_q * 512, 512
    a.stride_lse_b, a.stride_lse_h, a.stride_lse_s = h_q * s_q, s_q, 1
    assert N.lib.dsv4_shared_prefix_decode(C.byref(a), torch.cuda.current_stream().cuda_stream) == 0
    out = o2[GUARD:-GUARD].view(torch.bfloat16).view(b, s_q, h_q, 512)
    lse = e2[GUARD:-GUARD].view(torch.float32).view(b, h_q, s_q)
    x.check((out, lse))
    assert all(untouched(t) for t in (o, e, w, o2, e2))
