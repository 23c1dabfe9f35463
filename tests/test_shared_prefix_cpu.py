"""Refusals of the shared-prefix entry and its scratch sizes, without a GPU (no kernel runs)."""
import ctypes as C

import pytest
import torch

from deepseek_v4_kernel import _native as N
from deepseek_v4_kernel import ops


def shared_args(**kw):
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 15) & ~15
    a = N.SharedPrefixArgs()
    a.b, a.s_q, a.h_q, a.d_qk, a.d_v, a.kv_format = 3, 2, 16, 576, 512, N.KV_V32
    a.num_blocks, a.page_block_size, a.prefix_pages, a.max_pages = 40, 64, 20, 4
    a.sm_scale, a.stride_kv_block, a.stride_table = 0.04, 64 * 644, 4
    for f in ("q", "kv", "prefix_table", "prefix_length", "block_table", "suffix_length", "out", "lse", "o_accum",
              "lse_accum", "workspace"):
        setattr(a, f, p)
    a.stride_o_b, a.stride_o_s, a.stride_o_h = 2 * 16 * 512, 16 * 512, 512
    a.stride_lse_b, a.stride_lse_h, a.stride_lse_s = 32, 2, 1
    for k, v in kw.items():
        setattr(a, k, p + v if k in ("q", "kv", "out") and v else v)
    a._keep = buf
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(q=None), 1), (dict(kv=None), 1), (dict(out=None), 1), (dict(lse=None), 1), (dict(prefix_table=None), 1),
    (dict(prefix_length=None), 1), (dict(block_table=None), 1), (dict(suffix_length=None), 1), (dict(b=-1), 2),
    (dict(s_q=0), 2), (dict(h_q=0), 2), (dict(d_v=256), 2), (dict(num_blocks=0), 2), (dict(page_block_size=0), 2),
    (dict(prefix_pages=-1), 2), (dict(max_pages=-1), 2), (dict(prefix_splits=-1), 2), (dict(suffix_splits=65), 2),
    (dict(num_blocks=1 << 26), 2), (dict(prefix_pages=1 << 26), 2), (dict(max_pages=1 << 26), 2),
    (dict(b=1 << 20, s_q=1 << 12), 2), (dict(b=1 << 20), 2), (dict(stride_table=-1), 2), (dict(sm_scale=0.0), 2), (dict(sm_scale=-1.0), 2), (dict(sm_scale=float("nan")), 2),
    (dict(sm_scale=float("inf")), 2), (dict(prefix_pages=(1 << 25) - 1, max_pages=9), 2), (dict(d_qk=512), 3),
    (dict(kv_format=N.KV_MODEL1), 3), (dict(kv_format=N.KV_BF16), 3), (dict(stride_kv_block=64 * 644 - 16), 3),
    (dict(stride_kv_block=64 * 644 + 8), 4), (dict(kv=8), 4), (dict(q=2), 4), (dict(out=8), 4), (dict(stride_o_h=516), 4)])
def test_entry_refuses(kw, code):
    assert N.lib.dsv4_shared_prefix_decode(C.byref(shared_args(**kw)), None) == code


def test_entry_refuses_no_arguments_and_the_layout_of_the_block():
    assert N.lib.dsv4_shared_prefix_decode(None, None) == 1
    assert N.lib.dsv4_shared_prefix_scratch(None, 148, None, None) == 1
    assert C.sizeof(N.SharedPrefixArgs) == 14 * 4 + 12 * 8 + 8 * 8


def scratch(**kw):
    sets, nbytes = C.c_int32(-1), C.c_int64(-1)
    rc = N.lib.dsv4_shared_prefix_scratch(C.byref(shared_args(**kw)), 148, C.byref(sets), C.byref(nbytes))
    assert rc == 0
    return sets.value, nbytes.value


def test_scratch_follows_the_parts_that_exist():
    assert scratch(prefix_pages=0, max_pages=0) == (0, 0)
    assert scratch(prefix_splits=3, suffix_splits=2)[0] == 5
    assert scratch(prefix_pages=0, suffix_splits=2)[0] == 2
    assert scratch(max_pages=0, prefix_splits=3)[0] == 3
    sets, nbytes = scratch()
    assert 2 <= sets <= 256 and nbytes > 0 and scratch() == (sets, nbytes)
    with pytest.raises(AssertionError):
        scratch(s_q=0)


def test_operator_refuses_host_tensors():
    t, n = torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q, kv = torch.zeros(2, 1, 16, 576, dtype=torch.bfloat16), torch.zeros(4, 64, 1, 644, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.shared_prefix_decode_fwd(q, kv, n, n[:1], t, n, None, 512, 0.04)


@pytest.mark.parametrize("kw", [{}, dict(b=64, h_q=64, prefix_pages=512, max_pages=32), dict(b=16, h_q=64, prefix_pages=512, max_pages=1000),
                                dict(b=1, s_q=1, prefix_pages=1100), dict(flags=N.FLAG_SHARED_JOINED), dict(flags=N.FLAG_SHARED_LISTS),
                                dict(prefix_pages=0), dict(max_pages=0)])
def test_scratch_is_what_the_call_uses_whatever_number_of_sms_is_named(kw):
    """The call cannot know which number its scratch was sized with."""
    def sized(num_sms):
        sets, nbytes = C.c_int32(-1), C.c_int64(-1)
        assert N.lib.dsv4_shared_prefix_scratch(C.byref(shared_args(**kw)), num_sms, C.byref(sets), C.byref(nbytes)) == 0
        return sets.value, nbytes.value
    assert len({sized(n) for n in (2, 3, 20, 74, 132, 148, 160, 1000)}) == 1


@pytest.mark.parametrize("kw", [{}, dict(prefix_pages=100), dict(prefix_pages=5000), dict(max_pages=500), dict(flags=N.FLAG_SHARED_DENSE),
                                dict(flags=N.FLAG_SHARED_LISTS), dict(prefix_splits=3)])
def test_a_batch_of_no_request_needs_no_scratch(kw):
    assert scratch(b=0, **kw) == (0, 0)
    assert N.lib.dsv4_shared_prefix_decode(C.byref(shared_args(b=0, **kw)), None) in (0, 5, 6)      # (5, 6: no such device here)


@pytest.mark.parametrize("kw,per_token", [({}, 1152), (dict(d_qk=512, kv_format=N.KV_MODEL1, stride_kv_block=64 * 584), 1024)])
def test_workspace_is_bounded_however_wide_the_table(kw, per_token):
    batch = dict(b=64, s_q=1, h_q=64, num_blocks=1 << 16, max_pages=4, **kw)
    most = (4 << 30) // (per_token * 64)                                    # pages whose tokens fill 4 GiB
    for pages in (512, most // 2, most - 1000):
        assert scratch(prefix_pages=pages, **batch)[1] >= pages * 64 * per_token
    for pages in (most + 1, 1 << 17, 1 << 20, (1 << 25) - 2000):
        assert scratch(prefix_pages=pages, **batch)[1] <= pages * 64 * 4 + (1 << 20)
