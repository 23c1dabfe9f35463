"""Refusals of the slot-map entries: status codes of the C entries and errors of the
operators, without a GPU (no kernel runs)."""
import ctypes as C

import pytest
import torch

from deepseek_v4_kernel import _native as N
from deepseek_v4_kernel import ops


def slot_args(**kw):
    buf = (C.c_char * 4096)()
    p = (C.addressof(buf) + 15) & ~15
    a = N.SlotMapArgs()
    a.b, a.max_pages, a.page_block_size, a.n_slots, a.n_free, a.stride_table = 2, 4, 64, 8, 3, 4
    for f in ("block_table", "cached_lens", "new_lens", "free_pages", "slots", "positions", "cu_new",
              "cu_total", "n_taken"):
        setattr(a, f, p)
    for k, v in kw.items():
        setattr(a, k, v)
    a._keep = buf
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(cu_new=None), 1), (dict(cu_total=None), 1), (dict(n_taken=None), 1), (dict(block_table=None), 1),
    (dict(cached_lens=None), 1), (dict(new_lens=None), 1), (dict(free_pages=None), 1), (dict(slots=None), 1),
    (dict(positions=None), 1), (dict(b=-1), 2), (dict(b=16385), 2), (dict(max_pages=-1), 2),
    (dict(page_block_size=0), 2), (dict(n_slots=-1), 2), (dict(n_free=-1), 2), (dict(stride_table=3), 3)])
def test_slot_map_entry_refuses(kw, code):
    a = slot_args(**kw)
    assert N.lib.dsv4_build_slot_maps(C.byref(a), None) == code


def test_slot_map_entry_refuses_no_arguments():
    assert N.lib.dsv4_build_slot_maps(None, None) == 1
    assert N.lib.dsv4_page_indices(None, None) == 1


@pytest.mark.parametrize("kw,code", [
    (dict(n_rows=-1), 2), (dict(topk=-1), 2), (dict(b=-1), 2), (dict(max_pages=-1), 2), (dict(page_block_size=0), 2),
    (dict(s_q=0), 2), (dict(stride_positions=-1), 2), (dict(stride_table=-1), 2), (dict(positions=None), 1),
    (dict(indices=None), 1), (dict(block_table=None), 1), (dict(n_rows=0), 0), (dict(topk=0), 0)])
def test_page_indices_entry_refuses(kw, code):
    buf = (C.c_char * 64)()
    a = N.PageIndicesArgs()
    a.n_rows, a.topk, a.b, a.s_q, a.max_pages, a.page_block_size = 2, 4, 2, 1, 4, 64
    a.stride_table = a.stride_positions = 4
    a.block_table = a.positions = a.indices = C.addressof(buf)
    for k, v in kw.items():
        setattr(a, k, v)
    assert N.lib.dsv4_page_indices(C.byref(a), None) == code


def test_operators_refuse_host_tensors():
    t = torch.zeros(2, 4, dtype=torch.int32)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.build_slot_maps(t, n, n, n, 64, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.page_indices(t, torch.zeros(2, 1, 4, dtype=torch.int32), 64)


def test_struct_layouts():
    assert C.sizeof(N.SlotMapArgs) == 6 * 4 + 9 * 8 + 8
    assert C.sizeof(N.PageIndicesArgs) == 6 * 4 + 4 * 8 + 2 * 8
