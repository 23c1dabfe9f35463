"""The serving operators as one chain: pages and slots from request lengths, the cache write,
the prompts' attention, then decode steps behind the shared prompt."""
import pytest
import torch

from deepseek_v4_kernel import cuda as K
from deepseek_v4_kernel import ops

pytestmark = pytest.mark.gpu


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def test_prompt_then_decode_steps():
    gen = torch.Generator(device="cuda").manual_seed(0)
    page, h_q, b, prefix = 64, 16, 3, 333
    kv = torch.full((40, page, 1, 644), 0x7f, dtype=torch.uint8, device="cuda")
    free = torch.randperm(40, device="cuda", generator=gen).int()
    scale = 576 ** -0.5

    # the shared prompt is request 0 of its own table
    shared = torch.full((1, 8), -1, dtype=torch.int32, device="cuda")
    slots, pos, cu_q, cu_k, taken = ops.build_slot_maps(shared, ints([0]), ints([prefix]), free, page, 384)
    rows = torch.randn(384, 576, device="cuda", generator=gen).bfloat16()
    ops.kv_store_rows(rows, slots, kv)
    assert cu_q.tolist() == cu_k.tolist() == [0, prefix] and int(taken) == 6
    assert pos[:prefix].tolist() == list(range(prefix)) and (pos[prefix:] == -1).all()

    # its attention with the heads' keys and values written out; a chunk equals the whole
    q = torch.randn(prefix, 4, 192, device="cuda", generator=gen).bfloat16()
    k = torch.randn(prefix, 4, 192, device="cuda", generator=gen).bfloat16()
    v = torch.randn(prefix, 4, 128, device="cuda", generator=gen).bfloat16()
    whole = ops.dense_prefill_fwd(q, k, v, cu_q, cu_k, 192 ** -0.5)
    chunk = ops.dense_prefill_fwd(q[200:], k, v, ints([0, prefix - 200]), cu_k, 192 ** -0.5)
    # the weights' rounding may meet another reference: one step of the result each
    assert ((whole[0][200:].double() - chunk[0].double()).abs() <= 2.0 ** -6 * (1 + chunk[0].double().abs())).all()

    # decode steps of three requests behind it
    free = free[int(taken):].contiguous()
    table = torch.full((b, 4), -1, dtype=torch.int32, device="cuda")
    lens, stored = ints([0, 0, 0]), {r: [] for r in range(b)}
    for step in range(70):
        new = ints([1, 1 if step % 2 else 0, 1 if step > 66 else 0])
        slots, pos, _, cu, taken = ops.build_slot_maps(table, lens, new, free, page, 4)
        rows = torch.randn(4, 576, device="cuda", generator=gen).bfloat16()
        ops.kv_store_rows(rows, slots, kv)
        free = free[int(taken):].contiguous()
        lens = lens + new
        if step not in (0, 63, 64, 69):
            continue
        q = torch.randn(b, 1, h_q, 576, device="cuda", generator=gen).bfloat16()
        out, lse = ops.shared_prefix_decode_fwd(q, kv, shared[0, :6].contiguous(), ints([prefix]), table, lens, None, 512, scale)
        # the same through one list of logical positions per request
        both = torch.cat([shared[:, :5].expand(b, 5), shared[:, 5:6].expand(b, 1), table], 1).contiguous()
        positions = torch.full((b, 1, 10 * page), -1, dtype=torch.int32, device="cuda")
        total = []
        for r, n in enumerate(lens.tolist()):
            positions[r, 0, :prefix] = torch.arange(prefix, device="cuda")
            positions[r, 0, prefix:prefix + n] = 6 * page + torch.arange(n, device="cuda")
            total.append(prefix + n)
        want = ops.sparse_decode_fwd(q, kv, ops.page_indices(both, positions, page), ints(total), None, None, None,
                                     None, None, None, 512, scale)
        torch.cuda.synchronize()
        assert K.device_status() == 0
        # both round their weights and results to BF16: two half steps each of sums of |v| of about one
        assert ((out.double() - want[0].double()).abs() <= 4 * 2.0 ** -8 * (1 + want[0].double().abs())).all()
        assert ((lse - want[1]).abs() <= 1e-3).all()
