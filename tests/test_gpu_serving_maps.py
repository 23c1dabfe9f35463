"""Block tables and slot maps on the GPU against plain Python integers (exact equality)."""
import random

import pytest
import torch

from deepseek_v4_kernel import ops

pytestmark = pytest.mark.gpu
I32_MAX = 2 ** 31 - 1


def plain_maps(table, cached, new, free, page, n_slots):
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    slots, positions, cu_new, cu_total, taken = [], [], [0], [0], 0
    for r, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        old = min(-(-c // page), width)
        for j in range(old, min(-(-(c + n) // page), width)):
            table[r][j] = free[taken] if taken < len(free) else -1
            taken += 1
        for p in range(c, c + n):
            if len(slots) == n_slots:
                break
            ident = table[r][p // page] if p // page < width else -1
            slots.append(ident * page + p % page if ident >= 0 else -1)
            positions.append(min(p, I32_MAX))
        cu_new.append(min(cu_new[-1] + n, I32_MAX))
        cu_total.append(min(cu_total[-1] + c + n, I32_MAX))
    pad = n_slots - len(slots)
    return table, slots + [-1] * pad, positions + [-1] * pad, cu_new, cu_total, [taken]


def ints(v, shape=None):
    t = torch.tensor(v, dtype=torch.int32, device="cuda")
    return t if shape is None else t.view(shape)


def check_maps(table, cached, new, free, page, n_slots, dev_table=None):
    want = plain_maps(table, cached, new, free, page, n_slots)
    width = len(table[0]) if table else 0
    dt = ints(table, (len(table), width)) if dev_table is None else dev_table
    got = ops.build_slot_maps(dt, ints(cached), ints(new), ints(free), page, n_slots)
    assert dt.tolist() == want[0]
    assert got[0].dtype == torch.int64 and all(t.dtype == torch.int32 for t in got[1:])
    for g, w in zip(got, want[1:]):
        assert g.tolist() == w


@pytest.mark.parametrize("page", [1, 16, 48, 64])
@pytest.mark.parametrize("b", [1, 2, 63, 700])
def test_slot_maps_random(b, page):
    rng = random.Random(100 * b + page)
    cached = [rng.choice([0, 0, 1, page - 1, page, page + 1, rng.randrange(300)]) for _ in range(b)]
    new = [rng.choice([0, 1, 1, page, rng.randrange(200)]) for _ in range(b)]
    width = max(-(-(c + n) // page) for c, n in zip(cached, new)) + 2
    ids = list(range(b * width + 9))
    rng.shuffle(ids)
    table = [[ids.pop() if j < -(-c // page) else -7 for j in range(width)] for c in cached]
    for n_slots in {sum(new), sum(new) + 65, max(sum(new) - 3, 0)}:
        check_maps(table, cached, new, ids, page, n_slots)


def test_slot_maps_edges():
    check_maps([[-1, -1]], [0], [0], [], 64, 0)                        # nothing at all
    check_maps([[-1, -1]], [0], [0], [5], 64, 7)                       # only padding
    check_maps([[4, -1, -1]], [64], [65], [9, 8], 64, 65)              # starts on a page border
    check_maps([[4, -1, -1]], [63], [2], [9, 8], 64, 2)                # crosses one
    check_maps([[-1] * 3, [-1] * 3], [0, 0], [130, 70], [1, 2, 3], 64, 200)   # free list too short
    check_maps([[3, -1]], [10], [300], [1, 2, 3, 4], 64, 300)          # table too narrow
    check_maps([[-1, -1]], [10], [5], [1], 64, 5)                      # cached page without an id
    check_maps([[-1, -1]], [-3], [-9], [1], 64, 4)                     # negative lengths
    check_maps([[-1], [-1]], [0, 0], [3, 2], [-1, 6], 4, 5)            # negative id in the free list
    check_maps([[], []], [0, 3], [1, 2], [1], 4, 3)                    # no table columns
    check_maps([[-1], [-1]], [I32_MAX, I32_MAX], [0, 0], [1], 64, 2)   # sums saturate
    check_maps([[2, -1]], [I32_MAX], [I32_MAX], [1], 64, 2)
    assert [t.numel() for t in ops.build_slot_maps(ints([], (0, 4)), ints([]), ints([]), ints([1]), 64, 3)] == [3, 3, 1, 1, 1]


def test_slot_maps_many_requests():
    b = 16384
    rng = random.Random(0)
    cached, new = [rng.randrange(40) for _ in range(b)], [rng.choice([0, 1, 1, 17]) for _ in range(b)]
    table = [[r * 4 + j if j < -(-c // 16) else -1 for j in range(4)] for r, c in enumerate(cached)]
    check_maps(table, cached, new, list(range(b * 4, b * 8)), 16, sum(new) + 1)
    with pytest.raises(RuntimeError, match="16384"):
        ops.build_slot_maps(ints([[0]] * (b + 1)), ints([0] * (b + 1)), ints([0] * (b + 1)), ints([1]), 16, 1)


def test_slot_maps_strided_table_keeps_its_surroundings():
    big = torch.full((5, 40), -9, dtype=torch.int32, device="cuda")
    check_maps([[-9] * 6] * 5, [0] * 5, [70, 1, 0, 64, 65], list(range(20)), 16, 200, dev_table=big[:, 7:13])
    assert (big[:, :7] == -9).all() and (big[:, 13:] == -9).all()


def test_slot_maps_on_a_stream_and_in_a_graph():
    table = torch.full((3, 8), -1, dtype=torch.int32, device="cuda")
    cached, new, free = ints([0, 16, 5]), ints([1, 1, 1]), ints(list(range(50, 80)))
    table[1, 0], table[2, 0] = 7, 8
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.build_slot_maps(table.clone(), cached, new, free, 16, 3)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.build_slot_maps(table, cached, new, free, 16, 3)
    for c, n in (([0, 16, 5], [1, 1, 1]), ([1, 17, 6], [1, 1, 1]), ([0, 0, 0], [2, 0, 1])):
        before = table.tolist()
        cached.copy_(ints(c))
        new.copy_(ints(n))
        g.replay()
        torch.cuda.synchronize()
        want = plain_maps(before, c, n, free.tolist(), 16, 3)
        assert table.tolist() == want[0]
        assert [t.tolist() for t in out] == list(want[1:])


@pytest.mark.parametrize("page", [1, 48, 64, 256, 1000])
@pytest.mark.parametrize("shape", [(3, 1, 128), (2, 3, 63), (5, 2, 1), (1, 1, 2048), (4, 1, 2050)])
def test_page_indices_per_request(shape, page):
    b, s_q, topk = shape
    gen = torch.Generator().manual_seed(page)
    width = 9000 // page + 1
    table = torch.randint(-1, 900, (b, width), generator=gen).int()
    pos = torch.randint(-2, width * page + 70, shape, generator=gen).int()
    want = plain_indices(table, pos.view(b * s_q, topk), [r for r in range(b) for _ in range(s_q)], page)
    got = ops.page_indices(table.cuda(), pos.cuda(), page)
    assert got.dtype == torch.int32 and got.shape == pos.shape
    assert got.view(b * s_q, topk).tolist() == want


def plain_indices(table, pos, reqs, page):
    rows = []
    for r, row in zip(reqs, pos.tolist()):
        t = table[r].tolist() if r is not None else []
        one = []
        for p in row:
            ident = t[p // page] if 0 <= p and p // page < len(t) else -1
            s = ident * page + p % page
            one.append(s if ident >= 0 and s <= I32_MAX else -1)
        rows.append(one)
    return rows


@pytest.mark.parametrize("cu", [[0, 5, 5, 6, 12], [2, 5, 9, 9, 10], [0, 0, 0, 0, 12], [0, 0, 0, 0, 0]])
def test_page_indices_packed(cu):
    gen = torch.Generator().manual_seed(1)
    table, pos = torch.randint(0, 99, (4, 20), generator=gen).int(), torch.randint(-1, 330, (12, 36), generator=gen).int()
    reqs = [next((r for r in range(4) if cu[r] <= i < cu[r + 1]), None) for i in range(12)]
    want = plain_indices(table, pos, reqs, 16)
    assert ops.page_indices(table.cuda(), pos.cuda(), 16, ints(cu)).tolist() == want
    wide = torch.full((12, 50), 3, dtype=torch.int32, device="cuda")     # a column slice of something wider
    wide[:, 5:41] = pos.cuda()
    assert ops.page_indices(table.cuda(), wide[:, 5:41], 16, ints(cu)).tolist() == want


def test_page_indices_of_views():
    gen = torch.Generator().manual_seed(3)
    table, pos = torch.randint(0, 99, (4, 20), generator=gen).int(), torch.randint(-1, 330, (4, 3, 40), generator=gen).int()
    want = torch.tensor(plain_indices(table, pos.view(12, 40), [r for r in range(4) for _ in range(3)], 16)).view(4, 3, 40)
    dev = pos.cuda()
    for s in range(3):                               # one query token of several, and the same with an odd stride of size 1
        assert ops.page_indices(table.cuda(), dev[:, s:s + 1], 16).tolist() == want[:, s:s + 1].tolist()
        one = dev[:, s].contiguous().as_strided((4, 1, 40), (40, 7, 1))
        assert ops.page_indices(table.cuda(), one, 16).tolist() == want[:, s:s + 1].tolist()
    assert ops.page_indices(table.cuda(), dev[:, :, 4:36], 16).tolist() == want[:, :, 4:36].tolist()
    assert ops.page_indices(table.cuda(), dev.transpose(0, 1).contiguous().transpose(0, 1), 16).tolist() == want.tolist()
    assert ops.page_indices(table.cuda(), dev[:1].expand(4, 3, 40), 16).tolist() == \
        torch.tensor(plain_indices(table, pos[:1].expand(4, 3, 40).reshape(12, 40), [r for r in range(4) for _ in range(3)], 16)).view(4, 3, 40).tolist()
    wide = torch.full((4, 30), -5, dtype=torch.int32, device="cuda")
    wide[:, 3:23] = table.cuda()
    assert ops.page_indices(wide[:, 3:23], dev, 16).tolist() == want.tolist()


def test_page_indices_that_do_not_fit():
    table = ints([[I32_MAX, I32_MAX // 64, 33554431, 33554432]])
    pos = ints([[[0, 64, 127, 128, 191, 192, 193, 255, 256, I32_MAX]]])
    assert ops.page_indices(table, pos, 64).view(-1).tolist() == \
        plain_indices(table.cpu(), pos.view(1, -1).cpu(), [0], 64)[0]
    assert ops.page_indices(table, pos[..., :0], 64).shape == (1, 1, 0)


def test_operators_refuse():
    t, n = ints([[0, 1], [2, 3]]), ints([1, 1])
    with pytest.raises(RuntimeError):
        ops.build_slot_maps(t, n.long(), n, n, 64, 2)
    with pytest.raises(RuntimeError):
        ops.build_slot_maps(t, ints([1]), n, n, 64, 2)
    with pytest.raises(RuntimeError):
        ops.build_slot_maps(t, n, n, n, 0, 2)
    with pytest.raises(RuntimeError):
        ops.build_slot_maps(t[:1].expand(2, 2), n, n, n, 64, 2)          # rows share memory
    with pytest.raises(RuntimeError):
        ops.build_slot_maps(t.t(), n, n, n, 64, 2)
    with pytest.raises(RuntimeError):
        ops.page_indices(t, ints([[1, 2]]), 64)                          # packed rows without cu_seqlens
    with pytest.raises(RuntimeError):
        ops.page_indices(t, ints([[1, 2]]), 64, ints([0, 1]))            # b + 1 entries wanted
    with pytest.raises(RuntimeError):
        ops.page_indices(t, ints([[[1]], [[2]]]).long(), 64)
    with pytest.raises(RuntimeError):
        ops.page_indices(t, ints([[[1]], [[2]]]), 0)
