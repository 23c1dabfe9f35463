"""A token that is not finite shows in the rows that see it, in every form of an operator and
for every way of cutting its tokens: the softmax of a NaN score is NaN by its definition, and a
part with one must not be passed over when the parts are joined."""
import pytest
import torch

from deepseek_v4_kernel import _native as N
from deepseek_v4_kernel import cuda as K
from deepseek_v4_kernel import ops
from test_gpu_shared_prefix import SCORES, U, Batch

pytestmark = pytest.mark.gpu

# how a shared-prefix decode is done: as chosen, each form, forced splits, the cross-check kernel
WAYS = {"chosen": {}, "lists": dict(flags=N.FLAG_SHARED_LISTS), "joined": dict(flags=N.FLAG_SHARED_JOINED),
        "dense": dict(flags=N.FLAG_SHARED_DENSE), "1+1": dict(prefix_splits=1, suffix_splits=1),
        "3+2": dict(prefix_splits=3, suffix_splits=2), "40+5": dict(prefix_splits=40, suffix_splits=5),
        "simple": dict(flags=N.FLAG_IMPL_SIMPLE)}


def spoil(x, page, at, where):
    if where == "latent":                                  # 2^128 times the codes: infinities of both signs
        x.arena[page, 64 * (x.d + 128) + at * x.slots + 1] = 255
    else:                                                  # a rotary value that is NaN
        x.arena[page, at * (x.d + 128) + x.d:][:2] = 0xff


def check(x, got, want, spoilt):
    torch.cuda.synchronize()
    assert K.device_status() == 0
    out, lse = got[0], got[1].transpose(1, 2)
    assert torch.isnan(out[spoilt]).all() and torch.isnan(lse[spoilt]).all()
    fine = ~spoilt
    off = (out.double() - want[0]).abs() / (U * (want[1] + want[0].abs()) + SCORES * want[1] + 1e-30)
    assert not fine.any() or float(off[fine].max()) <= 1
    e = want[2].transpose(1, 2)
    assert ((lse.double() - e).abs()[fine] <= SCORES + 2e-6 * e.abs()[fine]).all()


@pytest.mark.parametrize("where", ["latent", "rope"])
@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("wide", [False, True])
def test_own_tokens(wide, way, layout, where):
    """`wide`: tables of 300 more columns, with which the own tokens are attended in a launch of their own."""
    x = Batch(layout, 7, 2, 16, 700, [40, 0, 129, 1, 300, 64, 2], 64, seed=3)
    want = x.definition()
    if wide:
        x.table = torch.cat([x.table, torch.full((7, 300), 2 ** 30, dtype=torch.int32, device="cuda")], 1)
    spoilt = torch.zeros(7, 2, dtype=torch.bool, device="cuda")
    for r, at in ((0, 39), (2, 127), (4, 299), (6, 0)):
        spoil(x, int(x.table[r, at // 64]), at % 64, where)
        spoilt[r] |= torch.arange(2, device="cuda") >= 1 - (x.suffix[r] - 1 - at)
    check(x, x.call(**WAYS[way]), want, spoilt)


@pytest.mark.parametrize("where", ["latent", "rope"])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("b,h_q,prefix,at", [(5, 16, 700, 699), (1, 16, 3000, 0), (2, 64, 5000, 2300), (9, 20, 130, 64)])
def test_tokens_of_the_prefix(b, h_q, prefix, at, way, where):
    x = Batch("V32", b, 1, h_q, prefix, [0, 9, 130, 1, 64, 2, 3, 0, 5][:b], 64, seed=4, sink=True)
    spoil(x, int(x.prefix_table[at // 64]), at % 64, where)
    check(x, x.call(**WAYS[way]), x.definition(), torch.ones(b, 1, dtype=torch.bool, device="cuda"))


@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("sink", [False, True])
def test_nothing_but_a_token_that_is_not_finite(sink, way):
    """No finite score ever sets a reference."""
    x = Batch("V32", 3, 1, 16, 0, [1, 0, 5], 64, sink=sink)
    want = x.definition()
    spoil(x, int(x.table[0, 0]), 0, "rope")
    got = x.call(**WAYS[way])
    torch.cuda.synchronize()
    assert K.device_status() == 0
    assert torch.isnan(got[0][0]).all() and torch.isnan(got[1][0]).all()
    assert (got[0][1] == 0).all() and torch.equal(got[1][1].double(), want[2][1])
    assert torch.isfinite(got[0][2]).all() and torch.isfinite(got[1][2]).all()


def test_joined_lists_of_many_splits_are_covered():
    """The sizes above reach JOINED calls whose partials are merged in a cluster, and such that are combined."""
    counts = {N.lib.dsv4_plan_splits(*a, 148) for a in ((7, 2, 16, 1088, 0), (1, 1, 16, 3008, 0), (2, 1, 64, 5200, 0),
                                                         (3, 1, 16, 128, 0), (9, 1, 20, 384, 0))}
    assert 1 in counts and any(n > 4 for n in counts)


@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
@pytest.mark.parametrize("simple", [0, N.FLAG_IMPL_SIMPLE])
@pytest.mark.parametrize("n_splits", [1, 2, 3, 4, 7])
@pytest.mark.parametrize("at", [0, 500, 899])
def test_sparse_decode_of_any_number_of_splits(at, n_splits, simple, layout):
    x = Batch(layout, 3, 1, 16, 900, [1, 1, 1], 64, seed=6)
    pos = torch.arange(900, device="cuda", dtype=torch.int32)
    idx = ops.page_indices(x.prefix_table[None], pos.view(1, 1, -1), 64).expand(3, 1, 900).contiguous()
    idx[1, 0, at] = -1                                     # request 1 does not list it
    flags = simple | N.FLAG_MASK_INVALID

    def call():
        return K.sparse_decode_fwd(x.q, x.kv, idx, None, None, None, None, None, None, None, 512, x.scale,
                                   n_splits=n_splits, flags=flags)[:2]
    clean = call()
    spoil(x, int(x.prefix_table[at // 64]), at % 64, "rope")
    out, lse = call()
    torch.cuda.synchronize()
    assert K.device_status() == 0
    for r in (0, 2):
        assert torch.isnan(out[r]).all() and torch.isnan(lse[r]).all()
    assert torch.equal(out[1], clean[0][1]) and torch.equal(lse[1], clean[1][1])


@pytest.mark.parametrize("simple", [0, N.FLAG_IMPL_SIMPLE])
@pytest.mark.parametrize("n_splits", [1, 2, 5])
def test_sparse_decode_of_one_token_that_is_not_finite(n_splits, simple):
    x = Batch("V32", 2, 1, 16, 64, [1, 1], 64, seed=7)
    spoil(x, int(x.prefix_table[0]), 5, "rope")
    idx = torch.full((2, 1, 400), -1, dtype=torch.int32, device="cuda")
    idx[0, 0, 7] = x.prefix_table[0] * 64 + 5
    out, lse, _, _ = K.sparse_decode_fwd(x.q, x.kv, idx, None, None, None, None, None, None, None, 512, x.scale,
                                         n_splits=n_splits, flags=simple | N.FLAG_MASK_INVALID)
    torch.cuda.synchronize()
    assert K.device_status() == 0
    assert torch.isnan(out[0]).all() and torch.isnan(lse[0]).all()
    assert (out[1] == 0).all() and (lse[1] == -float("inf")).all()


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("n_splits", [1, 2, 5, 16])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_values_far_below_the_largest_weight(dtype, n_splits, value):
    """The token with the value that is not finite weighs e^-200 of the last one: still not nothing."""
    n = 4000
    q, k = torch.zeros(1, 2, 128, dtype=dtype, device="cuda"), torch.zeros(n, 1, 128, dtype=dtype, device="cuda")
    v = torch.ones(n, 1, 128, dtype=dtype, device="cuda")
    q[..., 0], k[n - 1, 0, 0], v[37, 0, 5] = 200.0, 1.0, value
    cq, ck = (torch.tensor([0, m], dtype=torch.int32, device="cuda") for m in (1, n))
    out, ml, lse = K.dense_prefill_fwd(q, k, v, cq, ck, 1.0, n_splits=n_splits)
    torch.cuda.synchronize()
    assert K.device_status() == 0
    assert not torch.isfinite(out[..., 5]).any()
    rest = torch.cat([out[..., :5], out[..., 6:]], -1)
    assert ((rest.double() - 1).abs() <= torch.finfo(dtype).eps).all()
    assert (ml == 200).all() and ((lse - 200).abs() <= 1e-3).all()
