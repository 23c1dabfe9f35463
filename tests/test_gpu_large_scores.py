"""Scores of ten thousands and more: in every form, and for every way of cutting the tokens, the
softmax is that of the 64-bit definition.

Scores are built to be exact in 32 bits (multiples of 1/2 below 2^18) and to lie between BF16 numbers,
whose steps are 256 to 1024 there.  Bounds: inside a part the weights have the exponential's error
alone; a log-sum-exp e carries four roundings of 2^-24 |e| (reference times ln 2, the two constants,
the sum), so that the weights of two parts may differ by 8 * 2^-24 |e|."""
import pytest
import torch

from deepseek_v4_kernel import _native as N
from deepseek_v4_kernel import cuda as K
from deepseek_v4_kernel import ops
from test_gpu_not_finite import WAYS
from test_gpu_shared_prefix import SCORES, U, Batch

pytestmark = pytest.mark.gpu


def large(layout, b, h_q, prefix, suffix, seed, base=6144.0):
    """Scores base * 16 + 15 * (1 to 70) + (0 to 4) of both signs, and a head of ordinary ones."""
    x = Batch(layout, b, 1, h_q, prefix, suffix, 64, seed=seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    for table, count in [(x.prefix_table, prefix)] + [(x.table[r], s) for r, s in enumerate(suffix)]:
        if count:
            tok = torch.arange(count, device="cuda")
            latent = torch.randn(count, x.d, device="cuda", generator=g)
            latent[:, 0], latent[:, 1] = 16.0, 15.0
            latent[:, 2] = torch.randint(0, 9, (count,), device="cuda", generator=g) / 2
            ops.kv_store(latent.bfloat16(), torch.zeros(count, 64, dtype=torch.bfloat16, device="cuda"),
                         table.long()[tok // 64] * 64 + tok % 64, x.kv)
    x.q.zero_()
    h = torch.arange(h_q, device="cuda")
    x.q[..., 0] = torch.where(h % 3 == 0, base, -base)
    x.q[..., 1] = (h % 35) * 2 + 1
    x.q[..., 2] = 1
    x.q[:, :, h_q - 1, :2] = 0
    x.scale = 1.0
    return x


def check(got, want):
    torch.cuda.synchronize()
    assert K.device_status() == 0
    out, mag, lse = want
    e = lse.transpose(1, 2).abs()[..., None]
    bound = U * (mag + out.abs()) + (SCORES + 8 * 2.0 ** -24 * e) * mag
    assert not torch.isnan(got[0]).any()
    assert ((got[0].double() - out).abs() <= bound).all()
    assert ((got[1].double() - lse).abs() <= SCORES + 2e-6 * lse.abs()).all()


@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
@pytest.mark.parametrize("way", WAYS)
@pytest.mark.parametrize("b,h_q,prefix", [(5, 16, 700), (1, 20, 3000), (3, 64, 1300), (2, 128, 200)])
@pytest.mark.parametrize("base", [1024.0, 2048.0, 6144.0, 15872.0])
def test_shared_prefix(base, b, h_q, prefix, way, layout):
    x = large(layout, b, h_q, prefix, [9, 130, 1, 300, 64][:b], seed=h_q, base=base)
    check(x.call(**WAYS[way]), x.definition())


@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
@pytest.mark.parametrize("simple", [0, N.FLAG_IMPL_SIMPLE])
@pytest.mark.parametrize("n_splits", [1, 2, 3, 4, 7])
@pytest.mark.parametrize("h_q", [16, 32, 64])
def test_sparse_decode(h_q, n_splits, simple, layout):
    x = large(layout, 2, h_q, 900, [1, 1], seed=n_splits)
    idx = ops.page_indices(x.prefix_table[None], torch.arange(900, device="cuda", dtype=torch.int32).view(1, 1, -1), 64)
    got = K.sparse_decode_fwd(x.q, x.kv, idx.expand(2, 1, 900).contiguous(), None, None, None, None, None, None, None, 512,
                              x.scale, n_splits=n_splits, flags=simple)[:2]
    check(got, x.definition(suffix=[0, 0]))


def test_references_that_grow_past_the_border():
    """Scores that rise from tens to 60000 along the list: ordinary references are raised to large ones."""
    x = large("V32", 1, 64, 4000, [1], seed=3)
    tok = torch.arange(4000, device="cuda")
    latent = torch.randn(4000, 512, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    latent[:, 0], latent[:, 1] = (tok // 500 * 2).float(), 15.0
    latent[:, 2] = (tok * 7 % 9) / 2
    latent[:, 3] = 16.0
    x.q[..., 0] = torch.arange(64, device="cuda") * 64.0
    ops.kv_store(latent.bfloat16(), torch.zeros(4000, 64, dtype=torch.bfloat16, device="cuda"),
                 x.prefix_table.long()[tok // 64] * 64 + tok % 64, x.kv)
    idx = ops.page_indices(x.prefix_table[None], tok.int().view(1, 1, -1), 64)
    want = x.definition(suffix=[0])
    for n_splits in (1, 3, 4):
        got = K.sparse_decode_fwd(x.q, x.kv, idx, None, None, None, None, None, None, None, 512, x.scale, n_splits=n_splits)[:2]
        check(got, want)
