"""Decode of a batch behind a shared prefix against the definition in 64 bits.

Bounds.  With u = 2^-8 (half a BF16 step) an output may be off by the rounding of the weights,
u * sum p |v|, and its own, u * |o|; the scores are 32-bit sums of up to 576 products of about
one, scaled by 1/24: at most 577 * 2^-24 * 370 / 24 = 5.3e-4 off, and 8e-4 with the
exponential's error.  The log-sum-exp carries the scores' error alone."""
import math

import pytest
import torch

from deepseek_v4_kernel import _native as N
from deepseek_v4_kernel import cuda as K
from deepseek_v4_kernel import ops

pytestmark = pytest.mark.gpu
SCORES, U = 8e-4, 2.0 ** -8
FORMS = [0, N.FLAG_SHARED_LISTS, N.FLAG_SHARED_JOINED, N.FLAG_SHARED_DENSE]      # as chosen, and each of the three
LAYOUTS = {"V32": (512, 128, 4, 4), "MODEL1": (448, 64, 7, 8)}


class Batch:
    """A cache with a shared prefix and private suffixes on shuffled pages; the bytes of every
    token that no length covers are NaN codes with the largest scale."""

    def __init__(self, layout, b, s_q, h_q, prefix, suffix, page, seed=0, sink=False, pad=0, blocks_before=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        d, tile, n, slots = LAYOUTS[layout]
        self.layout, self.page, self.d, self.n_scale, self.tile, self.slots = layout, page, d, n, tile, slots
        self.prefix, self.suffix = prefix, list(suffix)
        pages = [-(-prefix // page)] + [-(-s // page) for s in suffix]
        blocks = sum(pages) + 3
        stride = -(-page * (d + 128 + slots) // 16) * 16 + pad
        total = blocks + blocks_before
        self.arena = torch.empty(total, stride, dtype=torch.uint8, device="cuda")
        used = self.arena[blocks_before:]
        used.fill_(0x7f)
        used[:, page * (d + 128):] = 0xff
        self.kv = torch.as_strided(self.arena, (total, page, 1, d + 128 + slots),
                                   (stride, d + 128 + slots, d + 128 + slots, 1))
        ids = (torch.randperm(blocks, device="cuda", generator=g) + blocks_before).int()
        self.prefix_table = ids[:pages[0]].contiguous()
        width = max(max(pages[1:], default=0), 1) + 1
        self.table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
        at = pages[0]
        for r, n_pages in enumerate(pages[1:]):
            self.table[r, :n_pages] = ids[at:at + n_pages]
            at += n_pages
        for table, count in [(self.prefix_table, prefix)] + [(self.table[r], s) for r, s in enumerate(suffix)]:
            if count:
                tok = torch.arange(count, device="cuda")
                where = table.long()[tok // page] * page + tok % page
                ops.kv_store(torch.randn(count, d, device="cuda", generator=g).bfloat16(),
                             torch.randn(count, 64, device="cuda", generator=g).bfloat16(), where, self.kv)
        self.prefix_length = torch.tensor([prefix], dtype=torch.int32, device="cuda")
        self.suffix_length = torch.tensor(self.suffix, dtype=torch.int32, device="cuda")
        self.q = torch.randn(b, s_q, h_q, d + 64, device="cuda", generator=g).bfloat16()
        self.sink = torch.randn(h_q, device="cuda", generator=g) if sink else None
        self.scale = (d + 64) ** -0.5

    def rows(self, table, count):
        """The first `count` tokens of a list of pages in 64 bits; None for a page outside the cache."""
        tok = torch.arange(count, device="cuda")
        ids, at = table.long()[tok // self.page], (tok % self.page)[:, None]
        fine = (ids >= 0) & (ids < self.kv.size(0))
        ids, at = ids[fine][:, None], at[fine]
        row = self.d + 128
        code = self.arena[ids, at * row + torch.arange(self.d, device="cuda")].view(torch.float8_e4m3fn).double()
        sc = self.arena[ids, self.page * row + at * self.slots + torch.arange(self.n_scale, device="cuda")].double()
        rope = self.arena[ids, at * row + self.d + torch.arange(128, device="cuda")].view(torch.bfloat16).double()
        return torch.cat([code * torch.exp2(sc - 127).repeat_interleave(self.tile, 1), rope], 1), tok[fine]

    def definition(self, prefix=None, suffix=None):
        prefix = self.prefix if prefix is None else prefix
        suffix = self.suffix if suffix is None else suffix
        b, s_q, h_q, _ = self.q.shape
        out = torch.zeros(b, s_q, h_q, 512, dtype=torch.float64, device="cuda")
        mag, lse = out.clone(), torch.full((b, h_q, s_q), -math.inf, dtype=torch.float64, device="cuda")
        pre, _ = self.rows(self.prefix_table, min(max(prefix, 0), self.prefix_table.numel() * self.page))
        for r in range(b):
            count = min(max(suffix[r], 0), self.table.size(1) * self.page)
            mine, tok = self.rows(self.table[r], count)
            for s in range(s_q):
                kv = torch.cat([pre, mine[tok < count - (s_q - 1 - s)]])
                x = (self.q[r, s].double() @ kv.t()) * self.scale
                e = torch.logsumexp(x, -1) if kv.size(0) else torch.full((h_q,), -math.inf, dtype=torch.float64, device="cuda")
                if self.sink is not None:
                    e = torch.logaddexp(e, self.sink.double())
                if kv.size(0):
                    w = torch.exp(x - e[:, None])
                    out[r, s], mag[r, s] = w @ kv[:, :512], w @ kv[:, :512].abs()
                lse[r, :, s] = e
        return out, mag, lse

    def call(self, **kw):
        return K.shared_prefix_decode_fwd(self.q, self.kv, self.prefix_table, self.prefix_length, self.table,
                                          self.suffix_length, self.sink, 512, self.scale, **kw)

    def check(self, got, want=None):
        out, mag, lse = self.definition() if want is None else want
        torch.cuda.synchronize()
        assert K.device_status() == 0
        off = (got[0].double() - out).abs() / (U * (mag + out.abs()) + SCORES * mag + 1e-30)
        assert not torch.isnan(off).any() and (off.numel() == 0 or float(off.max()) <= 1), f"{float(off.max()):.3g} times the bound"
        fine = torch.isfinite(lse)
        assert torch.equal(got[1][~fine].double(), lse[~fine])
        assert ((got[1].double() - lse).abs()[fine] <= SCORES + 2e-6 * lse.abs()[fine]).all()


@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("b,s_q,h_q", [(1, 1, 1), (4, 1, 16), (3, 2, 20), (5, 1, 64), (2, 3, 128), (17, 1, 8), (9, 1, 48)])
def test_batches(layout, b, s_q, h_q, form):
    suffix = [(37 * r) % 201 for r in range(b)]
    x = Batch(layout, b, s_q, h_q, 1000, suffix, 64, seed=b, sink=b % 2 == 0)
    x.check(x.call(flags=form))


@pytest.mark.parametrize("prefix", [0, 1, 63, 64, 65, 127, 128, 129, 2049])
@pytest.mark.parametrize("page", [16, 48, 64, 256])
@pytest.mark.parametrize("form", FORMS[1:])
def test_prefix_lengths_and_pages(prefix, page, form):
    x = Batch("V32", 6, 1, 32, prefix, [0, 1, 2, 127, 128, 300], page, seed=prefix)
    x.check(x.call(flags=form))


@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
@pytest.mark.parametrize("form", FORMS)
def test_rows_that_see_nothing(layout, form):
    for sink in (False, True):
        x = Batch(layout, 3, 2, 16, 0, [0, 1, 5], 64, sink=sink)
        got = x.call(flags=form)
        x.check(got)
        x.prefix_table = torch.zeros(3, dtype=torch.int32, device="cuda")      # a table, but no token of it
        x.check(x.call(flags=form))
        assert (got[0][0] == 0).all() and (got[0][1, 0] == 0).all()
    x = Batch(layout, 3, 1, 16, 0, [0, 0, 0], 64, sink=True)
    x.table = x.table[:, :0]
    got = x.call(flags=form)
    assert (got[0] == 0).all() and torch.equal(got[1], x.sink.view(1, 16, 1).expand(3, 16, 1))


@pytest.mark.parametrize("prefix_splits", [1, 2, 4, 7, 64])
@pytest.mark.parametrize("suffix_splits", [1, 2, 5])
def test_splits(prefix_splits, suffix_splits):
    x = Batch("V32", 5, 1, 40, 1500, [600, 0, 3, 1000, 129], 64, sink=True)
    x.check(x.call(prefix_splits=prefix_splits, suffix_splits=suffix_splits))


@pytest.mark.parametrize("form", FORMS)
def test_many_rows(form):
    """More 64-row blocks than SMs, an odd number of them."""
    x = Batch("V32", 150, 1, 65, 700, [r % 4 for r in range(150)], 64)
    x.check(x.call(flags=form))
    x = Batch("MODEL1", 80, 2, 128, 300, [r % 7 for r in range(80)], 64)
    x.check(x.call(flags=form))


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
def test_long_prefix(form, layout):
    x = Batch(layout, 12, 1, 64, 20000, [100 * r for r in range(12)], 64)
    x.check(x.call(flags=form))


def test_references_are_raised_along_the_prefix():
    """Scores that grow along the prefix: both softmax groups raise the references again and again."""
    x = Batch("V32", 5, 1, 64, 4000, [30] * 5, 64, seed=4)
    tok = torch.arange(4000, device="cuda")
    where = x.prefix_table.long()[tok // 64] * 64 + tok % 64
    g = torch.Generator(device="cuda").manual_seed(9)
    base = torch.randn(1, 512, device="cuda", generator=g)
    grow = (base * torch.linspace(0.0, 3.0, 4000, device="cuda")[:, None]).bfloat16()
    ops.kv_store(grow, torch.randn(4000, 64, device="cuda", generator=g).bfloat16(), where, x.kv)
    x.q[..., :512] = (base * torch.linspace(-1.0, 1.0, 5, device="cuda").view(5, 1, 1, 1)).bfloat16()
    out, mag, lse = x.definition()
    # 576 products and partial sums, each rounded to 2^-24 of at most sum |q k| = 512 * 3 / 24 * E[base^2]
    slack = 2 * 577 * 2.0 ** -24 * 3 * float((base * base).sum()) / 24 + SCORES
    for form in FORMS:
        got = x.call(flags=form)
        torch.cuda.synchronize()
        assert K.device_status() == 0
        assert ((got[0].double() - out).abs() <= U * (mag + out.abs()) + 2 * slack * mag).all()
        assert ((got[1].double() - lse).abs() <= slack + 2e-6 * lse.abs()).all()


def test_cross_check_kernels_agree():
    x = Batch("V32", 3, 2, 16, 200, [0, 40, 70], 16, sink=True)
    x.check(x.call(flags=N.FLAG_IMPL_SIMPLE))


def test_equal_to_one_list_per_request():
    x = Batch("V32", 4, 1, 64, 900, [10, 0, 200, 65], 64, sink=True)
    got = x.call()
    width = 900 + 200
    idx = torch.full((4, 1, width), -1, dtype=torch.int32, device="cuda")
    pos = torch.arange(width, device="cuda", dtype=torch.int32)
    for r, s in enumerate(x.suffix):
        idx[r, 0, :900] = ops.page_indices(x.prefix_table[None], pos[:900].view(1, 1, -1).contiguous(), 64).view(-1)
        if s:
            idx[r, 0, 900:900 + s] = ops.page_indices(x.table[r:r + 1], pos[:s].view(1, 1, -1).contiguous(), 64).view(-1)
    lens = torch.tensor([900 + s for s in x.suffix], dtype=torch.int32, device="cuda")
    want = ops.sparse_decode_fwd(x.q, x.kv, idx, lens, x.sink, None, None, None, None, None, 512, x.scale)
    x.check(got)
    x.check(want[:2])


@pytest.mark.parametrize("form", FORMS[1:])
def test_padded_page_stride_and_pages_beyond_4_gib(form):
    x = Batch("V32", 3, 1, 16, 130, [5, 64, 100], 64, pad=48)
    x.check(x.call(flags=form))
    before = (1 << 32) // (64 * 644) + 9
    x = Batch("V32", 3, 1, 16, 130, [5, 64, 100], 64, blocks_before=before)
    assert int(x.prefix_table.min()) * 64 * 644 > 1 << 32
    x.check(x.call(flags=form))


@pytest.mark.parametrize("form", FORMS[1:])
def test_pages_outside_the_cache_are_masked(form):
    x = Batch("V32", 3, 1, 16, 200, [70, 64, 130], 16)
    x.prefix_table[3], x.prefix_table[5], x.prefix_table[6] = -1, x.kv.size(0), 2 ** 31 - 1
    x.table[0, 1], x.table[2, 0], x.table[1, 3] = -5, 2 ** 30, x.kv.size(0) + 7
    x.check(x.call(flags=form))
    x.prefix_table.fill_(-1)                         # no token of the prefix at all
    x.check(x.call(flags=form))


@pytest.mark.parametrize("form", FORMS[1:])
def test_lengths_that_lie_are_clamped(form):
    x = Batch("V32", 4, 1, 16, 128, [64, 32, 16, 16], 16)
    x.table[:, 4] = x.table[:, 0]                    # the column behind the pages: filled rows again
    for r, s in enumerate([64, 32, 16, 16]):
        x.table[r, s // 16:4] = -1
    for p, s in ((2 ** 31 - 1, [2 ** 31 - 1, 70, 80, 1000]), (-4, [-1, -2 ** 31, 0, 3])):
        x.prefix_length.fill_(p)
        x.suffix_length.copy_(torch.tensor(s, dtype=torch.int32))
        x.check(x.call(flags=form), x.definition(p, s))


@pytest.mark.parametrize("layout", ["V32", "MODEL1"])
@pytest.mark.parametrize("form", FORMS)
def test_tokens_that_are_not_finite_reach_the_rows_that_see_them_alone(layout, form):
    x = Batch(layout, 7, 2, 16, 700, [40, 0, 129, 1, 300, 64, 2], 64, seed=3)
    want = x.definition()
    spoilt = torch.zeros(7, 2, dtype=torch.bool, device="cuda")
    for r, at, where in ((0, 39, "latent"), (2, 127, "latent"), (4, 299, "rope"), (6, 0, "latent")):
        page, at = int(x.table[r, at // 64]), at % 64
        spoilt[r] |= torch.arange(2, device="cuda") >= 1 - (x.suffix[r] - 1 - 64 * (0, 0, 1, 0, 4, 0, 0)[r] - at)
        if where == "latent":                              # 2^128 times the codes: infinities of both signs
            x.arena[page, 64 * (x.d + 128) + at * x.slots + 1] = 255
        else:
            x.arena[page, at * (x.d + 128) + x.d:][:2] = 0xff
    out, lse = x.call(flags=form)
    if form == N.FLAG_SHARED_DENSE:
        assert torch.isnan(out[spoilt]).all() and torch.isnan(lse.transpose(1, 2)[spoilt]).all()
    fine = ~spoilt
    off = (out.double() - want[0]).abs() / (U * (want[1] + want[0].abs()) + SCORES * want[1] + 1e-30)
    assert float(off[fine].max()) <= 1
    assert ((lse.double() - want[2]).abs().transpose(1, 2)[fine] <= SCORES + 2e-6 * want[2].abs().transpose(1, 2)[fine]).all()


@pytest.mark.parametrize("b", [1, 4, 20])
def test_a_row_of_one_set_that_is_not_finite(b):
    """Nothing but the set with the NaN holds tokens; few rows have more than 32 sets."""
    x = Batch("V32", b, 1, 16, 64, [40] * b, 64, seed=5)
    x.arena[int(x.table[b - 1, 0]), 39 * (x.d + 128) + x.d:][:2] = 0xff
    out, lse = x.call(flags=N.FLAG_SHARED_DENSE)
    assert torch.isnan(out[b - 1]).all() and torch.isnan(lse[b - 1]).all()
    assert torch.isfinite(out[:b - 1]).all() and torch.isfinite(lse[:b - 1]).all()


@pytest.mark.parametrize("form", FORMS[1:])
@pytest.mark.parametrize("pages", [300, 600])
def test_wide_tables_of_short_requests(pages, form):
    """A table that could hold far more own tokens than there are."""
    x = Batch("V32", 5, 2, 48, 700, [300, 0, 1, 129, 64], 64, seed=4, sink=True)
    x.table = torch.cat([x.table, torch.full((5, pages), 2 ** 30, dtype=torch.int32, device="cuda")], 1)
    x.check(x.call(flags=form))


@pytest.mark.parametrize("s_q,h_q", [(1, 8), (1, 24), (3, 16), (2, 64), (5, 40)])
def test_blocks_that_hold_parts_of_requests(s_q, h_q):
    suffix = [(53 * r * r) % 700 for r in range(23)]
    x = Batch("V32", 23, s_q, h_q, 3000, suffix, 64, seed=h_q)
    x.check(x.call(flags=N.FLAG_SHARED_DENSE))


@pytest.mark.parametrize("form", FORMS[1:])
def test_captured_and_replayed_with_other_lengths(form):
    x = Batch("V32", 6, 1, 64, 1000, [200, 100, 3, 0, 64, 65], 64)
    x.call(flags=form)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = x.call(flags=form)
    for p, s in ((1000, x.suffix), (0, [1, 100, 3, 0, 64, 65]), (777, [0] * 6), (1, [200, 1, 3, 0, 64, 2])):
        x.prefix_length.fill_(p)
        x.suffix_length.copy_(torch.tensor(s, dtype=torch.int32))
        g.replay()
        x.check(got, x.definition(p, s))


@pytest.mark.parametrize("form", FORMS[1:])
def test_streams_at_once_and_repeatability(form):
    x = Batch("V32", 8, 1, 64, 3000, [100] * 8, 64)
    first = x.call(flags=form)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for i in range(9):
        with torch.cuda.stream(streams[i % 3]):
            results.append(x.call(flags=form))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, first))
    x.check(first)


def test_operator_refuses():
    x = Batch("V32", 2, 1, 16, 100, [5, 6], 64)
    args = dict(q=x.q, kv=x.kv, prefix_table=x.prefix_table, prefix_length=x.prefix_length, block_table=x.table,
                suffix_length=x.suffix_length, attn_sink=None, d_v=512, sm_scale=0.04)
    ops.shared_prefix_decode_fwd(**args)
    for bad in (dict(q=x.q.float()), dict(q=x.q[0]), dict(q=x.q[..., :512]), dict(q=x.q.expand(2, 2, 16, 576)), dict(kv=x.kv[0]),
                dict(kv=x.kv.cpu()), dict(kv=x.kv[..., :640]), dict(d_v=256), dict(prefix_table=x.prefix_table.long()),
                dict(prefix_length=x.suffix_length), dict(prefix_length=x.prefix_length.cpu()), dict(block_table=x.table[:1]),
                dict(suffix_length=x.prefix_length), dict(attn_sink=torch.zeros(3, device="cuda")),
                dict(attn_sink=torch.zeros(16, device="cuda", dtype=torch.float64)), dict(block_table=x.table.t())):
        with pytest.raises(RuntimeError):
            ops.shared_prefix_decode_fwd(**{**args, **bad})
