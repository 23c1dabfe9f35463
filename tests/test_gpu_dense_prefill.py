"""Dense prefill of packed sequences against the definition in 64 bits.

Bounds.  With u = eps / 2 of the tensors' type, an output may be off by the rounding of the
weights, u * sum p |v|, and its own, u * |o|; the scores' 32-bit sums move the weights by at
most 3e-4 of themselves (192 products of 2^-24 each over logits of a few tens, and the
exponential's 2^-22).  The log-sum-exp and the largest logit carry the scores' error alone."""
import math

import pytest
import torch

from deepseek_v4_kernel import cuda as K
from deepseek_v4_kernel import ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
SCORES = 3e-4


def cu_of(lens):
    return torch.tensor([sum(lens[:i]) for i in range(len(lens) + 1)], dtype=torch.int32, device="cuda")


def definition(q, k, v, lq, lk, scale, causal, sink, q0=0, k0=0):
    """Outputs, sums of p |v|, largest logits and log-sum-exps in 64 bits; NaN and infinities
    of v reach the rows that see them and no others."""
    tq, h_q, _ = q.shape
    g = h_q // k.size(1)
    out = torch.full((tq, h_q, v.size(2)), math.nan, dtype=torch.float64, device="cuda")
    mag, ml, lse = out.clone(), out[..., 0].clone(), out[..., 0].clone()
    for a, c in zip(lq, lk):
        qs = q[q0:q0 + a].double().transpose(0, 1)
        ks = k[k0:k0 + c].double().transpose(0, 1).repeat_interleave(g, 0)
        vs = v[k0:k0 + c].double().transpose(0, 1).repeat_interleave(g, 0)
        see = torch.ones(a, c, dtype=torch.bool, device="cuda")
        if causal:
            see = see.tril(c - a)
        x = torch.where(see, (qs @ ks.transpose(1, 2)) * scale, -math.inf)
        if c == 0:
            x = torch.full((h_q, a, 1), -math.inf, dtype=torch.float64, device="cuda")
            vs, see = torch.zeros(h_q, 1, v.size(2), dtype=torch.float64, device="cuda"), torch.zeros(a, 1, dtype=torch.bool, device="cuda")
        m, e = x.amax(-1), torch.logsumexp(x, -1)
        both = e if sink is None else torch.logaddexp(e, sink.double().view(-1, 1).expand_as(e))
        none = e == -math.inf
        w = torch.where(none[..., None], torch.zeros_like(x), torch.exp(x - both[..., None]))
        w = torch.where(see, w, torch.zeros_like(w))
        fin = torch.where(torch.isfinite(vs), vs, torch.zeros_like(vs))
        o = w @ fin
        for special in (vs == math.inf, vs == -math.inf, torch.isnan(vs)):
            if special.any():
                hit = see.double() @ special.double() > 0
                val = torch.where(special, vs, torch.zeros_like(vs)).sum(1, keepdim=True)
                val = torch.where(special.any(1, keepdim=True), torch.where(torch.isnan(val), val, val.sign() * math.inf), val)
                o = torch.where(hit, o + val, o)
        out[q0:q0 + a] = o.transpose(0, 1)
        mag[q0:q0 + a] = (w @ fin.abs()).transpose(0, 1)
        ml[q0:q0 + a] = m.transpose(0, 1)
        lse[q0:q0 + a] = torch.where(none, torch.full_like(e, math.inf), e).transpose(0, 1)
        q0, k0 = q0 + a, k0 + c
    return out, mag, ml, lse


def check(got, want, dtype):
    out, ml, lse = got
    o, mag, wml, wlse = want
    torch.cuda.synchronize()
    assert K.device_status() == 0
    u = torch.finfo(dtype).eps / 2
    g = out.double()
    same = (g == o) | (torch.isnan(g) & torch.isnan(o))
    off = torch.where(same, torch.zeros_like(o), (g - o).abs())
    # results below fp16's normal range are rounded to its smallest step instead
    bound = u * (mag + o.abs()) + SCORES * mag + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    worst = float(torch.where(same, torch.zeros_like(off), off / bound).nan_to_num(1e9).max()) if off.numel() else 0.0
    assert worst <= 1, f"{worst:.3g} times the bound"
    for a, b in ((ml, wml), (lse, wlse)):
        fine = torch.isfinite(b)
        assert torch.equal(a[~fine].double().nan_to_num(7.0), b[~fine].nan_to_num(7.0))
        assert ((a.double() - b).abs()[fine] <= SCORES + 2e-6 * b.abs()[fine]).all()


def make(lq, lk, h_q, h_kv, d_qk, d_v, dtype, seed=0, std=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q = (torch.randn(sum(lq), h_q, d_qk, device="cuda", generator=g) * std).to(dtype)
    k = torch.randn(sum(lk), h_kv, d_qk, device="cuda", generator=g).to(dtype)
    v = torch.randn(sum(lk), h_kv, d_v, device="cuda", generator=g).to(dtype)
    return q, k, v


def run(q, k, v, lq, lk, causal=True, sink=None, scale=None, **kw):
    scale = q.size(2) ** -0.5 if scale is None else scale
    got = K.dense_prefill_fwd(q, k, v, cu_of(lq), cu_of(lk), scale, causal, sink, **kw)
    check(got, definition(q, k, v, lq, lk, scale, causal, sink), q.dtype)
    return got


DIMS = [(64, 64), (128, 128), (192, 128)]


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("h_q,h_kv", [(2, 2), (8, 2), (6, 2)])
def test_packed_lengths(d_qk, d_v, dtype, causal, h_q, h_kv):
    lens = [1, 127, 0, 128, 129, 2, 255, 257, 64, 0, 700]
    q, k, v = make(lens, lens, h_q, h_kv, d_qk, d_v, dtype)
    run(q, k, v, lens, lens, causal)


@pytest.mark.parametrize("h_q,h_kv", [(1, 1), (3, 1), (5, 1), (7, 7), (10, 2), (24, 2), (64, 1), (128, 1), (130, 1), (131, 1), (256, 1)])
def test_groups(h_q, h_kv):
    lq, lk = [1, 33, 150], [40, 33, 301]
    q, k, v = make(lq, lk, h_q, h_kv, 128, 128, BF16, seed=h_q)
    run(q, k, v, lq, lk)


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("causal", [True, False])
def test_contexts_and_rows_that_see_nothing(d_qk, d_v, causal):
    # contexts of odd lengths; more queries than keys (the first ones see nothing); no keys at all
    lq, lk = [5, 300, 1, 200, 40, 3, 7], [1000, 555, 4096, 100, 0, 2, 7]
    q, k, v = make(lq, lk, 8, 4, d_qk, d_v, BF16, seed=3)
    sink = torch.randn(8, device="cuda")
    run(q, k, v, lq, lk, causal)
    run(q, k, v, lq, lk, causal, sink)
    empty = [0] * len(lq)
    got = run(q, k[:0], v[:0], lq, empty, causal, sink)
    assert (got[0] == 0).all() and (got[1] == -math.inf).all() and (got[2] == math.inf).all()


@pytest.mark.parametrize("n_splits", [1, 2, 3, 7, 64])
@pytest.mark.parametrize("d_qk,d_v", DIMS)
def test_single_tokens_and_key_ranges(n_splits, d_qk, d_v):
    lq, lk = [1, 1, 2, 1, 1, 0, 1], [1, 5000, 129, 128, 1025, 64, 0]
    q, k, v = make(lq, lk, 16, 2, d_qk, d_v, FP16, seed=5)
    run(q, k, v, lq, lk, sink=torch.randn(16, device="cuda"), n_splits=n_splits)
    run(q, k, v, lq, lk, causal=False, n_splits=n_splits)


@pytest.mark.parametrize("b", [31, 32, 33, 70, 300])
@pytest.mark.parametrize("n_splits", [None, 2, 9, 64])
def test_ranges_of_many_uneven_sequences(b, n_splits):
    """More sequences than a warp has lanes; one of them holds most of the keys."""
    lq = [(0, 1, 1, 2, 1)[r % 5] for r in range(b)]
    lk = [(r * 37) % 400 if r != b - 2 else 9000 for r in range(b)]
    q, k, v = make(lq, lk, 4, 1, 64, 64, BF16, seed=b)
    run(q, k, v, lq, lk, n_splits=n_splits)


@pytest.mark.parametrize("n_splits", [None, 6])
def test_ranges_with_bounds_that_do_not_cover_the_tensors(n_splits):
    """Rows of no sequence stay as they are; bounds beyond the tensors are clamped."""
    q, k, v = make([40], [5000], 8, 2, 128, 128, BF16, seed=8)
    cq, ck = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([3, 4, 6], [10, 2000, 1 << 30]))
    out = torch.full_like(q, 7.0)
    got = K.dense_prefill_fwd(q, k, v, cq, ck, 0.1, True, None, out, n_splits=n_splits)
    check((got[0][3:6], got[1][3:6], got[2][3:6]),
          definition(q[3:6], k[10:], v[10:], [1, 2], [1990, 3000], 0.1, True, None), BF16)
    assert (out[:3] == 7).all() and (out[6:] == 7).all()


def test_key_ranges_of_long_rows():
    lq, lk = [300, 17], [1300, 900]
    q, k, v = make(lq, lk, 6, 3, 128, 128, BF16, seed=6)
    for n in (2, 5):
        run(q, k, v, lq, lk, n_splits=n)


@pytest.mark.parametrize("scale,std", [(1.0, 1.0), (1e-6, 1.0), (0.09, 30.0)])
def test_logits_of_every_size(scale, std):
    """Large logits: the reference is raised again and again; tiny ones: a plain mean.  The
    scores' absolute error grows with them, so the weights are held to what they allow."""
    lens = [400, 31]
    q, k, v = make(lens, lens, 4, 4, 64, 64, BF16, seed=7, std=std)
    k[:431] *= torch.linspace(0.1, 1.0, 431, device="cuda").view(-1, 1, 1).to(BF16)    # later keys larger
    got = K.dense_prefill_fwd(q, k, v, cu_of(lens), cu_of(lens), scale)
    o, mag, ml, lse = definition(q, k, v, lens, lens, scale, True, None)
    torch.cuda.synchronize()
    assert K.device_status() == 0
    # 64 products, each and each partial sum rounded to 2^-24 of at most sum |q k|
    worst = float((q.abs().double().transpose(0, 1) @ k.abs().double().transpose(0, 1).transpose(1, 2)).max()) * scale
    slack = 2 * 65 * 2 ** -24 * worst + SCORES
    u = torch.finfo(BF16).eps / 2
    assert ((got[0].double() - o).abs() <= u * (mag + o.abs()) + 2 * slack * mag + 1e-30).all()
    assert ((got[1].double() - ml).abs() <= slack).all() and ((got[2].double() - lse).abs() <= slack + 2e-6 * lse.abs()).all()


@pytest.mark.parametrize("d_qk,d_v", DIMS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_masked_places_may_hold_anything(d_qk, d_v, dtype):
    lq, lk = [200, 90, 260], [200, 300, 260]
    q, k, v = make(lq, lk, 4, 2, d_qk, d_v, dtype, seed=8)
    # the rows behind the last sequence, and a whole sequence between two others
    q2, k2, v2 = (torch.cat([t, torch.full_like(t[:150], math.nan)]) for t in (q, k, v))
    k2[200:500], v2[200:500] = math.nan, math.inf
    want = definition(q2, k2, v2, lq, lk, d_qk ** -0.5, True, None)
    got = K.dense_prefill_fwd(q2, k2, v2, cu_of(lq), cu_of(lk), d_qk ** -0.5)
    rows = torch.ones(700, dtype=torch.bool, device="cuda")
    rows[200:290], rows[550:] = False, False
    check([t[rows] for t in got], [t[rows] for t in want], dtype)
    assert torch.isnan(got[0][200:290]).all()                      # those do see NaN keys


@pytest.mark.parametrize("h_q,h_kv", [(2, 2), (8, 2)])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n_splits", [1, 3])
def test_later_values_do_not_reach_earlier_rows(h_q, h_kv, dtype, n_splits):
    lens = [300, 140]
    q, k, v = make(lens, lens, h_q, h_kv, 128, 128, dtype, seed=9)
    v[37, 0, 5], v[250, -1, 6], v[251, -1, 6], v[299, 0, 127] = math.inf, -math.inf, math.inf, math.nan
    v[300 + 139, 0, :] = math.nan
    k[290:300, 0] = k[290:300, 0] * 1.0
    run(q, k, v, lens, lens, n_splits=n_splits)


def test_nan_keys_show_in_the_rows_that_see_them():
    lens = [200]
    q, k, v = make(lens, lens, 2, 2, 128, 128, BF16, seed=10)
    clean = K.dense_prefill_fwd(q, k, v, cu_of(lens), cu_of(lens), 0.1)
    k[150] = math.nan
    got = K.dense_prefill_fwd(q, k, v, cu_of(lens), cu_of(lens), 0.1)
    assert torch.equal(got[0][:150], clean[0][:150]) and torch.equal(got[2][:150], clean[2][:150])
    assert torch.isnan(got[0][150:]).all() and torch.isnan(got[2][150:]).all()


def test_strides_and_rows_of_no_sequence():
    lq, lk = [70, 33], [100, 33]
    g = torch.Generator(device="cuda").manual_seed(11)
    wide = torch.randn(160, 9, 200, device="cuda", generator=g).to(BF16)
    q = wide[20:140, 1:7, 8:136]                                        # 120 rows, 103 of them in sequences
    up = torch.randn(150, 3, 256, device="cuda", generator=g).to(BF16)
    k, v = up[..., :128], up[..., 128:]
    hold = torch.full((130, 6, 160), 3.0, dtype=BF16, device="cuda")
    out = hold[5:125, :, 16:144]
    cq = torch.tensor([4, 74, 107], dtype=torch.int32, device="cuda")
    ck = torch.tensor([7, 107, 140], dtype=torch.int32, device="cuda")
    for n in (1, 2):
        hold.fill_(3.0)
        got = K.dense_prefill_fwd(q, k, v, cq, ck, 0.09, True, None, out, n_splits=n)
        assert got[0] is out
        want = definition(q, k, v, lq, lk, 0.09, True, None, q0=4, k0=7)
        check([t[4:107] for t in got], [t[4:107] for t in want], BF16)
        keep = torch.ones_like(hold, dtype=torch.bool)
        keep[9:112, :, 16:144] = False
        assert (hold[keep] == 3.0).all()
    # heads outermost
    qt, kt, vt = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in make(lq, lk, 6, 3, 128, 128, BF16))
    run(qt, kt, vt, lq, lk)


def test_offsets_beyond_32_bits():
    stride = 1 << 23                                                    # elements between tokens
    buf = torch.empty(300 * stride, dtype=BF16, device="cuda")          # 5 GB
    lens = [300]
    q, k, v = make(lens, lens, 1, 1, 128, 128, BF16, seed=12)
    far = [torch.as_strided(buf, (300, 1, 128), (stride, 128, 1), 256 * i) for i in range(4)]
    for f, t in zip(far, (q, k, v)):
        f.copy_(t)
    run(*far[:3], lens, lens, out=far[3])


def test_bounds_that_lie():
    """Bounds outside the tensors or descending are clamped: nothing outside is touched."""
    q, k, v = make([64], [64], 2, 2, 128, 128, BF16)
    guard = torch.full((96, 2, 128), 5.0, dtype=BF16, device="cuda")
    for cq, ck in (([-5, 1000], [-9, 77]), ([60, 10], [3, 1]), ([0, 64], [64, 0]), ([2 ** 31 - 1, -2 ** 31], [-2 ** 31, 2 ** 31 - 1]),
                   ([0, 70, 3, 64], [0, 64, 64, 2])):
        t = [torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cq, ck)]
        for n in (1, 2):
            K.dense_prefill_fwd(q, k, v, t[0], t[1], 0.1, True, None, guard[16:80], n_splits=n)
    torch.cuda.synchronize()
    assert K.device_status() == 0
    assert (guard[:16] == 5.0).all() and (guard[80:] == 5.0).all()


def test_empty_calls():
    q, k, v = make([3], [3], 2, 2, 64, 64, BF16)
    out, ml, lse = ops.dense_prefill_fwd(q[:0], k, v, cu_of([0]), cu_of([3]), 0.1)
    assert out.shape == (0, 2, 64) and ml.shape == lse.shape == (0, 2)
    ops.dense_prefill_fwd(q, k, v, cu_of([]), cu_of([]), 0.1)


def test_two_streams_at_once_and_repeatability():
    lens = [500, 300, 1]
    q, k, v = make(lens, lens, 8, 2, 128, 128, BF16, seed=13)
    cu = cu_of(lens)
    first = ops.dense_prefill_fwd(q, k, v, cu, cu, 0.09)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    results = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            results.append(ops.dense_prefill_fwd(q, k, v, cu, cu, 0.09))
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(r, first))


def test_captured_and_replayed_with_other_lengths():
    lq, lk = [1, 1, 1, 1], [900, 1, 300, 47]
    q, k, v = make([4], [2000], 8, 2, 128, 128, BF16, seed=14)
    cq, ck = cu_of(lq), cu_of(lk)
    ops.dense_prefill_fwd(q, k, v, cq, ck, 0.09)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.dense_prefill_fwd(q, k, v, cq, ck, 0.09)
    for lens in ([900, 1, 300, 47], [1, 1, 1, 1997], [0, 0, 5, 6]):
        ck.copy_(cu_of(lens))
        g.replay()
        check(got, definition(q, k, v, lq, lens, 0.09, True, None), BF16)


def test_operator_refuses():
    q, k, v = make([4], [4], 4, 2, 128, 128, BF16)
    cu = cu_of([4])
    good = (q, k, v, cu, cu, 0.1)
    ops.dense_prefill_fwd(*good)
    for bad in ((q.float(), k, v, cu, cu, 0.1), (q, k.half(), v, cu, cu, 0.1), (q[0], k, v, cu, cu, 0.1), (q[..., :96], k, v, cu, cu, 0.1),
                (q, k[:3], v, cu, cu, 0.1), (q[:, :3], k, v, cu, cu, 0.1), (q, k, v, cu.long(), cu, 0.1), (q, k, v, cu, cu_of([2, 2]), 0.1),
                (q, k, v, cu.cpu(), cu, 0.1), (q, k, v, cu, cu, 0.0), (q, k, v, cu, cu, -0.1), (q, k, v, cu, cu, math.nan),
                (q, k.cpu(), v, cu, cu, 0.1), (q, k[:, :1].expand(4, 2, 128), v, cu, cu, 0.1),
                (q, k, v, cu, cu, 0.1, True, torch.zeros(3, device="cuda")), (q, k, v, cu, cu, 0.1, True, None, q[:3]),
                (q.transpose(1, 2), k, v, cu, cu, 0.1)):
        with pytest.raises(RuntimeError):
            ops.dense_prefill_fwd(*bad)
