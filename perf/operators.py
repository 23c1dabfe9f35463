"""Cases of the serving operators around the sparse attention: block tables and slot maps,
dense causal prefill of packed sequences, decode of a batch that shares a long prefix.

`run` computes them in plain torch operations, or, with `own` set, through the package."""
import math
import os
import random
import sys

import torch

own = False          # set from outside: False = plain torch, True = this repository's operators

DEV = "cuda"
LAYOUTS = {"MODEL1": (448, 64, 7, 8), "V32": (512, 128, 4, 4)}  # latent values, values per scale, scales, scale bytes
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# --------------------------------------------------------------------------- the cases
def listed():
    return [
        # one decode step of 64 running requests: one new token each, most of them on a page they have
        {"name": "slots: decode step", "op": "slots", "b": 64, "page": 64, "cached": "4096:65536", "new": "1:1", "mix": 1},
        # admission of a batch of prompts, a third of them behind a cached prefix, pages of 48 tokens
        {"name": "slots: prompts admitted", "op": "slots", "b": 301, "page": 48, "cached": "0:5000", "new": "1:2048", "mix": 2},
        # the index lists of one sparse decode step: 64 requests, 2048 positions each
        {"name": "indices: decode step", "op": "indices", "lens": _text([1] * 64), "ctx": 32768, "topk": 2048, "page": 64, "packed": False},
        # the index lists of a sparse prefill of three packed sequences
        {"name": "indices: prefill", "op": "indices", "lens": "5000,1,3191", "ctx": 0, "topk": 2048, "page": 256, "packed": True},
        # short prompts admitted together, grouped heads
        {"name": "prefill: short prompts", "op": "prefill", "b": 13, "q": "1:300", "ctx": "0:0", "h_q": 16, "h_kv": 2,
         "d_qk": 128, "d_v": 128, "dtype": "bf16", "causal": True, "sink": False, "mix": 3},
        # one latent-attention prompt with the keys and values of every head written out, one tensor-parallel shard
        {"name": "prefill: one prompt of 8192", "op": "prefill", "b": 1, "q": "8192:8192", "ctx": "0:0", "h_q": 16, "h_kv": 16,
         "d_qk": 192, "d_v": 128, "dtype": "bf16", "causal": True, "sink": False, "mix": 4},
        # packed prompts of uneven lengths, some behind a cached context, grouped heads with sinks
        {"name": "prefill: packed and chunked", "op": "prefill", "b": 7, "q": "257:4096", "ctx": "0:2048", "h_q": 24, "h_kv": 4,
         "d_qk": 128, "d_v": 128, "dtype": "fp16", "causal": True, "sink": True, "mix": 5},
        # single tokens over contexts of up to 16384
        {"name": "prefill: single tokens", "op": "prefill", "b": 8, "q": "1:1", "ctx": "1000:16383", "h_q": 32, "h_kv": 8,
         "d_qk": 128, "d_v": 128, "dtype": "bf16", "causal": True, "sink": False, "mix": 6},
        # four samples of one prompt, a tensor-parallel shard of 16 heads
        {"name": "shared prefix: 4 samples", "op": "shared", "layout": "V32", "b": 4, "s_q": 1, "h_q": 16, "prefix": 2000,
         "suffix": "1:100", "page": 64, "sink": False, "mix": 7},
        # 16 requests behind one system prompt, all heads
        {"name": "shared prefix: 16 requests", "op": "shared", "layout": "V32", "b": 16, "s_q": 1, "h_q": 64, "prefix": 32768,
         "suffix": "1:1024", "page": 64, "sink": False, "mix": 8},
        # 64 requests, the largest
        {"name": "shared prefix: 64 requests", "op": "shared", "layout": "V32", "b": 64, "s_q": 1, "h_q": 64, "prefix": 32768,
         "suffix": "64:2048", "page": 64, "sink": False, "mix": 9},
        # two drafted tokens per request, the other cache layout, a sink, an odd number of heads and of tokens
        {"name": "shared prefix: drafted tokens", "op": "shared", "layout": "MODEL1", "b": 37, "s_q": 2, "h_q": 24, "prefix": 10007,
         "suffix": "0:500", "page": 256, "sink": True, "mix": 10},
    ]


# A case holds plain values: a range of lengths is "least:most", a list of them "n,n,n".
def _text(lens):
    return ",".join(map(str, lens))


def _lens(case):
    return [int(n) for n in case["lens"].split(",")]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(max(lo, 1)), math.log(max(hi, 1)))))))


def draw(rng):
    op = rng.choice(["slots", "indices", "prefill", "prefill", "shared", "shared"])
    mix = rng.randrange(1 << 20)
    if op == "slots":
        hi = rng.choice([1, 4, 300, 2000])
        return {"op": op, "b": _log_int(rng, 1, 400), "page": rng.choice([1, 16, 48, 64, 256]),
                "cached": "0:%d" % _log_int(rng, 1, 30000), "new": "%d:%d" % (rng.choice([0, 1]), hi), "mix": mix}
    if op == "indices":
        packed = rng.random() < 0.5
        if packed:
            lens = [_log_int(rng, 1, 1500) for _ in range(rng.randint(1, 5))]
        else:
            lens = [rng.choice([1, 2, 3])] * _log_int(rng, 1, 300)
        return {"op": op, "lens": _text(lens), "ctx": _log_int(rng, 1, 40000), "topk": rng.choice([1, 63, 128, 500, 2047, 2048]),
                "page": rng.choice([16, 48, 64, 256]), "packed": packed}
    if op == "prefill":
        d_qk, d_v = rng.choice([(64, 64), (128, 128), (192, 128)])
        h_kv = rng.choice([1, 2, 3, 4, 8])
        h_q = h_kv * rng.choice([1, 2, 3, 4, 5, 7, 8])
        cost = 2.0e9 / h_q                      # score entries per head of the largest listed case, roughly
        if rng.random() < 0.3:                  # single tokens, or a few, behind a context
            b, q, ctx = _log_int(rng, 1, 60), [1, rng.choice([1, 2, 5])], [0, _log_int(rng, 1, 20000)]
        else:
            b = _log_int(rng, 1, 24)
            top = max(1, min(6000, int(math.sqrt(cost / b / 2))))
            q, ctx = [rng.choice([0, 1, 17]), _log_int(rng, 1, top)], [0, rng.choice([0, 0, top])]
            q = sorted(q)
        return {"op": op, "b": b, "q": "%d:%d" % tuple(q), "ctx": "%d:%d" % tuple(ctx), "h_q": h_q, "h_kv": h_kv, "d_qk": d_qk, "d_v": d_v,
                "dtype": rng.choice(["bf16", "fp16"]), "causal": rng.random() < 0.8, "sink": rng.random() < 0.3, "mix": mix}
    layout = rng.choice(["V32", "V32", "MODEL1"])
    return {"op": op, "layout": layout, "b": _log_int(rng, 1, 64), "s_q": rng.choice([1, 1, 1, 2, 3]),
            "h_q": rng.choice([1, 8, 16, 20, 64]), "prefix": rng.choice([0, _log_int(rng, 1, 30000), _log_int(rng, 100, 30000)]),
            "suffix": "0:%d" % _log_int(rng, 1, 1500), "page": rng.choice([16, 48, 64, 256]), "sink": rng.random() < 0.4, "mix": mix}


def _spread(mix, n, span):
    """n whole numbers of a range, spread over their logarithm, the same for the same `mix`."""
    lo, hi = map(int, span.split(":"))
    rng = random.Random(mix)
    return [lo if hi <= lo else min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo + 1), math.log(hi + 1))) - 1))) for _ in range(n)]


def _pages(tokens, page):
    return (tokens + page - 1) // page


def _slot_lens(case):
    cached = _spread(case["mix"], case["b"], case["cached"])
    rng = random.Random(case["mix"] + 1)
    if case["cached"].startswith("0:"):
        cached = [c if rng.random() < 0.34 or int(case["new"].split(":")[1]) <= 4 else 0 for c in cached]
    return cached, _spread(case["mix"] + 2, case["b"], case["new"])


def _prefill_lens(case):
    q = _spread(case["mix"], case["b"], case["q"])
    q[0] = max(q[0], 1)
    return q, [n + c for n, c in zip(q, _spread(case["mix"] + 1, case["b"], case["ctx"]))]


# --------------------------------------------------------------------------- inputs
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device=DEV)


def _quantised(gen, tokens, layout):
    """Cache bytes of random tokens: [tokens, latent + 128] bytes and [tokens, scale bytes]."""
    d, tile, n, slots = LAYOUTS[layout]
    latent = torch.randn(tokens, n, tile, device=DEV, generator=gen).bfloat16().float()
    exp = torch.ceil(torch.log2(latent.abs().amax(-1).clamp_min(1e-4) / 448.0))
    body = torch.empty(tokens, d + 128, dtype=torch.uint8, device=DEV)
    body[:, :d] = (latent * torch.exp2(-exp).unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8).view(tokens, d)
    body[:, d:] = torch.randn(tokens, 64, device=DEV, generator=gen).bfloat16().view(torch.uint8)
    scales = torch.zeros(tokens, slots, dtype=torch.uint8, device=DEV)
    scales[:, :n] = (exp + 127).to(torch.uint8)
    return body, scales


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(seed)
    s = {"case": case}
    if case["op"] == "slots":
        cached, new = _slot_lens(case)
        page = case["page"]
        old = [_pages(c, page) for c in cached]
        full = [_pages(c + n, page) for c, n in zip(cached, new)]
        width = max(max(full), 1) + 3
        ids = torch.randperm(sum(full) + 7, device=DEV, generator=gen).int()
        held = torch.arange(width, device=DEV) < _ints(old)[:, None]
        table = torch.full((case["b"], width), -1, dtype=torch.int32, device=DEV)
        table[held] = ids[: sum(old)]
        s.update(table=table, free=ids[sum(old):].contiguous(), cached=_ints(cached), new=_ints(new),
                 n_slots=_pages(max(sum(new), 1), 64) * 64)
    elif case["op"] == "indices":
        lens, topk, page = _lens(case), case["topk"], case["page"]
        reach = torch.cat([torch.arange(1, n + 1, device=DEV) for n in lens]) + case["ctx"]   # tokens a row sees
        pos = (torch.rand(sum(lens), topk, device=DEV, generator=gen) * reach[:, None]).int()
        pos.masked_fill_(torch.arange(topk, device=DEV) >= reach[:, None], -1)
        need = [_pages(n + case["ctx"], page) for n in lens]
        ids = torch.randperm(sum(need) + 5, device=DEV, generator=gen).int()
        table = torch.full((len(lens), max(need)), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(max(need), device=DEV) < _ints(need)[:, None]] = ids[: sum(need)]
        cu = None
        if case["packed"]:
            cu = torch.zeros(len(lens) + 1, dtype=torch.int32, device=DEV)
            cu[1:] = _ints(lens).cumsum(0)
        else:
            pos = pos.view(len(lens), lens[0], topk)
        s.update(table=table, pos=pos, cu=cu)
    elif case["op"] == "prefill":
        ql, kl = _prefill_lens(case)
        dt, tq, tk = DTYPES[case["dtype"]], sum(ql), sum(kl)
        s["q"] = torch.randn(tq, case["h_q"], case["d_qk"], device=DEV, generator=gen).to(dt)
        s["k"] = torch.randn(tk, case["h_kv"], case["d_qk"], device=DEV, generator=gen).to(dt)
        # values are a column slice of the up-projection that also made the keys
        s["v"] = torch.randn(tk, case["h_kv"], 128 + case["d_v"], device=DEV, generator=gen).to(dt)[..., 128:]
        for name, n in (("cu_q", ql), ("cu_k", kl)):
            s[name] = torch.zeros(len(n) + 1, dtype=torch.int32, device=DEV)
            s[name][1:] = _ints(n).cumsum(0)
        s["scale"] = case["d_qk"] ** -0.5
        s["sink"] = torch.randn(case["h_q"], device=DEV, generator=gen) if case["sink"] else None
        s["max"] = (max(ql), max(kl))           # for the padded plain form
    else:
        d, _, _, slots = LAYOUTS[case["layout"]]
        page, b = case["page"], case["b"]
        suffix = _spread(case["mix"], b, case["suffix"])
        n_pre = _pages(case["prefix"], page)
        own_pages = [_pages(n, page) for n in suffix]
        blocks = n_pre + sum(own_pages) + 3
        body, scales = _quantised(gen, blocks * page, case["layout"])
        row = d + 128
        arena = torch.empty(blocks, -(-page * (row + slots) // 16) * 16, dtype=torch.uint8, device=DEV)
        arena[:, : page * row] = body.view(blocks, page * row)
        arena[:, page * row: page * (row + slots)] = scales.view(blocks, page * slots)
        ids = torch.randperm(blocks, device=DEV, generator=gen).int()
        width = max(max(own_pages), 1) + 1
        table = torch.full((b, width), -1, dtype=torch.int32, device=DEV)
        table[torch.arange(width, device=DEV) < _ints(own_pages)[:, None]] = ids[n_pre: n_pre + sum(own_pages)]
        s.update(arena=arena, kv=torch.as_strided(arena, (blocks, page, 1, row + slots), (arena.stride(0), row + slots, row + slots, 1)),
                 prefix_table=ids[:n_pre].contiguous(), prefix_length=_ints([case["prefix"]]),
                 table=table, suffix=_ints(suffix), longest=max(suffix),
                 q=torch.randn(b, case["s_q"], case["h_q"], d + 64, device=DEV, generator=gen).bfloat16(),
                 scale=(d + 64) ** -0.5, sink=torch.randn(case["h_q"], device=DEV, generator=gen) if case["sink"] else None)
    return s


# --------------------------------------------------------------------------- one pass
def _ops():
    root = os.path.join(os.getcwd(), "deepseek-v4-flash-sm120_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from deepseek_v4_kernel import ops
    return ops


_kernels = None


def run(s):
    global _kernels
    op = s["case"]["op"]
    if own:
        if _kernels is None:
            _kernels = _ops()
        if op == "slots":
            return (s["table"],) + tuple(_kernels.build_slot_maps(s["table"], s["cached"], s["new"], s["free"], s["case"]["page"], s["n_slots"]))
        if op == "indices":
            return _kernels.page_indices(s["table"], s["pos"], s["case"]["page"], s["cu"])
        if op == "prefill":
            return _kernels.dense_prefill_fwd(s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], s["scale"], s["case"]["causal"], s["sink"])
        return _kernels.shared_prefix_decode_fwd(s["q"], s["kv"], s["prefix_table"], s["prefix_length"], s["table"], s["suffix"],
                                                 s["sink"], 512, s["scale"])
    return {"slots": _plain_slots, "indices": _plain_indices, "prefill": _plain_prefill, "shared": _plain_shared}[op](s)


def _plain_slots(s):
    table, cached, new, free, page = s["table"], s["cached"].long(), s["new"].long(), s["free"], s["case"]["page"]
    b, width = table.shape
    end = new.cumsum(0)
    old = (cached + page - 1) // page
    need = (cached + new + page - 1) // page - old
    first = need.cumsum(0) - need                                   # of a request's pages in the free list
    col = torch.arange(width, device=DEV)[None]
    fresh = (col >= old[:, None]) & (col < (old + need)[:, None])
    at = (first[:, None] + col - old[:, None]).clamp(0, free.numel() - 1)
    full = torch.where(fresh, free[at], table)
    tok = torch.arange(s["n_slots"], device=DEV)
    r = torch.searchsorted(end, tok, right=True).clamp(max=b - 1)
    live = tok < end[-1]
    pos = cached[r] + tok - (end - new)[r]
    pos = torch.where(live, pos, torch.zeros_like(pos))
    slots = torch.where(live, full[r, pos // page].long() * page + pos % page, torch.full_like(pos, -1))
    zero = torch.zeros(1, dtype=torch.int64, device=DEV)
    return (full, slots, torch.where(live, pos, torch.full_like(pos, -1)).int(), torch.cat([zero, end]).int(),
            torch.cat([zero, (cached + new).cumsum(0)]).int(), need.sum().view(1).int())


def _plain_indices(s):
    pos, table, page = s["pos"], s["table"], s["case"]["page"]
    if s["cu"] is None:
        req = torch.arange(table.size(0), device=DEV).view(-1, 1, 1)
    else:
        req = (torch.searchsorted(s["cu"], torch.arange(pos.size(0), device=DEV, dtype=torch.int32), right=True) - 1).view(-1, 1)
    p = pos.long()
    ids = table[req, (p // page).clamp(0, table.size(1) - 1)].long()
    return torch.where((p < 0) | (p // page >= table.size(1)) | (ids < 0), torch.full_like(p, -1), ids * page + p % page).int()


def _plain_prefill(s):
    """All sequences padded to the longest one."""
    cu_q, cu_k, (mq, mk) = s["cu_q"].long(), s["cu_k"].long(), s["max"]
    h_q, h_kv, d_v = s["q"].size(1), s["k"].size(1), s["v"].size(2)
    lq, lk = cu_q.diff(), cu_k.diff()
    b = lq.numel()
    i, j = torch.arange(mq, device=DEV), torch.arange(mk, device=DEV)
    iq = (cu_q[:-1, None] + i).clamp(max=max(s["q"].size(0) - 1, 0))
    ik = (cu_k[:-1, None] + j).clamp(max=max(s["k"].size(0) - 1, 0))
    out = torch.zeros(s["q"].size(0), h_q, d_v, dtype=s["q"].dtype, device=DEV)
    top = torch.full((s["q"].size(0), h_q), -math.inf, device=DEV)
    lse = torch.full((s["q"].size(0), h_q), math.inf, device=DEV)
    if mq == 0:
        return out, top, lse
    see = (j[None, None] < lk[:, None, None]) & (i[None, :, None] < lq[:, None, None])
    if s["case"]["causal"]:
        see = see & (j[None, None] <= i[None, :, None] + (lk - lq)[:, None, None])
    q = s["q"][iq].float().transpose(1, 2).reshape(b, h_kv, (h_q // h_kv) * mq, -1)
    k, v = s["k"][ik].float().transpose(1, 2), s["v"][ik].float().transpose(1, 2)
    x = torch.matmul(q, k.transpose(2, 3)).view(b, h_q, mq, mk)
    x.mul_(s["scale"]).masked_fill_(~see[:, None], -math.inf)
    m = x.amax(-1) if mk else torch.full((b, h_q, mq), -math.inf, device=DEV)
    x.sub_(m.clamp_min(-1e30)[..., None]).exp_()
    l = x.sum(-1)
    o = torch.matmul(x.view(b, h_kv, (h_q // h_kv) * mq, mk), v).view(b, h_q, mq, d_v)
    full_lse = m + l.log()
    whole = l if s["sink"] is None else l + (s["sink"][None, :, None] - m).exp()
    o = torch.where((l > 0)[..., None], o / whole[..., None], torch.zeros_like(o))
    live = i[None] < lq[:, None]
    out[iq[live]] = o.transpose(1, 2)[live].to(out.dtype)
    top[iq[live]] = m.transpose(1, 2)[live]
    lse[iq[live]] = torch.where(l > 0, full_lse, torch.full_like(l, math.inf)).transpose(1, 2)[live]
    return out, top, lse


def _rows(s, table):
    """fp32 rows [..., pages * page, latent + 64] of the pages in `table`; those of a negative page are zero."""
    d, tile, n, slots = LAYOUTS[s["case"]["layout"]]
    page, row = s["case"]["page"], LAYOUTS[s["case"]["layout"]][0] + 128
    got = s["arena"][table.clamp_min(0).long()]
    body = got[..., : page * row].reshape(*table.shape, page, row)
    scale = got[..., page * row: page * (row + slots)].reshape(*table.shape, page, slots)[..., :n]
    latent = body[..., :d].contiguous().view(torch.float8_e4m3fn).float().view(*table.shape, page, n, tile)
    latent = (latent * torch.exp2(scale.float() - 127.0)[..., None]).reshape(*table.shape, page, d).bfloat16().float()
    rope = body[..., d:].contiguous().view(torch.bfloat16).float()
    full = torch.cat([latent, rope], -1)
    return full.reshape(*table.shape[:-1], table.size(-1) * page, d + 64)


def _plain_shared(s):
    b, s_q, h_q, d_qk = s["q"].shape
    q = s["q"].float() * s["scale"]
    pre, mine = _rows(s, s["prefix_table"]), _rows(s, s["table"])
    x = torch.matmul(q.view(b * s_q * h_q, d_qk), pre.t()).view(b, s_q * h_q, -1)
    x = x.masked_fill(torch.arange(pre.size(0), device=DEV) >= s["prefix_length"], -math.inf)
    y = torch.matmul(q.view(b, s_q * h_q, d_qk), mine.transpose(1, 2)).view(b, s_q, h_q, -1)
    sees = s["suffix"].view(b, 1, 1, 1) - (s_q - 1 - torch.arange(s_q, device=DEV)).view(1, s_q, 1, 1)
    y = y.masked_fill(torch.arange(y.size(-1), device=DEV) >= sees, -math.inf).view(b, s_q * h_q, -1)
    n = x.size(-1)
    x = torch.cat([x, y], -1)
    m = x.amax(-1, keepdim=True)
    x = (x - m.clamp_min(-1e30)).exp()
    l = x.sum(-1)
    o = torch.matmul(x[..., :n].reshape(b * s_q * h_q, n), pre[:, :512]).view(b, s_q * h_q, 512) + torch.matmul(x[..., n:], mine[..., :512])
    l, m, o = l.view(b, s_q, h_q), m.view(b, s_q, h_q), o.view(b, s_q, h_q, 512)
    lse = m + l.log()
    if s["sink"] is not None:
        lse = torch.logaddexp(lse, s["sink"].expand_as(lse))
    weight = torch.where(l > 0, (m - lse).exp(), torch.zeros_like(l))
    return (o * weight[..., None]).bfloat16(), lse.transpose(1, 2).contiguous()


# --------------------------------------------------------------------------- the least work
def work(case):
    if case["op"] == "slots":
        cached, new = _slot_lens(case)
        touched = sum(_pages(c + n, case["page"]) - c // case["page"] for c, n in zip(cached, new))
        return {"bytes": 16 * case["b"] + 8 * touched + 12 * (_pages(max(sum(new), 1), 64) * 64), "flops": sum(new) * 4}
    if case["op"] == "indices":
        n = sum(_lens(case)) * case["topk"]
        return {"bytes": 8 * n + 4 * sum(_pages(k + case["ctx"], case["page"]) for k in _lens(case)), "flops": 3 * n}
    if case["op"] == "prefill":
        ql, kl = _prefill_lens(case)
        pairs = 0
        for a, c in zip(ql, kl):
            pairs += a * (c - a) + a * (a + 1) // 2 if case["causal"] else a * c
        tq, tk = sum(ql), sum(kl)
        return {"bytes": 2 * (tq * case["h_q"] * (case["d_qk"] + case["d_v"]) + tk * case["h_kv"] * (case["d_qk"] + case["d_v"])) + 8 * tq * case["h_q"],
                "flops": pairs * case["h_q"] * 2 * (case["d_qk"] + case["d_v"])}
    d, _, _, slots = LAYOUTS[case["layout"]]
    suffix = _spread(case["mix"], case["b"], case["suffix"])
    rows = case["b"] * case["s_q"] * case["h_q"]
    return {"bytes": (case["prefix"] + sum(suffix)) * (d + 128 + slots) + rows * (2 * (d + 64) + 2 * 512 + 4),
            "flops": 2 * (d + 64 + 512) * case["h_q"] * case["s_q"] * (case["b"] * case["prefix"] + sum(suffix))}


# --------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    if case["op"] in ("slots", "indices"):
        return None
    s = prepare(case, seed)
    return _exact_prefill(s) if case["op"] == "prefill" else _exact_shared(s)


def _softmax64(x, sink):
    """Rows of logits in 64 bits -> weights (the sink among the sum), the largest logit, log of the sum without and with the sink."""
    if x.size(-1) == 0:
        x = torch.full((*x.shape[:-1], 1), -math.inf, dtype=torch.float64, device=DEV)
        top = x[..., 0]
        lse = top
    else:
        top, lse = x.amax(-1), torch.logsumexp(x, -1)
    both = lse if sink is None else torch.logaddexp(lse, sink.double().expand_as(lse))
    w = torch.where(torch.isfinite(lse)[..., None], torch.exp(x - torch.where(torch.isfinite(both), both, torch.zeros_like(both))[..., None]), torch.zeros_like(x))
    return w, top, lse, both


def _exact_prefill(s):
    tq, h_q, _ = s["q"].shape
    g = h_q // s["k"].size(1)
    out = torch.zeros(tq, h_q, s["v"].size(2), dtype=torch.float64, device=DEV)
    top = torch.full((tq, h_q), -math.inf, dtype=torch.float64, device=DEV)
    lse = torch.full((tq, h_q), math.inf, dtype=torch.float64, device=DEV)
    cu_q, cu_k = s["cu_q"].tolist(), s["cu_k"].tolist()
    for n in range(len(cu_q) - 1):
        q0, q1, k0, k1 = cu_q[n], cu_q[n + 1], cu_k[n], cu_k[n + 1]
        ban = None
        if s["case"]["causal"]:
            ban = torch.ones(q1 - q0, k1 - k0, dtype=torch.bool, device=DEV).triu((k1 - k0) - (q1 - q0) + 1)
        for h in range(h_q):
            x = s["scale"] * (s["q"][q0:q1, h].double() @ s["k"][k0:k1, h // g].double().t())
            if ban is not None:
                x = x.masked_fill(ban, -math.inf)
            w, t, e, _ = _softmax64(x, None if s["sink"] is None else s["sink"][h])
            out[q0:q1, h] = w[:, : k1 - k0] @ s["v"][k0:k1, h // g].double()
            top[q0:q1, h] = t
            lse[q0:q1, h] = torch.where(torch.isfinite(e), e, torch.full_like(e, math.inf))
    return out, top, lse


def _rows64(s, page_ids, count):
    """The first `count` tokens of a list of pages, in 64 bits, from the bits of their e4m3 codes."""
    d, tile, n, slots = LAYOUTS[s["case"]["layout"]]
    page, row = s["case"]["page"], d + 128
    tok = torch.arange(count, device=DEV)
    ids, at = page_ids.long()[tok // page], (tok % page)[:, None]
    code = s["arena"][ids[:, None], at * row + torch.arange(d, device=DEV)].int()
    e, f = (code >> 3) & 15, (code & 7).double()
    size = torch.where(e > 0, (1 + f / 8) * torch.pow(2.0, e.double() - 7), f / 8 * 2.0 ** -6)
    latent = torch.where(code > 127, -size, size)
    sc = s["arena"][ids[:, None], page * row + at * slots + torch.arange(n, device=DEV)].double()
    latent = latent * torch.pow(2.0, sc - 127).repeat_interleave(tile, 1)
    halves = s["arena"][ids[:, None], at * row + d + torch.arange(128, device=DEV)].int().view(count, 64, 2)
    rope = ((halves[..., 0] | (halves[..., 1] << 8)) << 16).view(torch.float32).double()
    return torch.cat([latent, rope], 1)


def _exact_shared(s):
    b, s_q, h_q, d_qk = s["q"].shape
    n = int(s["prefix_length"])
    pre = _rows64(s, s["prefix_table"], n)
    out = torch.zeros(b, s_q, h_q, 512, dtype=torch.float64, device=DEV)
    lse = torch.zeros(b, h_q, s_q, dtype=torch.float64, device=DEV)
    for r, k in enumerate(s["suffix"].tolist()):
        mine = _rows64(s, s["table"][r], k)
        for t in range(s_q):
            rows = torch.cat([pre, mine[: max(0, k - (s_q - 1 - t))]])
            w, _, _, both = _softmax64(s["scale"] * (s["q"][r, t].double() @ rows.t()), s["sink"])
            out[r, t] = w[:, : rows.size(0)] @ rows[:, :512]
            lse[r, :, t] = both
    return out, lse
