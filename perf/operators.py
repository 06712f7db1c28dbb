"""The paged key/value cache and the attention that reads it, as cases to time and to compare.

Four operators of a program that serves a quantized model: the page tables of a batch, built on the device from its
requests' lengths; the append of new key and value rows to the cache; attention over the cache, causal, optionally with a
sliding window and a few first tokens that stay visible; and attention for a batch that shares a long prefix. Head counts
are those of the benchmark's layers (hidden 4096 as 32 heads of 128, k and v of 1024 as 8 heads) and generic ones.

run() computes them in plain torch operations, or through tcb_amd.QuantBackend where `own` is true.
"""
import math

import torch

own = False

DEV = "cuda:0"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# padded score elements of the largest plain pass, and cache elements (k and v together) of the largest cache
MOST_SCORES = 1 << 31
MOST_CACHE = 1_900_000_000


def listed():
    heads = dict(q_heads=32, kv_heads=8, dim=128)
    return [
        # a decode step of sixteen chats: one token each, a page now and then; nothing but latency
        dict(name="tables 16 tokens", kind="tables", reqs=16, prompts=0, new=1, old=2000, page=16, spare=64),
        # a server that takes in a thousand requests at once, prompts of every length among them
        dict(name="tables 1024 prompts", kind="tables", reqs=1024, prompts=700, new=511, old=4000, page=32, spare=9000),
        # the fp32 k and v rows of a merged qkv product of sixteen tokens into a bf16 cache
        dict(name="append 16 tokens", kind="append", src="f32", dtype="bf16", tokens=16, page=16, pages=2048, **heads),
        # a prompt of 8192 tokens with 16-bit rows
        dict(name="append prompt 8192", kind="append", src="bf16", dtype="bf16", tokens=8192, page=32, pages=1024, **heads),
        # the smallest attention: one chat, one token, a short history
        dict(name="token 1 x 300", kind="attn", dtype="bf16", reqs=1, prompts=0, new=1, kv=300, page=16, window=0, sinks=0, **heads),
        # ordinary serving: 64 chats of every length up to 8192, one token each
        dict(name="tokens 64 x 8192", kind="attn", dtype="bf16", reqs=64, prompts=0, new=1, kv=8192, page=16, window=0, sinks=0, **heads),
        # one chat over a very long history: the split along the keys
        dict(name="token 1 x 131071", kind="attn", dtype="f16", reqs=1, prompts=0, new=1, kv=131071, page=64, window=0, sinks=0, **heads),
        # streaming chats with a window and sinks, other head counts
        dict(name="tokens 48 window 1000", kind="attn", dtype="f16", reqs=48, prompts=0, new=1, kv=20000, page=32, window=1000, sinks=4,
             q_heads=24, kv_heads=4, dim=64),
        # a long prompt, causal: matrix products
        dict(name="prompt 8192", kind="attn", dtype="bf16", reqs=1, prompts=1, new=8192, kv=8192, page=32, window=0, sinks=0, **heads),
        # a server's mixed step: ragged prompt chunks behind a cached history and token steps of other chats, windowed
        dict(name="mixed window 1024", kind="attn", dtype="bf16", reqs=40, prompts=8, new=901, kv=6001, page=16, window=1024, sinks=4, **heads),
        # a batch behind one system prompt, a token each
        dict(name="shared 32 x 4096", kind="shared", dtype="bf16", reqs=32, new=1, prefix=4096, suffix=300, page=16, **heads),
        # many samples of one long document, two tokens each, a prefix that ends inside a page
        dict(name="shared 192 x 30001", kind="shared", dtype="f16", reqs=192, new=2, prefix=30001, suffix=700, page=32, **heads),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["tables", "append", "attn", "attn", "attn", "shared", "shared"])
    page = rng.choice([16, 16, 32, 64, 128])
    if kind == "tables":
        reqs = _log_int(rng, 1, 2000)
        return dict(kind=kind, reqs=reqs, prompts=rng.choice([0, rng.randint(0, reqs)]), new=_log_int(rng, 1, 900),
                    old=_log_int(rng, 1, 9000), page=page, spare=_log_int(rng, 16, 20000))
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    shape = dict(q_heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 6, 8]), kv_heads=kv_heads, dim=rng.choice([64, 96, 128, 128, 128, 256]))
    row = kv_heads * shape["dim"]
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "append":
        tokens = _log_int(rng, 1, 8192)
        return dict(kind=kind, src=rng.choice(["f32", dtype]), dtype=dtype, tokens=tokens, page=page,
                    pages=-(-tokens // page) + rng.randint(1, 2000), **shape)
    if kind == "shared":
        reqs, new = _log_int(rng, 2, 256), rng.choice([1, 1, 1, 2, 4])
        prefix = min(_log_int(rng, 256, 32768), MOST_SCORES // (4 * reqs * new * shape["q_heads"]))
        suffix = min(_log_int(rng, new, 1500), MOST_CACHE // (4 * reqs * row))
        return dict(kind=kind, dtype=dtype, reqs=reqs, new=new, prefix=prefix, suffix=max(new, suffix), page=page, **shape)
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    sinks = rng.choice([0, 4, rng.randint(1, 100)]) if window else 0
    how = rng.choice(["token", "token", "prompt", "mixed"])
    reqs = _log_int(rng, 1, 128) if how != "prompt" else rng.randint(1, 6)
    prompts = {"token": 0, "prompt": reqs, "mixed": rng.randint(1, min(reqs, 8))}[how]
    new = 1 if how == "token" else _log_int(rng, 2, 8192)
    kv = _log_int(rng, 16, 131072 if reqs < 4 else 16384)
    kv = max(1, min(kv, MOST_CACHE // (4 * reqs * row)))
    if prompts:
        kv = min(kv, MOST_SCORES // (4 * prompts * shape["q_heads"]))
        new = max(1, min(new, kv, 64 * MOST_SCORES // (shape["dim"] * prompts * shape["q_heads"] * kv)))
    return dict(kind=kind, dtype=dtype, reqs=reqs, prompts=prompts, new=new, kv=kv, page=page, window=window, sinks=sinks, **shape)


# ---- lengths: ragged, the same for every seed (a case's work follows from the case), the first request the longest ----

def _ragged(most, n, step):
    """n lengths in 1..most, the first `most` itself, the others spread evenly."""
    return [max(1, math.ceil(most * (1.0 - (i * step) % 1.0))) for i in range(n)]


def _lengths(case):
    """(new tokens, cached and new tokens) of each request: the first `prompts` bring up to `new`, the others one token."""
    reqs, prompts = case["reqs"], case["prompts"]
    new = _ragged(case["new"], prompts, 0.3819660113) + [1] * (reqs - prompts)
    if case["kind"] == "tables":
        old = [o - 1 for o in _ragged(case["old"], reqs, 0.6180339887)]
        return new, [o + n for o, n in zip(old, new)]
    return new, [max(n, k) for n, k in zip(new, _ragged(case["kv"], reqs, 0.6180339887))]


def _pages(kv, page):
    return [-(-k // page) for k in kv]


# ---- inputs --------------------------------------------------------------------------------------------------------

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) & 0x7FFFFFFF)
    return g


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _randn(shape, seed, dtype):
    return torch.randn(shape, generator=_gen(seed), device=DEV, dtype=dtype)


class State:
    kv = None  # the framework's descriptor of the cache, made by the first pass

    def __init__(self, case):
        self.case = case


def _table(pages, total, seed):
    """Page numbers of every request in a shuffled pool of `total`, rows padded with -1."""
    order = torch.randperm(total, generator=_gen(seed), device=DEV).to(torch.int32)
    starts, most = [0], max(pages)
    for p in pages:
        starts.append(starts[-1] + p)
    j, counts = torch.arange(most, device=DEV), _ints(pages)
    at = _ints(starts[:-1]).long().unsqueeze(1) + j
    return torch.where(j < counts.unsqueeze(1), order[at.clamp(max=total - 1)], -1).to(torch.int32).contiguous(), order, starts[-1]


def prepare(case, seed):
    s, kind, page = State(case), case["kind"], case["page"]
    if kind == "tables":
        new, kv = _lengths(case)
        old = [k - n for k, n in zip(kv, new)]
        have, need = _pages(old, page), _pages(kv, page)
        s.old, s.add, s.most = _ints(old), _ints(new), max(need) + 1
        # a pool of all pages in use and enough free ones, in the order in which a program gave them back
        total = sum(have) + max(case["spare"], sum(need) - sum(have))
        s.table, order, used = _table([max(h, 1) for h in have], total + len(have), seed)
        s.table = torch.nn.functional.pad(s.table, (0, s.most - s.table.shape[1]), value=-1).contiguous()
        s.table[torch.arange(s.most, device=DEV) >= _ints(have).unsqueeze(1)] = -1
        s.free = order[used:].clone() if order[used:].numel() else torch.zeros(1, dtype=torch.int32, device=DEV)
        s.nfree = order.numel() - used
        s.n = sum(new) + 7  # a buffer a little larger than the step
        s.outs = [s.table, torch.empty(len(new) + 1, dtype=torch.int32, device=DEV), torch.empty(len(new), dtype=torch.int32, device=DEV),
                  torch.empty(s.n, dtype=torch.int32, device=DEV), torch.empty(1, dtype=torch.int32, device=DEV)]
        torch.cuda.synchronize()
        return s
    hk, hq, d, t = case["kv_heads"], case["q_heads"], case["dim"], TYPES[case["dtype"]]
    if kind == "append":
        s.rows = _randn((case["tokens"], (hq + 2 * hk) * d), seed * 31, TYPES[case["src"]])
        s.k, s.v = (torch.zeros((case["pages"], hk, page, d), dtype=t, device=DEV) for _ in range(2))
        s.slots = torch.randperm(case["pages"] * page, generator=_gen(seed * 31 + 1), device=DEV)[:case["tokens"]].to(torch.int32)
        if case["tokens"] > 1:  # consecutive places of shuffled pages, as the tables give them
            order = torch.randperm(case["pages"], generator=_gen(seed * 31 + 1), device=DEV)
            i = torch.arange(case["tokens"], device=DEV)
            s.slots = (order[i // page] * page + i % page).to(torch.int32)
        torch.cuda.synchronize()
        return s
    if kind == "attn":
        s.new, s.lens = _lengths(case)
        counts = _pages(s.lens, page)
    else:
        s.new = [case["new"]] * case["reqs"]
        s.lens = [max(case["new"], n) for n in _ragged(case["suffix"], case["reqs"], 0.6180339887)]
        counts = _pages(s.lens, page) + _pages([case["prefix"]], page)
    total = sum(counts) + 3
    s.table, _, _ = _table(counts, total, seed * 31)
    if kind == "shared":
        s.prefix = s.table[-1, :counts[-1]].clone()
        s.table = s.table[:-1, :max(counts[:-1])].clone()
    starts = [0]
    for n in s.new:
        starts.append(starts[-1] + n)
    s.tokens = starts[-1]
    s.q_start, s.kv_len = _ints(starts), _ints(s.lens)
    s.k, s.v = (_randn((total, hk, page, d), seed * 31 + i, t) for i in (1, 2))
    # rows of a merged qkv product; some heads look sharply at few keys, as in trained models
    s.rows = _randn((s.tokens, (hq + 2 * hk), d), seed * 31 + 3, t)
    s.rows *= torch.linspace(0.25, 2.0, hq + 2 * hk, device=DEV).to(t).unsqueeze(1)
    s.rows = s.rows.view(s.tokens, -1)
    s.out = torch.empty((s.tokens, hq * d), dtype=t, device=DEV)
    torch.cuda.synchronize()
    return s


# ---- the operators in plain form ------------------------------------------------------------------------------------

def _plain_tables(s):
    page, most = s.case["page"], s.most
    old, add = s.old.long(), s.add.long()
    have, need = (old + page - 1) // page, (old + add + page - 1) // page
    grow = torch.where(need <= most, need - have, 0)
    base = grow.cumsum(0) - grow
    fits = (need <= most) & ((grow == 0) | (base + grow <= s.nfree))
    j = torch.arange(most, device=DEV)
    fresh = fits.unsqueeze(1) & (j >= have.unsqueeze(1)) & (j < need.unsqueeze(1))
    at = (base.unsqueeze(1) + j - have.unsqueeze(1)).clamp(0, s.free.numel() - 1)
    table, q_start, kv_len, slots, used = s.outs
    table.copy_(torch.where(fresh, s.free[at], table))
    q_start[0] = 0
    q_start[1:] = add.cumsum(0)
    kv_len.copy_(old + torch.where(fits, add, 0))
    t = torch.arange(s.n, device=DEV)
    r = torch.searchsorted(q_start[1:].long(), t, right=True).clamp(max=old.numel() - 1)
    pos = old[r] + t - q_start[r]
    slot = table[r, (pos // page).clamp(max=most - 1)].long() * page + pos % page
    slots.copy_(torch.where((t < q_start[-1]) & fits[r], slot, -1))
    used[0] = torch.where(fits, base + grow, 0).amax()
    return s.outs


def _plain_append(s):
    case = s.case
    hk, hq, d, page = case["kv_heads"], case["q_heads"], case["dim"], case["page"]
    rows = s.rows.view(case["tokens"], hq + 2 * hk, d)
    p, i = (s.slots // page).long(), (s.slots % page).long()
    s.k[p, :, i] = rows[:, hq:hq + hk].to(s.k.dtype)
    s.v[p, :, i] = rows[:, hq + hk:].to(s.v.dtype)
    return [s.k, s.v]


def _cached(c, table, n):
    """Rows of the cache in order, fp32 [requests, heads, n, dim]."""
    g = c[table.clamp(min=0).long()].float()
    r, p, h, page, d = g.shape
    return g.permute(0, 2, 1, 3, 4).reshape(r, h, p * page, d)[:, :, :n]


def _visible(pos, kv, n, window, sinks):
    """Whether the query at pos [requests, new] sees key j < n."""
    j, p = torch.arange(n, device=DEV), pos.unsqueeze(2)
    see = (j <= p) & (j < kv.view(-1, 1, 1))
    if window:
        see &= (j > p - window) | (j < sinks)
    return see


def _queries(s, first, count, most):
    """Query rows of `count` requests padded to `most` tokens, fp32 [requests, kv heads, group, tokens, dim], and their tokens."""
    case = s.case
    hk, hq, d = case["kv_heads"], case["q_heads"], case["dim"]
    start, new = s.q_start[first:first + count].long(), s.q_start[first + 1:first + count + 1].long()
    at = start.unsqueeze(1) + torch.arange(most, device=DEV)
    real = at < new.unsqueeze(1)
    q = s.rows[at.clamp(max=s.tokens - 1)].view(count, most, hq + 2 * hk, d)[:, :, :hq].float()
    return q.view(count, most, hk, hq // hk, d).permute(0, 2, 3, 1, 4), at, real, new - start


def _plain_attn_group(s, first, count):
    if not count:
        return
    case = s.case
    most, n = max(s.new[first:first + count]), max(s.lens[first:first + count])
    q, at, real, new = _queries(s, first, count, most)
    kv = s.kv_len[first:first + count].long()
    pages = -(-n // case["page"])
    k, v = (_cached(c, s.table[first:first + count, :pages], n) for c in (s.k, s.v))
    r, hk, g, m, d = q.shape
    x = torch.matmul((q * d ** -0.5).reshape(r, hk, g * m, d), k.transpose(2, 3)).view(r, hk, g, m, n)
    pos = (kv - new).unsqueeze(1) + torch.arange(most, device=DEV)
    see = _visible(pos, kv, n, case["window"], case["sinks"]).view(r, 1, 1, m, n)
    x.masked_fill_(~see, -math.inf)
    x.sub_(x.amax(4, keepdim=True).clamp(min=-1e30)).exp_()
    total = x.sum(4, keepdim=True)
    y = torch.matmul(x.view(r, hk, g * m, n), v).view(r, hk, g, m, d) / total
    y = y.permute(0, 3, 1, 2, 4).reshape(r, m, hk * g * d)
    s.out[at[real]] = y[real].to(s.out.dtype)


def _plain_shared(s):
    case = s.case
    most, n, pre = case["new"], max(s.lens), case["prefix"]
    q, at, real, new = _queries(s, 0, case["reqs"], most)
    r, hk, g, m, d = q.shape
    q = q * d ** -0.5
    kp, vp = (_cached(c, s.prefix.unsqueeze(0), pre)[0] for c in (s.k, s.v))
    k, v = (_cached(c, s.table, n) for c in (s.k, s.v))
    x0 = torch.matmul(q.permute(1, 0, 2, 3, 4).reshape(hk, r * g * m, d), kp.transpose(1, 2)).view(hk, r, g, m, pre)
    x1 = torch.matmul(q.reshape(r, hk, g * m, d), k.transpose(2, 3)).view(r, hk, g, m, n).permute(1, 0, 2, 3, 4)
    kv = s.kv_len.long()
    see = _visible((kv - new).unsqueeze(1) + torch.arange(most, device=DEV), kv, n, 0, 0)
    x1 = x1.masked_fill(~see.view(1, r, 1, m, n), -math.inf)
    top = torch.maximum(x0.amax(4, keepdim=True), x1.amax(4, keepdim=True))
    x0, x1 = x0.sub_(top).exp_(), (x1 - top).exp_()
    total = x0.sum(4, keepdim=True) + x1.sum(4, keepdim=True)
    y = torch.matmul(x0.view(hk, r * g * m, pre), vp).view(hk, r, g, m, d)
    y = y + torch.matmul(x1.permute(1, 0, 2, 3, 4).reshape(r, hk, g * m, n), v).view(r, hk, g, m, d).permute(1, 0, 2, 3, 4)
    y = (y / total).permute(1, 3, 0, 2, 4).reshape(r, m, hk * g * d)
    s.out[at[real]] = y[real].to(s.out.dtype)
    return s.out


def _plain(s):
    kind = s.case["kind"]
    if kind == "attn":
        _plain_attn_group(s, 0, s.case["prompts"])
        _plain_attn_group(s, s.case["prompts"], s.case["reqs"] - s.case["prompts"])
        return s.out
    return {"tables": _plain_tables, "append": _plain_append, "shared": _plain_shared}[kind](s)


# ---- the framework's operators ---------------------------------------------------------------------------------------

_backend = []


def _tb():
    if not _backend:
        from tcb_amd import QuantBackend
        _backend.append(QuantBackend(0))
    return _backend[0]


def run(s):
    if not own:
        return _plain(s)
    import tcb_amd
    tb, case, io = _tb(), s.case, {"f16": tcb_amd.F16, "bf16": tcb_amd.BF16, "f32": tcb_amd.F32}
    if case["kind"] == "tables":
        table, q_start, kv_len, slots, used = s.outs
        tb.PageTables(case["reqs"], case["page"], s.old.data_ptr(), s.add.data_ptr(), s.free.data_ptr(), s.nfree, table.data_ptr(), s.most,
                      q_start.data_ptr(), kv_len.data_ptr(), slots.data_ptr(), s.n, used.data_ptr())
        return s.outs
    hk, hq, d = case["kv_heads"], case["q_heads"], case["dim"]
    if s.kv is None:
        s.kv = tcb_amd.KVCache(io[case["dtype"]], s.k.shape[0], case["page"], hk, d, s.k.data_ptr(), s.v.data_ptr())
    row = (hq + 2 * hk) * d
    if case["kind"] == "append":
        k = s.rows.data_ptr() + hq * d * s.rows.element_size()
        tb.KVAppend(s.kv, case["tokens"], k, k + hk * d * s.rows.element_size(), io[case["src"]], row, s.slots.data_ptr())
        return [s.k, s.v]
    if case["kind"] == "attn":
        tb.Attention(s.kv, s.rows.data_ptr(), row, s.out.data_ptr(), hq * d, s.tokens, hq, case["reqs"], s.q_start.data_ptr(), s.kv_len.data_ptr(),
                     s.table.data_ptr(), s.table.shape[1], max_new=max(s.new), window=case["window"], sinks=case["sinks"])
    else:
        tb.AttentionShared(s.kv, s.rows.data_ptr(), row, s.out.data_ptr(), hq * d, s.tokens, hq, case["reqs"], s.q_start.data_ptr(),
                           s.kv_len.data_ptr(), s.table.data_ptr(), s.table.shape[1], s.prefix.data_ptr(), case["prefix"], max_new=case["new"])
    return s.out


# ---- what a pass cannot do without -------------------------------------------------------------------------------------

def _seen(new, kv, window, sinks):
    """(query-key pairs, keys that some query sees) of a request."""
    first = kv - new  # position of its first query
    if not window:
        return new * first + new * (new + 1) // 2, kv
    pairs = 0
    for p in range(first, kv):
        low = max(0, p - window + 1)
        pairs += p + 1 - low + min(sinks, low)
    low = max(0, first - window + 1)
    return pairs, kv - low + min(sinks, low)


def work(case):
    kind, page = case["kind"], case["page"]
    if kind == "tables":
        new, kv = _lengths(case)
        fresh = sum(_pages(kv, page)) - sum(_pages([k - n for k, n in zip(kv, new)], page))
        # lengths in and out, starts, the free pages taken and written into tables, one table entry read and one slot written per new token
        return {"bytes": 4 * (4 * len(new) + 2 * fresh + sum(_pages(new, page)) + sum(new) + 8), "flops": 2 * sum(new)}
    hk, hq, d = case["kv_heads"], case["q_heads"], case["dim"]
    if kind == "append":
        e = 4 if case["src"] == "f32" else 2
        return {"bytes": case["tokens"] * (2 * hk * d * (e + 2) + 4), "flops": 2 * case["tokens"] * hk * d}
    if kind == "attn":
        new, kv = _lengths(case)
        seen = [_seen(n, k, case["window"], case["sinks"]) for n, k in zip(new, kv)]
        pairs, keys, tokens = sum(p for p, _ in seen), sum(k for _, k in seen), sum(new)
    else:
        new = case["new"]
        kv = [max(new, n) for n in _ragged(case["suffix"], case["reqs"], 0.6180339887)]
        tokens = new * case["reqs"]
        pairs = tokens * case["prefix"] + sum(_seen(new, k, 0, 0)[0] for k in kv)
        keys = case["prefix"] + sum(kv)
    return {"bytes": 2 * (2 * keys * hk * d + 2 * tokens * hq * d) + 4 * (keys // page + 3 * case["reqs"]), "flops": 4 * pairs * hq * d}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------

def _softmax_rows(x, see):
    x = torch.where(see, x, torch.full_like(x, -math.inf))
    e = torch.exp(x - x.max(-1, keepdim=True).values)
    return e / e.sum(-1, keepdim=True)


def exact(case, seed):
    """Attention request by request and head by head; tables in integers on the host; None where nothing is rounded in between."""
    kind = case["kind"]
    if kind == "tables":
        return None
    s = prepare(case, seed)
    hk, hq, d, page = case["kv_heads"], case["q_heads"], case["dim"], case["page"]
    if kind == "append":
        places = s.slots.tolist()
        out = [s.k.double(), s.v.double()]
        at = torch.tensor(places, device=DEV)
        for which, c in enumerate(out):
            for h in range(hk):
                c[at.div(page, rounding_mode="floor"), h, at.remainder(page)] = \
                    s.rows[:, (hq + which * hk + h) * d:(hq + which * hk + h + 1) * d].double()
        return out
    out = torch.zeros((s.tokens, hq * d), dtype=torch.float64, device=DEV)
    window, sinks = case.get("window", 0), case.get("sinks", 0)
    pre = case.get("prefix", 0)
    lead = [[], []]
    if pre:  # the prefix's rows before everybody's own
        lead = [c[s.prefix.long()].double().transpose(1, 2).reshape(-1, hk, d)[:pre] for c in (s.k, s.v)]
    t0 = 0
    for i, (n, own_len) in enumerate(zip(s.new, s.lens)):
        k, v = (c[s.table[i, :-(-own_len // page)].long()].double().transpose(1, 2).reshape(-1, hk, d)[:own_len] for c in (s.k, s.v))
        if pre:
            k, v = torch.cat([lead[0], k]), torch.cat([lead[1], v])
        length = pre + own_len
        j, p = torch.arange(length, device=DEV), torch.arange(length - n, length, device=DEV).unsqueeze(1)
        see = j <= p
        if window:
            see = see & ((p - j < window) | (j < sinks))
        q = s.rows[t0:t0 + n].double().view(n, -1, d)
        for h in range(hq if n > 8 else 0):
            w = _softmax_rows(q[:, h] @ k[:, h * hk // hq].t() / math.sqrt(d), see)
            out[t0:t0 + n, h * d:(h + 1) * d] = w @ v[:, h * hk // hq]
        if n <= 8:  # few rows: all heads of a kv head at once
            qs = q[:, :hq].reshape(n, hk, hq // hk, d).permute(1, 0, 2, 3).reshape(hk, -1, d)
            x = torch.bmm(qs, k.permute(1, 2, 0).contiguous()) / math.sqrt(d)
            w = _softmax_rows(x, see.repeat_interleave(hq // hk, 0).unsqueeze(0))
            y = torch.bmm(w, v.permute(1, 0, 2).contiguous()).view(hk, n, hq // hk, d)
            out[t0:t0 + n] = y.permute(1, 0, 2, 3).reshape(n, hq * d)
        t0 += n
    return out
