"""The rest of a token step around the quantized products, as cases to time and to compare.

Four operators of a program that serves a quantized model: rotary positions (one axis for text; time, height and width for images and
video) on the q and k heads of a merged product's rows; a paged key/value cache held in 4 bits, written and read back; causal
attention over that cache, with grouped heads, a sliding window and a few first tokens that stay visible; and the choice of a
token from the head's logits by temperature, top-k, top-p and min-p. Head counts and vocabulary are those of the benchmark's layers
(hidden 4096 as 32 heads of 128, k and v of 1024 as 8 heads, vocabulary 128256) and generic ones.

run() computes them in plain torch operations, or through tcb_amd.QuantBackend where `own` is true.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
# padded score elements of the largest plain pass, and cache elements (k and v together) of the largest cache
MOST_SCORES = 1 << 31
MOST_CACHE = 1_200_000_000
MOST_LOGITS = 256 * 128256


def listed():
    heads = dict(q_heads=32, kv_heads=8, dim=128)
    rope = dict(base=500000.0, neighbours=False, dealt=False, ladders=False, factors=False)
    return [
        # positions of a decode step of sixteen chats: latency
        dict(name="rope 16 tokens", kind="rope", dtype="bf16", tokens=16, pairs="64", far=100000, **rope, **heads),
        # a prompt of images and text, three axes, rows of the merged product in bf16: every element once
        dict(name="rope images 8192", kind="rope", dtype="bf16", tokens=8192, pairs="24 20 20", far=20000, **heads,
             base=1000000.0, neighbours=False, dealt=True, ladders=False, factors=True),
        # the fp32 k and v rows of a merged qkv product of sixteen tokens into the 4-bit cache, and back
        dict(name="cache 16 tokens", kind="cache", dtype="f32", tokens=16, page=16, pages=2048, **heads),
        # a prompt's 16-bit rows
        dict(name="cache prompt 8192", kind="cache", dtype="bf16", tokens=8192, page=32, pages=1024, **heads),
        # the smallest attention: one chat, one token, a short history
        dict(name="token 1 x 300", kind="attn", dtype="bf16", reqs=1, prompts=0, new=1, kv=300, page=16, window=0, sinks=0, **heads),
        # ordinary serving: 64 chats of every length up to 8192, one token each
        dict(name="tokens 64 x 8192", kind="attn", dtype="bf16", reqs=64, prompts=0, new=1, kv=8192, page=16, window=0, sinks=0, **heads),
        # one chat over a very long history: the split along the keys
        dict(name="token 1 x 131071", kind="attn", dtype="f16", reqs=1, prompts=0, new=1, kv=131071, page=64, window=0, sinks=0, **heads),
        # a long prompt, causal: matrix products
        dict(name="prompt 8192", kind="attn", dtype="bf16", reqs=1, prompts=1, new=8192, kv=8192, page=32, window=0, sinks=0, **heads),
        # a server's mixed step: ragged prompt chunks behind a cached history and token steps of other chats, windowed, other head counts
        dict(name="mixed window 1000", kind="attn", dtype="f16", reqs=40, prompts=8, new=901, kv=6001, page=32, window=1000, sinks=4,
             q_heads=24, kv_heads=4, dim=64),
        # one chat's next token, the usual settings
        dict(name="sample 1 x 128256", kind="sample", dtype="f32", rows=1, vocab=128256, how="usual"),
        # sixteen chats, half of which have switched a filter off, in another vocabulary and 16 bits (many equal logits)
        dict(name="sample 16 x 151936", kind="sample", dtype="bf16", rows=16, vocab=151936, how="mixed"),
        # a large batch, every setting there is, from certain rows to flat ones
        dict(name="sample 256 x 128256", kind="sample", dtype="f32", rows=256, vocab=128256, how="mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "cache", "attn", "attn", "attn", "sample", "sample"])
    if kind == "sample":
        vocab = _log_int(rng, 500, 200000)
        return dict(kind=kind, dtype=rng.choice(["f32", "f32", "f16", "bf16"]), vocab=vocab,
                    rows=_log_int(rng, 1, min(256, MOST_LOGITS // vocab)), how=rng.choice(["usual", "mixed"]))
    page = rng.choice([16, 16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    shape = dict(q_heads=kv_heads * rng.choice([1, 2, 4, 4, 5, 6, 8]), kv_heads=kv_heads, dim=rng.choice([64, 96, 128, 128, 128, 192, 256]))
    row = kv_heads * shape["dim"]
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "rope":
        axes, half = rng.choice([1, 1, 2, 3, 3]), shape["dim"] // 2
        each = max(1, (half if rng.random() < 0.7 else half // 2) // axes)
        pairs = [each] * axes
        pairs[0] += rng.randint(0, half - each * axes)
        width = (shape["q_heads"] + shape["kv_heads"]) * shape["dim"]
        return dict(kind=kind, dtype=rng.choice(["f32", dtype]), tokens=_log_int(rng, 1, min(8192, 8192 * 2560 // width)), pairs=" ".join(map(str, pairs)),
                    far=_log_int(rng, 100, 1000000), base=rng.choice([10000.0, 500000.0, 1000000.0]), neighbours=rng.random() < 0.4,
                    dealt=rng.random() < 0.4, ladders=rng.random() < 0.3, factors=rng.random() < 0.3, **shape)
    if kind == "cache":
        tokens = _log_int(rng, 1, 8192 * 1024 // max(row, 1024))
        return dict(kind=kind, dtype=rng.choice(["f32", dtype]), tokens=tokens, page=page, pages=-(-tokens // page) + rng.randint(1, 1000), **shape)
    window = rng.choice([0, 0, _log_int(rng, 16, 4096)])
    sinks = rng.choice([0, 4, rng.randint(1, 100)]) if window else 0
    how = rng.choice(["token", "token", "few", "prompt", "mixed"])
    reqs = _log_int(rng, 1, 128) if how != "prompt" else rng.randint(1, 6)
    prompts = {"token": 0, "few": reqs, "prompt": reqs, "mixed": rng.randint(1, min(reqs, 8))}[how]
    new = 1 if how == "token" else rng.randint(2, 24) if how == "few" else _log_int(rng, 2, 8192)
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
    return new, [max(n, k) for n, k in zip(new, _ragged(case["kv"], reqs, 0.6180339887))]


def _pages(kv, page):
    return [-(-k // page) for k in kv]


def _pairs(case):
    """Pairs that each axis turns."""
    return [int(n) for n in case["pairs"].split()]


def _axes(case):
    """The axis of every pair and its place in that axis's ladder."""
    each, axis, place = _pairs(case), [], []
    left = list(each)
    a = 0
    for _ in range(sum(left)):
        while left[a] == 0:
            a = (a + 1) % len(left)
        axis.append(a)
        place.append(each[a] - left[a])
        left[a] -= 1
        if case["dealt"]:
            a = (a + 1) % len(left)
    return axis, place


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
    kv = spec = None  # the framework's descriptors of the cache and of the axes, made by the first pass

    def __init__(self, case):
        self.case = case


# The cache's planes [page][head][sixteen rows][9 * dim bytes]: codes, then scales (include/trhip.h). Nibble `at` of a dword of codes:
AT_K = [0, 4, 1, 5, 2, 6, 3, 7]                    # of eight elements in a row
AT_V = [[0, 1], [4, 5], [2, 3], [6, 7]]            # of two elements of four rows


def _quantise(x):
    """Codes 0..15 (uint8) and scales (f16, of a block of 32 elements) of rows [..., dim]."""
    b = x.float().unflatten(-1, (-1, 32))
    size = b.abs()
    first = torch.where(size == size.amax(-1, keepdim=True), torch.arange(32, device=DEV), 31).amin(-1, keepdim=True)
    m = b.gather(-1, first).squeeze(-1)
    part, e = torch.frexp(m.abs() * 0.125)
    unit = ((e - 5).clamp(min=-126) + 127).to(torch.int32).bitwise_left_shift(23).view(torch.float32)  # 2^(e - 5), to the last bit
    d = (torch.round(part * 32) * unit).clamp(max=7936.0).half()
    d = torch.where(m < 0, d, -d)
    whole = torch.round(b.double() / d.double().unsqueeze(-1)).clamp(-8, 7) + 8
    codes = torch.where((d == 0).unsqueeze(-1), 8.0, whole).to(torch.uint8)
    return codes.flatten(-2), d


def _pack(codes, scales, values):
    """A plane of codes [pages, heads, page, dim] and scales [pages, heads, page, dim / 32]."""
    pages, heads, page, dim = codes.shape
    t, n = page // 16, dim // 32
    if values:  # rows 4 q + i, elements 32 n + 2 r + s
        c = codes.view(pages, heads, t, 4, 4, n, 16, 2).permute(0, 1, 2, 3, 6, 5, 4, 7)
        order = [4 * 0 + 0] * 8
        for i in range(4):
            for s in range(2):
                order[AT_V[i][s]] = 2 * i + s
    else:  # rows r, elements 32 g + 8 q + i
        c = codes.view(pages, heads, t, 16, n, 4, 8).permute(0, 1, 2, 5, 3, 4, 6)
        order = [AT_K.index(at) for at in range(8)]
    nib = c.reshape(pages, heads, t, 16 * dim // 8, 8)[..., order]
    code_bytes = (nib[..., 0::2] | (nib[..., 1::2] << 4)).reshape(pages, heads, t, 8 * dim)
    s = scales.view(pages, heads, t, 4, 4, n).transpose(4, 5).reshape(pages, heads, t, 16 * n).contiguous().view(torch.uint8)
    return torch.cat([code_bytes, s], -1)


def _open(tiles, values):
    """Values, fp32 [..., rows, dim], of a plane's pieces [..., tiles, 9 * dim]."""
    lead, dim = tiles.shape[:-2], tiles.shape[-1] // 9
    t, n = tiles.shape[-2], dim // 32
    tiles = tiles.reshape(-1, t, 9 * dim)
    code = tiles[..., :8 * dim]
    nib = torch.stack([code & 15, code >> 4], -1)
    scale = tiles[..., 8 * dim:].contiguous().view(torch.float16).view(-1, t, 4, n, 4).float()  # rows 4 q + i of group n
    if values:
        c = nib.view(-1, t, 4, 16, n, 8)[..., sum(AT_V, [])].view(-1, t, 4, 16, n, 4, 2).permute(0, 1, 2, 5, 4, 3, 6).reshape(-1, t, 4, 4, n, 32)
    else:
        c = nib.view(-1, t, 4, 16, n, 8)[..., AT_K].permute(0, 1, 3, 4, 2, 5).reshape(-1, t, 4, 4, n, 32)
    return ((c.float() - 8) * scale.transpose(3, 4).unsqueeze(-1)).reshape(*lead, 16 * t, dim)


def _table(pages, total, seed):
    """Page numbers of every request in a shuffled pool of `total`, rows padded with -1."""
    order = torch.randperm(total, generator=_gen(seed), device=DEV).to(torch.int32)
    starts, most = [0], max(pages)
    for p in pages:
        starts.append(starts[-1] + p)
    j, counts = torch.arange(most, device=DEV), _ints(pages)
    at = _ints(starts[:-1]).long().unsqueeze(1) + j
    return torch.where(j < counts.unsqueeze(1), order[at.clamp(max=total - 1)], -1).to(torch.int32).contiguous()


def _prepare_sample(s, seed):
    case = s.case
    rows, vocab, g = case["rows"], case["vocab"], _gen(seed * 31)
    # logits as models give them: they fall with the logarithm of the rank, more or less steeply from row to row, with noise
    s.logits = torch.empty((rows, vocab), dtype=TYPES[case["dtype"]], device=DEV)
    steep = torch.rand(rows, generator=g, device=DEV) * 1.2 + 1.1
    for r in range(rows):
        rank = torch.randperm(vocab, generator=g, device=DEV).float() + 1.0
        s.logits[r] = (12.0 - steep[r] * rank.log() + 0.3 * torch.randn(vocab, generator=g, device=DEV)).to(s.logits.dtype)
    i = torch.arange(rows, device=DEV)
    if case["how"] == "usual":
        s.temperature, s.top_k = torch.full((rows,), 0.8, device=DEV), torch.full((rows,), 50, dtype=torch.int32, device=DEV)
        s.top_p, s.min_p = torch.full((rows,), 0.95, device=DEV), torch.full((rows,), 0.02, device=DEV)
    else:
        s.temperature = torch.where(i % 8 == 5, 0.0, 0.6 + 0.1 * (i % 7))
        s.top_k = torch.where(i % 2 == 0, 0, 20 + 7 * (i % 40)).to(torch.int32)
        s.top_p = torch.where(i % 4 == 2, 1.0, 0.85 + 0.02 * (i % 7))
        s.min_p = torch.where(i % 4 >= 2, 0.0, 0.01 * (i % 5))
    s.u = torch.rand(rows, generator=g, device=DEV)
    s.token, s.logprob = torch.empty(rows, dtype=torch.int32, device=DEV), torch.empty(rows, device=DEV)


def prepare(case, seed):
    s, kind = State(case), case["kind"]
    if kind == "sample":
        _prepare_sample(s, seed)
        torch.cuda.synchronize()
        return s
    hk, hq, d, t = case["kv_heads"], case["q_heads"], case["dim"], TYPES[case["dtype"]]
    row = (hq + 2 * hk) * d
    if kind == "rope":
        tokens = case["tokens"]
        s.rows = _randn((tokens, row), seed * 31, t)
        s.pos = torch.randint(0, case["far"], (len(_pairs(case)), tokens), generator=_gen(seed * 31 + 1), device=DEV, dtype=torch.int32)
        if len(_pairs(case)) == 1:  # text: places in a row, from anywhere
            s.pos = (s.pos[:, :1] + torch.arange(tokens, device=DEV)).to(torch.int32).contiguous()
        s.factors = None
        if case["factors"]:  # slow frequencies stretched, fast ones as they were
            s.factors = torch.linspace(1.0, 0.125, sum(_pairs(case)), device=DEV)
        s.out = torch.empty((tokens, (hq + hk) * d), dtype=t, device=DEV)
        torch.cuda.synchronize()
        return s
    page = case["page"]
    if kind == "cache":
        tokens, pages = case["tokens"], case["pages"]
        s.rows = _randn((tokens, row), seed * 31, t)
        order = torch.randperm(pages, generator=_gen(seed * 31 + 1), device=DEV)
        i = torch.arange(tokens, device=DEV)
        s.slots = (order[i // page] * page + i % page).to(torch.int32)
        s.k, s.v = (torch.zeros((pages, hk, page // 16, 9 * d), dtype=torch.uint8, device=DEV) for _ in range(2))
        s.back = torch.empty((2, tokens, hk * d), dtype=t, device=DEV)
        torch.cuda.synchronize()
        return s
    s.new, s.lens = _lengths(case)
    counts = _pages(s.lens, page)
    total = sum(counts) + 3
    s.table = _table(counts, total, seed * 31)
    starts = [0]
    for n in s.new:
        starts.append(starts[-1] + n)
    s.tokens = starts[-1]
    s.q_start, s.kv_len = _ints(starts), _ints(s.lens)
    s.k, s.v = (torch.empty((total, hk, page // 16, 9 * d), dtype=torch.uint8, device=DEV) for _ in range(2))
    some = max(1, (1 << 25) // (hk * page * d))
    for plane, i in ((s.k, 1), (s.v, 2)):
        for a in range(0, total, some):
            n = min(some, total - a)
            plane[a:a + n] = _pack(*_quantise(_randn((n, hk, page, d), seed * 31 + i + 10 * a, torch.float32)), i == 2)
    # rows of a merged qkv product; some heads look sharply at few keys, as in trained models
    s.rows = _randn((s.tokens, (hq + 2 * hk), d), seed * 31 + 3, t)
    s.rows *= torch.linspace(0.25, 2.0, hq + 2 * hk, device=DEV).to(t).unsqueeze(1)
    s.rows = s.rows.view(s.tokens, -1)
    s.out = torch.empty((s.tokens, hq * d), dtype=t, device=DEV)
    torch.cuda.synchronize()
    return s


# ---- the operators in plain form ------------------------------------------------------------------------------------

def _plain_rope(s):
    case = s.case
    d, n, p = case["dim"], case["q_heads"] + case["kv_heads"], sum(_pairs(case))
    axis, place = _axes(case)
    axis = torch.tensor(axis, device=DEV)
    if case["ladders"]:
        slope = torch.tensor(place, dtype=torch.float64, device=DEV) / torch.tensor(_pairs(case), dtype=torch.float64, device=DEV)[axis]
    else:
        slope = torch.arange(p, dtype=torch.float64, device=DEV) / p
    freq = torch.pow(torch.tensor(case["base"], dtype=torch.float64, device=DEV), -slope)
    if s.factors is not None:
        freq = freq * s.factors.double()
    angle = s.pos.double()[axis].t() * freq  # [tokens, pairs], in 64 bits: a far position times a frequency keeps few bits in 32
    c, q = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)
    x = s.rows[:, :n * d].float().view(-1, n, d)
    y = x.clone()
    a, b = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if case["neighbours"] else (slice(0, p), slice(p, 2 * p))
    y[..., a] = x[..., a] * c - x[..., b] * q
    y[..., b] = x[..., a] * q + x[..., b] * c
    s.out.copy_(y.view(-1, n * d).to(s.out.dtype))
    return s.out


def _plain_cache(s):
    case = s.case
    hk, hq, d, page, t = case["kv_heads"], case["q_heads"], case["dim"], case["page"], s.back.dtype
    rows = s.rows.view(-1, hq + 2 * hk, d)
    p, i = (s.slots // page).long(), (s.slots % page).long()
    if not hasattr(s, "codes"):
        s.codes = torch.zeros((2, case["pages"], hk, page, d), dtype=torch.uint8, device=DEV)
        s.scales = torch.zeros((2, case["pages"], hk, page, d // 32), dtype=torch.float16, device=DEV)
    for which in range(2):
        codes, scales = _quantise(rows[:, hq + which * hk:hq + (which + 1) * hk])
        s.codes[which][p, :, i], s.scales[which][p, :, i] = codes, scales
        c, m = s.codes[which][p, :, i].float(), s.scales[which][p, :, i].float()
        s.back[which] = ((c.unflatten(-1, (-1, 32)) - 8) * m.unsqueeze(-1)).to(t).view(-1, hk * d)
    return s.back


def _cached(plane, table, n, values):
    """Rows of the cache in order, fp32 [requests, heads, n, dim]."""
    g = plane[table.clamp(min=0).long()].transpose(1, 2)  # [requests, heads, pages, tiles, bytes]
    return _open(g.flatten(2, 3), values)[:, :, :n]


def _plain_attn_group(s, first, count):
    if not count:
        return
    case = s.case
    hk, hq, d = case["kv_heads"], case["q_heads"], case["dim"]
    m, n = max(s.new[first:first + count]), max(s.lens[first:first + count])
    start, new = s.q_start[first:first + count].long(), s.q_start[first + 1:first + count + 1].long()
    at = start.unsqueeze(1) + torch.arange(m, device=DEV)
    real, new = at < new.unsqueeze(1), new - start
    g = hq // hk
    q = s.rows[at.clamp(max=s.tokens - 1)].view(count, m, hq + 2 * hk, d)[:, :, :hq].float()
    q = q.view(count, m, hk, g, d).permute(0, 2, 3, 1, 4)
    kv = s.kv_len[first:first + count].long()
    table = s.table[first:first + count, :-(-n // case["page"])]
    k = _cached(s.k, table, n, False)
    x = torch.matmul((q * d ** -0.5).reshape(count, hk, g * m, d), k.transpose(2, 3)).view(count, hk, g, m, n)
    del k
    j, p = torch.arange(n, device=DEV), ((kv - new).unsqueeze(1) + torch.arange(m, device=DEV)).unsqueeze(2)
    see = (j <= p) & (j < kv.view(-1, 1, 1))
    if case["window"]:
        see &= (j > p - case["window"]) | (j < case["sinks"])
    x.masked_fill_(~see.view(count, 1, 1, m, n), -math.inf)
    x.sub_(x.amax(4, keepdim=True).clamp(min=-1e30)).exp_()
    total = x.sum(4, keepdim=True)
    v = _cached(s.v, table, n, True)
    y = torch.matmul(x.view(count, hk, g * m, n), v).view(count, hk, g, m, d) / total
    y = y.permute(0, 3, 1, 2, 4).reshape(count, m, hq * d)
    s.out[at[real]] = y[real].to(s.out.dtype)


def _plain_attn(s):
    _plain_attn_group(s, 0, s.case["prompts"])
    _plain_attn_group(s, s.case["prompts"], s.case["reqs"] - s.case["prompts"])
    return s.out


def _plain_sample(s):
    x = s.logits.double()  # sums over a whole vocabulary, and values next to a border
    rows, vocab = x.shape
    sorted_, order = torch.sort(x, dim=1, descending=True, stable=True)
    t = s.temperature.double().unsqueeze(1)
    w = torch.exp((sorted_ - sorted_[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(vocab, device=DEV)
    k = torch.where((s.top_k > 0) & (s.top_k < vocab), s.top_k, vocab).unsqueeze(1)
    k = torch.where(t > 0, k, 1)
    keep = rank < k
    w = torch.where(keep, w, 0.0)
    run = w.cumsum(1)
    before = torch.cat([torch.zeros_like(run[:, :1]), run[:, :-1]], 1)
    p = s.top_p.double().unsqueeze(1)
    keep &= (before < p * run[:, -1:]) | (p >= 1.0)
    keep &= w >= s.min_p.double().clamp(max=1.0).unsqueeze(1)
    keep[:, 0] = True
    kept = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    run = kept.cumsum(1)
    over = run > s.u.double().unsqueeze(1) * run[:, -1:]
    last = vocab - 1 - kept.flip(1).gt(0).long().argmax(1)
    pick = torch.where(over.any(1), over.long().argmax(1), last)
    s.token.copy_(pick)
    s.logprob.copy_(torch.log(kept.gather(1, pick.unsqueeze(1)).squeeze(1) / run[:, -1]))
    return s.token, s.logprob


# ---- the framework's operators ---------------------------------------------------------------------------------------

_backend = []


def _tb():
    if not _backend:
        from tcb_amd import QuantBackend
        _backend.append(QuantBackend(0))
    return _backend[0]


def run(s):
    case = s.case
    if not own:
        return {"rope": _plain_rope, "cache": _plain_cache, "attn": _plain_attn, "sample": _plain_sample}[case["kind"]](s)
    import tcb_amd
    tb, io = _tb(), {"f32": tcb_amd.F32, "f16": tcb_amd.F16, "bf16": tcb_amd.BF16}[case["dtype"]]
    if case["kind"] == "sample":
        tb.Sample(s.logits.data_ptr(), io, case["vocab"], case["rows"], case["vocab"], s.u.data_ptr(), s.token.data_ptr(), s.logprob.data_ptr(),
                  temperature=s.temperature.data_ptr(), top_k=s.top_k.data_ptr(), top_p=s.top_p.data_ptr(), min_p=s.min_p.data_ptr())
        return s.token, s.logprob
    hk, hq, d = case["kv_heads"], case["q_heads"], case["dim"]
    row = (hq + 2 * hk) * d
    if case["kind"] == "rope":
        if s.spec is None:
            s.spec = tcb_amd.RopeSpec(_pairs(case), case["base"], neighbours=case["neighbours"], dealt=case["dealt"], ladders=case["ladders"],
                                      factors=s.factors.data_ptr() if s.factors is not None else None)
        tb.Rope(s.spec, s.rows.data_ptr(), row, s.out.data_ptr(), (hq + hk) * d, io, case["tokens"], hq + hk, d, s.pos.data_ptr(), case["tokens"])
        return s.out
    if s.kv is None:
        s.kv = tcb_amd.KV4Cache(s.k.shape[0], case["page"], hk, d, s.k.data_ptr(), s.v.data_ptr())
    if case["kind"] == "cache":
        k = s.rows.data_ptr() + hq * d * s.rows.element_size()
        tb.KV4Append(s.kv, case["tokens"], k, k + hk * d * s.rows.element_size(), io, row, s.slots.data_ptr())
        tb.KV4Read(s.kv, case["tokens"], s.back[0].data_ptr(), s.back[1].data_ptr(), io, hk * d, s.slots.data_ptr())
        return s.back
    tb.KV4Attention(s.kv, s.rows.data_ptr(), io, row, s.out.data_ptr(), hq * d, s.tokens, hq, case["reqs"], s.q_start.data_ptr(),
                    s.kv_len.data_ptr(), s.table.data_ptr(), s.table.shape[1], max_new=max(s.new), window=case["window"], sinks=case["sinks"])
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
    kind, e = case["kind"], 4 if case["dtype"] == "f32" else 2
    if kind == "sample":  # logits in, settings, numbers and tokens; an exponential and a sum a logit
        return {"bytes": case["rows"] * (case["vocab"] * e + 28), "flops": 3 * case["rows"] * case["vocab"]}
    hk, hq, d = case["kv_heads"], case["q_heads"], case["dim"]
    if kind == "rope":
        return {"bytes": case["tokens"] * (2 * (hq + hk) * d * e + 4 * len(_pairs(case))), "flops": 6 * case["tokens"] * (hq + hk) * sum(_pairs(case))}
    if kind == "cache":  # rows in, 4.5 bits an element out, the same back
        return {"bytes": case["tokens"] * (2 * (2 * hk * d * e + 2 * hk * d * 9 // 16) + 8), "flops": 8 * case["tokens"] * hk * d}
    new, kv = _lengths(case)
    seen = [_seen(n, k, case["window"], case["sinks"]) for n, k in zip(new, kv)]
    pairs, keys, tokens = sum(p for p, _ in seen), sum(k for _, k in seen), sum(new)
    return {"bytes": 2 * keys * hk * d * 9 // 16 + 4 * tokens * hq * d + 4 * (keys // case["page"] + 3 * case["reqs"]), "flops": 4 * pairs * hq * d}


# ---- the same from the definitions, in 64 bits ------------------------------------------------------------------------

def _exact_rope(s):
    case = s.case
    d, n, p = case["dim"], case["q_heads"] + case["kv_heads"], sum(_pairs(case))
    out = s.rows[:, :n * d].double().view(-1, n, d).clone()
    axis, place = _axes(case)
    for i in range(p):
        slope = place[i] / _pairs(case)[axis[i]] if case["ladders"] else i / p
        f = math.exp(-slope * math.log(case["base"])) * (float(s.factors[i]) if s.factors is not None else 1.0)
        z = torch.polar(torch.ones(case["tokens"], dtype=torch.float64, device=DEV), s.pos[axis[i]].double() * f).unsqueeze(1)
        a, b = (2 * i, 2 * i + 1) if case["neighbours"] else (i, i + p)
        w = torch.complex(out[:, :, a].clone(), out[:, :, b].clone()) * z
        out[:, :, a], out[:, :, b] = w.real, w.imag
    return out.view(-1, n * d)


def _exact_blocks(x):
    """What blocks [..., 32] of float64 values become in 4 bits: by comparing with every level there is."""
    size = x.abs()
    most = size.amax(-1, keepdim=True)
    m = torch.zeros_like(most)
    for i in range(31, -1, -1):  # the first of the largest stays
        m = torch.where(size[..., i:i + 1] == most, x[..., i:i + 1], m)
    a = m.abs() / 8
    def lowest(y):  # the power of two at or below y, by its exponent's bits
        return y.view(torch.int64).bitwise_right_shift(52).bitwise_left_shift(52).view(torch.float64)
    unit = lowest(a.clamp(min=2.0 ** -200)) / 16
    d = torch.round(a / unit) * unit
    unit = torch.clamp(lowest(d.clamp(min=2.0 ** -200)) / 1024, min=2.0 ** -24)
    d = torch.round(d / unit) * unit  # to f16
    d = torch.clamp(d, max=7936.0) * -torch.sign(m)
    best, far = torch.zeros_like(x), torch.full_like(x, math.inf)
    for level in (0, -2, 2, -4, 4, -6, 6, -8, -1, 1, -3, 3, -5, 5, -7, 7):  # even ones first: they win where two are as near
        off = (x - level * d).abs()
        best, far = torch.where(off < far, level * d, best), torch.minimum(off, far)
    return best


def _exact_values(plane, pages, page, n, values):
    """Float64 [n, heads, dim] of keys 0 .. n - 1, byte by byte from the planes' layout."""
    heads, dim = plane.shape[1], plane.shape[3] // 9
    groups = dim // 32
    j, e = torch.arange(n, device=DEV).unsqueeze(1), torch.arange(dim, device=DEV)
    r, g = j % 16, e // 32
    if values:
        dword = ((r // 4) * 16 + e % 32 // 2) * groups + g
        nib = torch.tensor(AT_V, device=DEV)[(r % 4).expand(n, dim), (e % 2).expand(n, dim)]
    else:
        dword = ((e % 32 // 8) * 16 + r) * groups + g
        nib = torch.tensor(AT_K, device=DEV)[e % 8].expand(n, dim)
    scale_at = 4 * dim + (r // 4 * groups + g) * 4 + r % 4  # in f16 units from the piece's start
    out = torch.empty((n, heads, dim), dtype=torch.float64, device=DEV)
    tile = (pages.long()[torch.arange(n, device=DEV) // page], torch.arange(n, device=DEV) % page // 16)
    for h in range(heads):
        piece = plane[tile[0], h, tile[1]]
        byte = piece.gather(1, dword * 4 + nib // 2)
        code = (byte.long() >> (4 * (nib % 2))) & 15
        out[:, h] = (code - 8) * piece.view(torch.float16).gather(1, scale_at).double()
    return out


def _exact_attn(s):
    case = s.case
    hk, hq, d, page = case["kv_heads"], case["q_heads"], case["dim"], case["page"]
    out = torch.zeros((s.tokens, hq * d), dtype=torch.float64, device=DEV)
    window, sinks, t0 = case["window"], case["sinks"], 0
    for i, (n, length) in enumerate(zip(s.new, s.lens)):
        k, v = (_exact_values(c, s.table[i], page, length, c is s.v) for c in (s.k, s.v))
        j, p = torch.arange(length, device=DEV), torch.arange(length - n, length, device=DEV).unsqueeze(1)
        see = j <= p
        if window:
            see = see & ((p - j < window) | (j < sinks))
        q = s.rows[t0:t0 + n].double().view(n, -1, d)
        for h in range(hq):
            x = torch.where(see, q[:, h] @ k[:, h * hk // hq].t() / math.sqrt(d), -math.inf)
            w = torch.exp(x - x.max(-1, keepdim=True).values)
            out[t0:t0 + n, h * d:(h + 1) * d] = (w / w.sum(-1, keepdim=True)) @ v[:, h * hk // hq]
        t0 += n
    return out


def _exact_sample(s):
    logits = s.logits.double().cpu().numpy()
    settings = [x.cpu().numpy() for x in (s.temperature, s.top_k, s.top_p, s.min_p, s.u)]
    tokens, logs = [], []
    for x, t, k, p, low, u in zip(logits, *settings):
        order = np.argsort(-x, kind="stable")
        if t <= 0:
            order = order[:1]
        elif 0 < k < len(x):
            order = order[:k]
        w = np.exp((x[order] - x[order[0]]) / (float(t) if t > 0 else 1.0))
        n = len(order)
        if p < 1:
            n = max(1, int(np.searchsorted(np.cumsum(w), float(p) * w.sum(), side="left")) + 1)
        n = min(n, max(1, int((w >= min(float(low), 1.0)).sum())))
        by_index = np.argsort(order[:n])
        run = np.cumsum(w[:n][by_index])
        at = min(int(np.searchsorted(run, float(u) * run[-1], side="right")), n - 1)
        tokens.append(int(order[:n][by_index][at]))
        logs.append(float(np.log(w[:n][by_index][at] / run[-1])))
    return torch.tensor(tokens, dtype=torch.int32, device=DEV), torch.tensor(logs, dtype=torch.float64, device=DEV)


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "rope":
        return _exact_rope(s)
    if kind == "attn":
        return _exact_attn(s)
    if kind == "sample":
        return _exact_sample(s)
    hk, hq, d = case["kv_heads"], case["q_heads"], case["dim"]
    rows = s.rows.double().view(-1, hq + 2 * hk, d)
    return torch.stack([_exact_blocks(rows[:, hq + w * hk:hq + (w + 1) * hk].unflatten(-1, (-1, 32))).reshape(-1, hk * d) for w in range(2)])
