"""From a chat's rows to its next token, all calls of a step together: page tables, the quantized q/k/v product, rotary positions, the append
to the 4-bit cache, attention over it, the products behind it, sampling; the token's row is the next step's. Every call's output is
compared with its plain form on the output before it."""
import ctypes

import numpy as np
import pytest
import torch

import kv4_ref as K4
import paged_ref as R
import tcb_amd
from tcb_amd import BF16, F32, MODE_FAST, Q4K, _lib, synth
from test_gpu_rope import HALF, turned
from test_gpu_sample import choose

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
HIDDEN, HEADS, KV_HEADS, DIM, PAGE, VOCAB = 256, 8, 2, 64, 16, 1000
TURN = HEADS + KV_HEADS
ROW = (TURN + KV_HEADS) * DIM
PAIRS = (8, 12, 12)


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Model:
    def __init__(self, tb, chats, most):
        self.tb, self.most = tb, most
        self.qkv = tb.FromQuantized(Q4K, synth.quant_weights(Q4K, ROW, HIDDEN, seed=1), ROW, HIDDEN)
        self.o = tb.FromQuantized(Q4K, synth.quant_weights(Q4K, HIDDEN, HEADS * DIM, seed=2), HIDDEN, HEADS * DIM)
        self.head = tb.FromQuantized(Q4K, synth.quant_weights(Q4K, VOCAB, HIDDEN, seed=3), VOCAB, HIDDEN)
        self.kv = tb.NewKV4Cache(chats * most, PAGE, KV_HEADS, DIM)
        self.rope = tcb_amd.RopeSpec(PAIRS, base=500000.0, dealt=True)

    def buffers(self, tokens, chats):
        b = dict(raw=(tokens, ROW), rows=(tokens, ROW), att=(tokens, HEADS * DIM))
        b = {n: torch.zeros(s, dtype=torch.bfloat16, device=DEV) for n, s in b.items()}
        b.update(y=torch.zeros((tokens, HIDDEN), device=DEV), logits=torch.zeros((tokens, VOCAB), device=DEV),
                 token=ints([-5] * tokens), logprob=torch.zeros(tokens, device=DEV))
        return b

    def run(self, b, x, tokens, chats, new, pos, start, lens, table, slots, setting, window=0, sinks=0):
        """All of a step's calls but the page tables, on the context's stream."""
        tb = self.tb
        tb.GemmTyped(tokens, ROW, HIDDEN, x.data_ptr(), F32, self.qkv, b["raw"].data_ptr(), BF16, mode=MODE_FAST)
        tb.Rope(self.rope, b["raw"].data_ptr(), ROW, b["rows"].data_ptr(), ROW, BF16, tokens, TURN, DIM, pos.data_ptr(), tokens)
        tb.KV4Append(self.kv, tokens, b["rows"].data_ptr() + 2 * HEADS * DIM, b["raw"].data_ptr() + 2 * TURN * DIM, BF16, ROW, slots.data_ptr())
        tb.KV4Attention(self.kv, b["rows"].data_ptr(), BF16, ROW, b["att"].data_ptr(), HEADS * DIM, tokens, HEADS, chats, start.data_ptr(),
                        lens.data_ptr(), table.data_ptr(), self.most, max_new=new, window=window, sinks=sinks)
        tb.GemmTyped(tokens, HIDDEN, HEADS * DIM, b["att"].data_ptr(), BF16, self.o, b["y"].data_ptr(), F32, mode=MODE_FAST)
        tb.GemmTyped(tokens, VOCAB, HIDDEN, b["y"].data_ptr(), F32, self.head, b["logits"].data_ptr(), F32, mode=MODE_FAST)
        t, k, p, low, u = (a.data_ptr() for a in setting)
        tb.Sample(b["logits"].data_ptr(), F32, VOCAB, tokens, VOCAB, u, b["token"].data_ptr(), b["logprob"].data_ptr(), t, k, p, low)

    def release(self):
        self.qkv.release(), self.o.release(), self.head.release(), self.kv.release()


def settings(tokens, seed):
    rng = np.random.default_rng(seed)
    rows = [rng.choice(c, tokens) for c in ([0.0, 0.6, 1.0, 1.3], [0, 0, 40, 200], [1.0, 0.9, 0.95], [0.0, 0.02])] + [rng.random(tokens)]
    return [torch.tensor(a, dtype=torch.int32 if i == 1 else torch.float32, device=DEV) for i, a in enumerate(rows)]


@pytest.mark.parametrize("window,sinks", [(0, 0), (32, 4)])
def test_chats(backend, window, sinks):
    """Prompts together, then tokens, with another chat's prompt in between; and at the end the whole cache."""
    tb, prompts, late, steps = backend, (37, 150, 1), 61, 7
    chats, most = len(prompts) + 1, 12
    m = Model(tb, chats, most)
    gen = torch.Generator().manual_seed(3)
    embed = torch.randn((VOCAB, HIDDEN), generator=gen).to(DEV)
    free = torch.randperm(chats * most, generator=gen).to(torch.int32).to(DEV)
    table = torch.full((chats, most), -1, dtype=torch.int32, device=DEV)
    old, taken = ints([0] * chats), 0
    texts = [torch.randint(0, VOCAB, (n,), generator=gen).tolist() for n in prompts + (late,)]
    keys, values = [[np.zeros((0, KV_HEADS, DIM))] * chats for _ in range(2)]
    for step in range(steps):
        add = [n if step == 0 else 1 for n in prompts] + [0 if step < 2 else late if step == 2 else 1]
        tokens = sum(add)
        ids = [t for text, n in zip(texts, add) for t in (text[-n:] if n else [])]
        x = embed[torch.tensor(ids, device=DEV)].contiguous()
        first = [len(text) - n if n else 0 for text, n in zip(texts, add)]
        line = np.concatenate([np.arange(a, a + n) for a, n in zip(first, add)]).astype(np.int32)
        pos = np.stack([line, line // 7, line % 7]).astype(np.int32)
        start, lens, slots, used = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (chats + 1, chats, tokens, 1))
        n, where, setting, b = ints(add), torch.from_numpy(pos).to(DEV), settings(tokens, step), m.buffers(tokens, chats)
        torch.cuda.synchronize()
        tb.PageTables(chats, PAGE, old.data_ptr(), n.data_ptr(), free.data_ptr() + 4 * taken, free.numel() - taken, table.data_ptr(), most,
                      start.data_ptr(), lens.data_ptr(), slots.data_ptr(), tokens, used.data_ptr())
        m.run(b, x, tokens, chats, max(add), where, start, lens, table, slots, setting, window, sinks)
        tb.ctx.sync()
        old, taken = lens, taken + int(used)
        # positions
        raw = b["raw"].cpu().double().numpy().reshape(tokens, -1, DIM)
        rows = b["rows"].cpu().double().numpy().reshape(tokens, -1, DIM)
        want, tol = turned(raw[:, :TURN], pos, PAIRS, 500000.0, False, True, False, None)
        assert np.isfinite(raw).all()
        assert (np.abs(rows[:, :TURN] - want) <= tol + HALF["bf16"] * (np.abs(want) + tol) + 2.0 ** -134).all(), step
        assert (rows[:, TURN:] == 0).all()
        # the cache, then attention over it
        att, at = b["att"].cpu().double().numpy().reshape(tokens, HEADS, DIM), 0
        for c in range(chats):
            keys[c] = np.concatenate([keys[c], rows[at:at + add[c], HEADS:TURN]])
            values[c] = np.concatenate([values[c], raw[at:at + add[c], TURN:]])
            if add[c]:
                k, v = (K4.values(*K4.quantize(a)) for a in (keys[c], values[c]))
                o, spread, reach = R.attend(rows[at:at + add[c], :HEADS], k, v, len(k) - add[c], DIM ** -0.5, window, sinks)
                tol = K4.bound("bf16", DIM, len(k), add[c] * (HEADS // KV_HEADS) > 96, o, spread, reach, np.abs(v).max())
                assert (np.abs(att[at:at + add[c]] - o) <= tol).all(), (step, c)
            at += add[c]
        # the tokens
        logits, token, logprob = (b[i].cpu().numpy() for i in ("logits", "token", "logprob"))
        t, k, p, low, u = (a.cpu().numpy() for a in setting)
        for r in range(tokens):
            want, log, close = choose(logits[r], float(t[r]), int(k[r]), float(p[r]), float(low[r]), float(u[r]))
            assert close or (token[r] == want and abs(logprob[r] - log) <= 2.0 ** -23 * abs(log) + 1e-11), (step, r)
        for c, e in enumerate(np.cumsum(add)):
            if add[c]:
                texts[c] = texts[c] + [int(token[e - 1])]
    # what the cache holds, page by page
    pages = table.cpu().numpy()
    for c in range(chats):
        n = len(keys[c])
        at = ints([int(pages[c, j // PAGE]) * PAGE + j % PAGE for j in range(n)])
        back = torch.zeros((2, n, KV_HEADS * DIM), device=DEV)
        torch.cuda.synchronize()
        tb.KV4Read(m.kv, n, back[0].data_ptr(), back[1].data_ptr(), F32, KV_HEADS * DIM, at.data_ptr())
        tb.ctx.sync()
        for got, a in zip(back.cpu().double().numpy(), (keys[c], values[c])):
            assert np.array_equal(got.reshape(a.shape), K4.values(*K4.quantize(a)))
    m.release()


def test_a_captured_step(backend):
    """A token of each chat in one graph: replays follow their inputs and give the bits of the eager calls, with eager work in between."""
    tb, chats, most, start_at = backend, 5, 8, (3, 16, 31, 90, 0)
    m, e = Model(tb, chats, most), Model(tb, chats, most)
    gen = torch.Generator().manual_seed(5)
    embed = torch.randn((VOCAB, HIDDEN), generator=gen).to(DEV)
    table = torch.randperm(chats * most, generator=gen).to(torch.int32).view(chats, most).to(DEV)
    fill = torch.randn((2, chats * most * PAGE, KV_HEADS * DIM), generator=gen).to(DEV)
    every, start = torch.arange(chats * most * PAGE, dtype=torch.int32, device=DEV), torch.arange(chats + 1, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    for a in (m, e):
        tb.KV4Append(a.kv, every.numel(), fill[0].data_ptr(), fill[1].data_ptr(), F32, KV_HEADS * DIM, every.data_ptr())
    x, pos, slots, lens = torch.zeros((chats, HIDDEN), device=DEV), ints([[0] * chats] * 3), ints([0] * chats), ints([1] * chats)
    setting, b, want = settings(chats, 9), m.buffers(chats, chats), e.buffers(chats, chats)
    where = (chats, chats, 1, pos, start, lens, table, slots, setting)
    torch.cuda.synchronize()
    e.run(want, x, *where)  # (its workspaces are there before a graph takes them)
    tb.ctx.sync()
    lib, g = _lib.lib(), ctypes.c_void_p()
    assert lib.trhip_graph_begin(tb.ctx.h) == 0
    m.run(b, x, *where)
    assert lib.trhip_graph_end(tb.ctx.h, ctypes.byref(g)) == 0
    ids, at = [1, 2, 3, 4, 5], list(start_at)
    for step in range(6):
        x.copy_(embed[torch.tensor(ids, device=DEV)])
        pos.copy_(ints([at, [a // 7 for a in at], [a % 7 for a in at]]))
        slots.copy_(torch.stack([table[c, a // PAGE] * PAGE + a % PAGE for c, a in enumerate(at)]))
        lens.copy_(ints([a + 1 for a in at]))
        for old, new in zip(setting, settings(chats, 20 + step)):
            old.copy_(new)
        torch.cuda.synchronize()
        e.run(want, x, *where)
        tb.ctx.sync()
        assert lib.trhip_graph_launch(tb.ctx.h, g) == 0
        tb.ctx.sync()
        for name in b:
            assert torch.equal(b[name], want[name]), (step, name)
        ids, at = b["token"].tolist(), [a + 1 for a in at]
        assert all(0 <= i < VOCAB for i in ids)
    assert lib.trhip_graph_destroy(g) == 0
    m.release(), e.release()
