"""A quantized attention block over a paged key/value cache: a layer's products with the cache and the attention between the merged
q/k/v product and the output projection (no rotation of q and k by position: a model that has one applies it there, with Rope).

A few chats are served together. Their prompts come in at once, then each step brings a token of every chat (and another
chat's prompt in between). All of it goes through the same four calls a step: page tables from the lengths, the quantized
q/k/v product, the append of its k and v rows, attention of its q rows. Last, several samples continue one chat, whose keys they
share as a prefix. Every step's rows are compared with the block run on the whole text at once.

  python examples/attention_block.py
"""
import os
import sys

import torch  # before the library: one HIP runtime in the process, torch's

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from tcb_amd import BF16, F32, MODE_FAST, Q4K, QuantBackend, synth  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, PAGE = 1024, 8, 2, 128, 16
ROW = (HEADS + 2 * KV_HEADS) * DIM  # a row of the merged q/k/v product
DEV = "cuda:0"


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Block:
    """One layer's attention: weights, cache, page tables of up to `chats` chats of `most` keys."""

    def __init__(self, tb, chats, most, seed=1):
        self.tb, self.most = tb, -(-most // PAGE)
        self.qkv = tb.FromQuantized(Q4K, synth.quant_weights(Q4K, ROW, HIDDEN, seed=seed), ROW, HIDDEN)
        self.o = tb.FromQuantized(Q4K, synth.quant_weights(Q4K, HIDDEN, HEADS * DIM, seed=seed + 1), HIDDEN, HEADS * DIM)
        pages = chats * self.most
        self.kv = tb.NewKVCache(BF16, pages, PAGE, KV_HEADS, DIM)
        self.free = torch.randperm(pages, device=DEV).to(torch.int32)
        self.taken = 0
        self.table = torch.full((chats, self.most), -1, dtype=torch.int32, device=DEV)
        self.lens = torch.zeros(chats, dtype=torch.int32, device=DEV)

    def step(self, x, add, window=0, sinks=0):
        """x [tokens, HIDDEN]: add[i] tokens of chat i, in order. Returns the block's output rows."""
        tb, n, tokens, chats = self.tb, ints(add), x.shape[0], len(add)
        start, lens, slots, used = (torch.empty(m, dtype=torch.int32, device=DEV) for m in (chats + 1, chats, tokens, 1))
        rows = torch.empty((tokens, ROW), dtype=torch.bfloat16, device=DEV)
        att = torch.empty((tokens, HEADS * DIM), dtype=torch.bfloat16, device=DEV)
        y = torch.empty((tokens, HIDDEN), device=DEV)
        torch.cuda.synchronize()  # torch's stream to the context's
        tb.PageTables(chats, PAGE, self.lens.data_ptr(), n.data_ptr(), self.free.data_ptr() + 4 * self.taken, self.free.numel() - self.taken,
                      self.table.data_ptr(), self.most, start.data_ptr(), lens.data_ptr(), slots.data_ptr(), tokens, used.data_ptr())
        tb.GemmTyped(tokens, ROW, HIDDEN, x.data_ptr(), F32, self.qkv, rows.data_ptr(), BF16, mode=MODE_FAST)
        k = rows.data_ptr() + 2 * HEADS * DIM
        tb.KVAppend(self.kv, tokens, k, k + 2 * KV_HEADS * DIM, BF16, ROW, slots.data_ptr())
        tb.Attention(self.kv, rows.data_ptr(), ROW, att.data_ptr(), HEADS * DIM, tokens, HEADS, chats, start.data_ptr(), lens.data_ptr(),
                     self.table.data_ptr(), self.most, max_new=max(add), window=window, sinks=sinks)
        tb.GemmTyped(tokens, HIDDEN, HEADS * DIM, att.data_ptr(), BF16, self.o, y.data_ptr(), F32, mode=MODE_FAST)
        tb.ctx.sync()
        self.lens = lens
        self.taken += int(used)
        return y

    def samples(self, x, chat, prefix):
        """One token each of x.shape[0] samples that continue `chat` behind its first `prefix` keys (nothing is kept of them)."""
        tb, n = self.tb, x.shape[0]
        own = torch.arange(n, dtype=torch.int32, device=DEV).view(n, 1) + self.taken
        own = self.free[own.long()].contiguous()  # a page of its own for each
        slots, one, start = (own.view(-1) * PAGE).contiguous(), ints([1] * n), torch.arange(n + 1, dtype=torch.int32, device=DEV)
        rows = torch.empty((n, ROW), dtype=torch.bfloat16, device=DEV)
        att = torch.empty((n, HEADS * DIM), dtype=torch.bfloat16, device=DEV)
        y = torch.empty((n, HIDDEN), device=DEV)
        lead = self.table[chat].contiguous()
        torch.cuda.synchronize()
        tb.GemmTyped(n, ROW, HIDDEN, x.data_ptr(), F32, self.qkv, rows.data_ptr(), BF16, mode=MODE_FAST)
        k = rows.data_ptr() + 2 * HEADS * DIM
        tb.KVAppend(self.kv, n, k, k + 2 * KV_HEADS * DIM, BF16, ROW, slots.data_ptr())
        tb.AttentionShared(self.kv, rows.data_ptr(), ROW, att.data_ptr(), HEADS * DIM, n, HEADS, n, start.data_ptr(), one.data_ptr(),
                           own.data_ptr(), 1, lead.data_ptr(), prefix, max_new=1)
        tb.GemmTyped(n, HIDDEN, HEADS * DIM, att.data_ptr(), BF16, self.o, y.data_ptr(), F32, mode=MODE_FAST)
        tb.ctx.sync()
        return y

    def release(self):
        self.qkv.release(), self.o.release(), self.kv.release()


def near(got, want):
    """Largest difference of any row over that row's largest value: the same sums, cut differently, in 16-bit rows."""
    return float(((got - want).abs().amax(1) / want.abs().amax(1)).max())


def run(tb, prompts=(37, 200, 5), late=90, steps=20, window=0, sinks=0, say=print):
    """Returns the largest difference of any step's rows from the whole texts' (and of the samples' from theirs)."""
    gen = torch.Generator(device=DEV).manual_seed(7)
    chats = len(prompts) + 1
    texts = [torch.randn((n + steps, HIDDEN), generator=gen, device=DEV) for n in tuple(prompts) + (late,)]
    block = Block(tb, chats + 8, max(t.shape[0] for t in texts) + PAGE)
    whole = Block(tb, chats + 8, max(t.shape[0] for t in texts) + PAGE)
    want = []
    for i, t in enumerate(texts):
        y = whole.step(t.contiguous(), [0] * i + [t.shape[0]] + [0] * (chats + 7 - i), window, sinks)
        want.append(y)
    worst, at = 0.0, [0] * chats
    for step in range(steps + 1):
        add = [n if step == 0 else 1 for n in prompts] + [0 if step < 3 else late if step == 3 else 1]
        x = torch.cat([t[a:a + n] for t, a, n in zip(texts, at, add)])
        y = block.step(x, add + [0] * 8, window, sinks)
        ref = torch.cat([w[a:a + n] for w, a, n in zip(want, at, add)])
        worst = max(worst, near(y, ref))
        at = [a + n for a, n in zip(at, add)]
    say("%d steps of %d chats: within %.1e of the whole texts" % (steps + 1, chats, worst))
    if not window:
        prefix = prompts[1]
        x = texts[1][prefix:prefix + 1].repeat(6, 1) * torch.linspace(0.5, 1.0, 6, device=DEV).unsqueeze(1)
        y = block.samples(x.contiguous(), 1, prefix)
        off = near(y[5:], want[1][prefix:prefix + 1])
        say("6 samples behind %d shared keys: the last within %.1e of its text" % (prefix, off))
        worst = max(worst, off)
    block.release(), whole.release()
    return worst


if __name__ == "__main__":
    tb = QuantBackend(0)
    run(tb)
    run(tb, prompts=(300, 40), late=500, window=128, sinks=4)
    tb.close()
