"""Attention over a paged cache (trhip_attn, trhip_attn_shared) against the float64 form in paged_ref.py."""
import ctypes

import numpy as np
import pytest
import torch

import paged_ref as R
import tcb_amd
from tcb_amd import TrhipError, _lib

pytestmark = pytest.mark.gpu
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"bf16": tcb_amd.BF16, "f16": tcb_amd.F16}
NAN_BITS = {"bf16": 0x7FC1, "f16": 0x7E01}


class Batch:
    """A step's inputs: shuffled pages; every key that no request holds, and every page entry past a request's, is poison."""

    def __init__(self, dtype, heads, kv_heads, dim, page, new, kv, prefix=0, seed=0, spare=2, poison=True):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.heads, self.kv_heads, self.dim, self.page = dtype, heads, kv_heads, dim, page
        self.new, self.kv, self.prefix = list(new), list(kv), prefix
        t = TORCH[dtype]
        counts = [-(-n // page) for n in self.kv] + [-(-prefix // page)]
        total = sum(counts) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.most = max(counts[:-1] + [1])
        self.table = np.full((len(self.kv), self.most), -7, np.int32)
        at = 0
        for i, c in enumerate(counts[:-1]):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.prefix_table = np.array(order[at:at + counts[-1]] + [-9], np.int32)
        self.k, self.v = (torch.randn((total, kv_heads, page, dim), generator=g).to(t) for _ in range(2))
        if poison:
            keep = torch.zeros((total, page), dtype=torch.bool)
            for i, n in enumerate(self.kv):
                for j in range(n):
                    keep[self.table[i, j // page], j % page] = True
            for j in range(prefix):
                keep[self.prefix_table[j // page], j % page] = True
            for plane in (self.k, self.v):
                plane.permute(0, 2, 1, 3)[~keep] = float("nan")
        self.tokens = sum(self.new)
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.q = torch.randn((max(self.tokens, 1), heads, dim), generator=g).to(t)

    def run(self, tb, window=0, sinks=0, scale=None, max_new=None, pad=0, shift=0, out_pad=0, out_shift=0):
        """The operator's rows as float32 [tokens, heads, dim]; pad, shift: elements between rows and in front."""
        width, dev = self.heads * self.dim, "cuda:0"
        q = torch.zeros(shift + self.tokens * (width + pad) + 8, dtype=TORCH[self.dtype], device=dev)
        rows = q[shift:shift + self.tokens * (width + pad)].view(self.tokens, width + pad)
        rows[:, :width] = self.q[:self.tokens].reshape(self.tokens, width).to(dev)
        out = torch.full((out_shift + self.tokens * (width + out_pad) + 8,), 7.0, dtype=TORCH[self.dtype], device=dev)
        k, v = self.k.to(dev), self.v.to(dev)
        start, lens = torch.from_numpy(self.start).to(dev), torch.tensor(self.kv, dtype=torch.int32, device=dev)
        table, prefix = torch.from_numpy(self.table).to(dev), torch.from_numpy(self.prefix_table).to(dev)
        kv = tcb_amd.KVCache(CODE[self.dtype], k.shape[0], self.page, self.kv_heads, self.dim, k.data_ptr(), v.data_ptr())
        args = (kv, q.data_ptr() + 2 * shift, width + pad, out.data_ptr() + 2 * out_shift, width + out_pad, self.tokens, self.heads,
                len(self.kv), start.data_ptr(), lens.data_ptr(), table.data_ptr(), self.most)
        max_new = max(self.new) if max_new is None else max_new
        torch.cuda.synchronize()
        if self.prefix:
            tb.AttentionShared(*args, prefix.data_ptr(), self.prefix, max_new=max_new, scale=scale)
        else:
            tb.Attention(*args, max_new=max_new, window=window, sinks=sinks, scale=scale)
        tb.ctx.sync()
        whole = out[out_shift:out_shift + self.tokens * (width + out_pad)].view(self.tokens, width + out_pad)
        assert (whole[:, width:] == 7.0).all() and (out[:out_shift] == 7.0).all() and (out[out_shift + whole.numel():] == 7.0).all()
        return whole[:, :width].float().cpu().numpy().reshape(self.tokens, self.heads, self.dim)

    def want(self, window=0, sinks=0, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        outs, tols = [], []
        k, v = self.k.float().numpy(), self.v.float().numpy()
        lead = [R.rows_of(c, self.prefix_table, self.prefix, self.page) for c in (k, v)]
        for i, (n, m) in enumerate(zip(self.new, self.kv)):
            q = self.q[self.start[i]:self.start[i + 1]].float().numpy()
            kk, vv = (np.concatenate([l, R.rows_of(c, self.table[i], m, self.page)]) for l, c in zip(lead, (k, v)))
            o, spread, reach = R.attend(q, kk, vv, m - n, scale, window, sinks, self.prefix)
            outs.append(o)
            tols.append(R.bound(self.dtype, self.dim, m + self.prefix, o, spread, reach))
        return np.concatenate(outs), np.concatenate(tols)

    def check(self, tb, window=0, sinks=0, scale=None, **how):
        got = self.run(tb, window, sinks, scale, **how)
        want, tol = self.want(window, sinks, scale)
        off = np.abs(got - want) - tol
        assert np.isfinite(want).all()
        assert np.isfinite(got).all(), "%d values are not finite" % (~np.isfinite(got)).sum()
        worst = np.unravel_index(np.argmax(off), off.shape)
        assert off.max() <= 0, "at %s: got %r want %r, allowed %r" % (worst, got[worst], want[worst], tol[worst])
        return got


HEADS = [(1, 1), (4, 1), (8, 8), (10, 2), (12, 4), (33, 1), (40, 1)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [8, 64, 72, 96, 128, 200, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_tokens(backend, dtype, dim, page):
    """One token a request: lengths around tiles, pages and pieces, no key but its own, a long one."""
    for heads, kv_heads in ([(4, 1), (10, 2)] if dim != 128 else HEADS):
        print(dtype, dim, page, heads, kv_heads, flush=True)
        lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 300, 1025]
        Batch(dtype, heads, kv_heads, dim, page, [1] * len(lens), lens, seed=dim + page).check(backend)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 1, 128), (6, 2, 64), (2, 2, 256), (5, 1, 96)])
def test_prompts(backend, dtype, heads, kv_heads, dim):
    """Prompts from nothing and behind a history, of odd lengths, beside requests that bring one token or none."""
    print(dtype, heads, kv_heads, dim, flush=True)
    new, kv = [77, 1, 0, 130, 33, 5, 1], [77, 200, 50, 190, 33, 300, 1]
    Batch(dtype, heads, kv_heads, dim, 32, new, kv, seed=3).check(backend)
    Batch(dtype, heads, kv_heads, dim, 16, [257], [257], seed=4).check(backend)
    Batch(dtype, heads, kv_heads, dim, 16, [40], [700], seed=5).check(backend)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (7, 0), (7, 3), (32, 4), (33, 0), (100, 40), (100, 200), (4096, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
def test_window_and_sinks(backend, dtype, window, sinks):
    print(dtype, window, sinks, flush=True)
    Batch(dtype, 4, 2, 64, 16, [1, 60, 3, 1, 150], [500, 300, 41, 7, 150], seed=6).check(backend, window, sinks)
    Batch(dtype, 8, 2, 128, 32, [1] * 6, [1, 9, 33, 200, 640, 1000], seed=7).check(backend, window, sinks)


def test_hidden_pages_are_not_read(backend):
    """Pages between the first tokens and the window: their entries name pages of NaN, or none at all."""
    for new in (1, 50):
        b = Batch("bf16", 4, 1, 128, 16, [new], [800], seed=8)
        want, tol = b.want(64, 4)
        low = 800 - new - 64 + 1
        for at, j in enumerate(range(1, low // 16)):
            b.table[0, j] = [-1, 2 ** 31 - 1, -2 ** 31][at % 3]
        got = b.run(backend, 64, 4)
        assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("plane", ["k", "v"])
def test_a_key_reaches_only_the_tokens_that_see_it(backend, dtype, value, plane):
    """A bad key in the middle of a prompt: earlier tokens, and later ones whose window has passed it, are untouched."""
    for window, sinks in ((0, 0), (20, 0), (20, 2)):
        print(dtype, value, plane, window, flush=True)
        b = Batch(dtype, 4, 2, 64, 16, [90, 3, 40], [90, 50, 200], seed=9)
        clean = b.run(backend, window, sinks)
        bad = {0: 37, 1: 48, 2: 171}
        for i, j in bad.items():
            getattr(b, plane)[b.table[i, j // 16], 0, j % 16, 5] = value
        got = b.run(backend, window, sinks)
        for i, j in bad.items():
            for t in range(b.new[i]):
                row, p = b.start[i] + t, b.kv[i] - b.new[i] + t
                if R.visible(p, j, window, sinks):
                    if plane == "v":
                        assert not np.isfinite(got[row, 0, 5])
                        assert np.isfinite(got[row, 0, 6])
                    elif value != value:
                        assert np.isnan(got[row, 0]).all()
                else:
                    assert np.array_equal(got[row], clean[row]) or np.abs(got[row] - clean[row]).max() <= 2.0 ** -7 * np.abs(clean[row]).max()
                    assert np.isfinite(got[row]).all()
                assert np.isfinite(got[row, 2:]).all()  # the other kv head


def whole(b, window=0, sinks=0, scale=None):
    """want() on the GPU in float64, for batches too large for the loop: every request's heads as matrix products."""
    dev, outs, tols = "cuda:0", [], []
    scale = b.dim ** -0.5 if scale is None else scale
    for i, (n, m) in enumerate(zip(b.new, b.kv)):
        pages = [int(x) for x in b.prefix_table[:-(-b.prefix // b.page)]], [int(x) for x in b.table[i, :-(-m // b.page)]]
        kv = []
        for plane in (b.k, b.v):
            parts = [plane[p].to(dev).double().transpose(1, 2).reshape(-1, b.kv_heads, b.dim)[:c] for p, c in zip(pages, (b.prefix, m))]
            kv.append(torch.cat(parts).repeat_interleave(b.heads // b.kv_heads, 1).transpose(0, 1))
        q = b.q[b.start[i]:b.start[i + 1]].to(dev).double().transpose(0, 1)
        s = torch.matmul(q, kv[0].transpose(1, 2).contiguous()) * scale
        j = torch.arange(b.prefix + m, device=dev) - b.prefix
        p = (torch.arange(n, device=dev) + m - n).unsqueeze(1)
        see = (j < 0) | ((j <= p) & ((window == 0) | (j > p - window) | (j < sinks)))
        e = torch.softmax(s.masked_fill(~see, -float("inf")), 2)
        o, spread = torch.matmul(e, kv[1]), torch.matmul(e, kv[1].abs())
        reach = scale * torch.matmul(q.abs(), kv[0].abs().transpose(1, 2).contiguous()).masked_fill(~see, 0).amax(2, keepdim=True)
        o, spread, reach = (x.transpose(0, 1).cpu().numpy() for x in (o, spread, reach))
        outs.append(o)
        tols.append(R.bound(b.dtype, b.dim, m + b.prefix, o, spread, reach))
    return np.concatenate(outs), np.concatenate(tols)


def check_whole(tb, b, window=0, sinks=0, scale=None, **how):
    got = b.run(tb, window, sinks, scale, **how)
    want, tol = whole(b, window, sinks, scale)
    off = np.abs(got - want) - tol
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(off), off.shape)
    assert off.max() <= 0, "at %s: got %r want %r, allowed %r" % (worst, got[worst], want[worst], tol[worst])
    return got


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 4, 64), (5, 1, 96), (4, 2, 256), (3, 1, 200)])
def test_long_prompts(backend, dtype, heads, kv_heads, dim):
    """Blocks in pairs and an odd one, tiles that end anywhere, a short chunk behind a long history (pieces that are joined)."""
    for new, kv, page in (([700], [700], 16), ([129, 64, 500], [900, 1500, 513], 32), ([40], [9000], 64), ([33, 1, 200], [5000, 3000, 260], 16)):
        print(dtype, heads, kv_heads, dim, new, kv, flush=True)
        b = Batch(dtype, heads, kv_heads, dim, page, new, kv, seed=30)
        got = check_whole(backend, b)
        assert np.array_equal(got, b.run(backend))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(128, 0), (130, 4), (300, 64), (1000, 1), (257, 700)])
def test_long_prompts_in_a_window(backend, dtype, window, sinks):
    for heads, kv_heads, dim in ((8, 2, 128), (4, 4, 64), (2, 1, 256)):
        print(dtype, window, sinks, dim, flush=True)
        check_whole(backend, Batch(dtype, heads, kv_heads, dim, 16, [600, 1, 77, 300], [900, 1300, 2000, 300], seed=31), window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(20, 0), (37, 3), (64, 16), (300, 5), (513, 40)])
def test_keys_that_no_token_sees(backend, dtype, window, sinks):
    """Bad keys and values everywhere between the first tokens and the window of a request's first new token: next to the seen
    ones in a piece, a page and a block."""
    for heads, kv_heads, dim in ((4, 1, 128), (4, 2, 64), (33, 1, 128), (2, 1, 256)):
        for new, kv in (([1, 1, 2, 1], [600, 561, 577, 900]), ([1, 60, 130, 300], [700, 641, 800, 1200])):
            print(dtype, window, sinks, heads, dim, new, flush=True)
            b = Batch(dtype, heads, kv_heads, dim, 32, new, kv, seed=33)
            want, tol = whole(b, window, sinks)
            for i, (n, m) in enumerate(zip(new, kv)):
                for j in range(sinks, m - n - window + 1):
                    page, row = b.table[i, j // 32], j % 32
                    b.k[page, :, row] = float("nan")
                    b.v[page, :, row] = float("inf") if j % 2 else float("nan")
            got = b.run(backend, window, sinks)
            assert np.isfinite(got).all()
            assert (np.abs(got - want) <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 128), (4, 1, 64), (6, 1, 256), (33, 1, 96)])
def test_chunks_of_a_few_tiles(backend, dtype, heads, kv_heads, dim):
    """Requests of two and three tiles of 32 rows, alone and beside longer ones, whole and in pieces, in a window, behind a prefix."""
    g = heads // kv_heads
    most = 96 // g
    new = [most, 1, max(most // 2, 1), max(most - 1, 1), max(33 // g, 1)]
    for kv in ([most, 1, 300, 77, 40], [5000, 2600, 9000, 700, 33 + most]):
        print(dtype, heads, kv_heads, dim, new, kv, flush=True)
        b = Batch(dtype, heads, kv_heads, dim, 16, new, kv, seed=34)
        got = check_whole(backend, b)
        assert np.array_equal(got, b.run(backend))
        check_whole(backend, b, 50, 3)
        check_whole(backend, Batch(dtype, heads, kv_heads, dim, 16, new + [most + 1, 200], kv + [900, 200], seed=35))
        check_whole(backend, Batch(dtype, heads, kv_heads, dim, 16, [max(most // 3, 1)] * 3, [9, 200, 70], prefix=1003, seed=36))


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_bad_key_in_a_chunk_of_a_few_tiles(backend, dtype, value):
    for window, sinks in ((0, 0), (40, 4)):
        b = Batch(dtype, 4, 1, 128, 16, [24, 10], [600, 300], seed=37)
        clean = b.run(backend, window, sinks)
        for j in (575, 576, 583, 590, 599):
            b.v[b.table[0, j // 16], 0, j % 16, 7] = value
            got = b.run(backend, window, sinks)
            for t in range(24):
                if any(R.visible(576 + t, k, window, sinks) for k in (575, 576, 583, 590, 599) if k <= j):
                    assert not np.isfinite(got[t, :, 7]).any() and np.isfinite(got[t, :, 8]).all()
                else:
                    assert np.abs(got[t] - clean[t]).max() <= 2.0 ** -7 * np.abs(clean[t]).max()
            assert np.array_equal(got[24:], clean[24:])


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_a_late_key_reaches_only_the_tokens_that_see_it(backend, dtype, value):
    """As above for keys far into long prompts: at a block's edge, in its middle, the last, and one that a window passes."""
    for heads, kv_heads, dim, window, sinks in ((4, 1, 128, 0, 0), (4, 1, 128, 200, 4), (2, 2, 64, 0, 0), (2, 1, 256, 150, 0)):
        for j in (447, 448, 460, 499, 300):
            print(dtype, value, dim, window, j, flush=True)
            b = Batch(dtype, heads, kv_heads, dim, 16, [200, 1], [500, 300], seed=32)
            clean = b.run(backend, window, sinks)
            b.v[b.table[0, j // 16], 0, j % 16, 7] = value
            b.k[b.table[0, j // 16], 0, j % 16, 7] = 1e3
            got = b.run(backend, window, sinks)
            g = heads // kv_heads
            for t in range(200):
                if R.visible(300 + t, j, window, sinks):
                    assert not np.isfinite(got[t, :g, 7]).any()
                    assert np.isfinite(got[t, :g, 8]).all()
                else:
                    assert np.abs(got[t, :g] - clean[t, :g]).max() <= 2.0 ** -7 * np.abs(clean[t, :g]).max()
            assert np.array_equal(got[200], clean[200]) and np.isfinite(got[:, g:]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scores_that_grow_along_the_keys(backend, dtype):
    """References raised again and again, by little and by much, and sharp rows whose last keys hold nearly all weight."""
    for grow in (0.02, 1.0, 30.0):
        for new, kv in (([200], [700]), ([1], [700]), ([1], [20000])):
            b = Batch(dtype, 4, 1, 128, 64, new, kv, seed=33)
            b.q[:] = b.q.abs()
            for j in range(kv[0]):
                b.k[b.table[0, j // 64], 0, j % 64] *= 0.05
                b.k[b.table[0, j // 64], 0, j % 64] += grow * j / kv[0] * 4
            check_whole(backend, b)


def test_far_scores_in_long_prompts(backend):
    """Scores past 2^20 in units of log2, of both signs: the differences are taken first; equal ones average."""
    for x in (-1e30, 1e30, 3e4):
        b = Batch("bf16", 4, 1, 128, 16, [150], [700], seed=34)
        b.q[:] = 0
        b.q[:, :, 0] = 1e30 if abs(x) > 1e20 else 1e3
        for j in range(700):
            b.k[b.table[0, j // 16], 0, j % 16] = 0
            b.k[b.table[0, j // 16], 0, j % 16, 0] = x * (1e-28 if abs(x) > 1e20 else 1)
        check_whole(backend, b, scale=1.0)


def test_rows_that_see_nothing_are_zero(backend):
    """No keys, or fewer than the tokens the request brings: the first tokens sit before key 0."""
    b = Batch("bf16", 4, 2, 64, 16, [1, 5, 70, 2], [0, 3, 40, 2], seed=10)
    got = b.check(backend)
    assert (got[0] == 0).all() and (got[1:3] == 0).all() and (got[6:36] == 0).all() and (got[36] != 0).any()
    for new, kv in (([300], [200]), ([200, 40], [0, 10])):
        b = Batch("f16", 4, 1, 128, 16, new, kv, seed=24)
        got = b.check(backend)
        assert (got[:new[0] - kv[0]] == 0).all()


def test_scores_of_the_lowest_and_highest_values(backend):
    """Scores far from 0 on both sides, and keys whose scores are all -Inf: 0 / 0 as in the formula."""
    b = Batch("bf16", 1, 1, 64, 16, [1, 1, 1], [40, 40, 40], seed=11)
    b.q[:] = 0
    b.q[:, :, 0] = 1e30
    for i, x in enumerate((-1e30, 1e30, -3e38)):
        for j in range(40):
            b.k[b.table[i, j // 16], 0, j % 16] = 0
            b.k[b.table[i, j // 16], 0, j % 16, 0] = x if i == 2 else x * (1e-30 if i else 1e-28)
    got = b.run(backend, scale=1.0)
    for i in (0, 1):
        mean = np.mean([b.v[b.table[i, j // 16], 0, j % 16].float().numpy() for j in range(40)], axis=0)
        assert float(np.abs(got[i, 0] - mean).max()) <= 2.0 ** -7 * b.v.float().nan_to_num().abs().max().item()
    assert np.isnan(got[2]).all()


@pytest.mark.parametrize("shift,pad,out_shift,out_pad", [(0, 8, 0, 4), (1, 0, 1, 0), (3, 5, 2, 1), (8, 1, 4, 3)])
def test_strides_and_alignment(backend, shift, pad, out_shift, out_pad):
    b = Batch("f16", 6, 2, 72, 16, [1, 50, 2], [80, 50, 33], seed=12)
    b.check(backend, pad=pad, shift=shift, out_pad=out_pad, out_shift=out_shift)


def test_long_cache_split_along_the_keys(backend):
    """One token over many keys: the pieces' results join to the same, run after run."""
    for heads, kv_heads, n in ((8, 1, 20011), (4, 4, 9000)):
        b = Batch("bf16", heads, kv_heads, 128, 64, [1], [n], seed=13, poison=False)
        b.q *= 3
        first = b.check(backend)
        assert all(np.array_equal(first, b.run(backend)) for _ in range(3))


def test_many_requests(backend):
    """More requests than a wave has lanes, most with a token, some with none."""
    new = [i % 3 != 0 for i in range(700)]
    kv = [1 + (i * 37) % 90 if n else (i % 2) * 20 for i, n in enumerate(new)]
    Batch("f16", 4, 2, 64, 16, [int(n) for n in new], kv, seed=14).check(backend)


@pytest.mark.parametrize("max_new", [0, 1, 8, 1000])
def test_max_new_is_a_hint(backend, max_new):
    b = Batch("bf16", 8, 2, 128, 16, [90, 1, 300, 9], [90, 400, 320, 30], seed=15)
    b.check(backend, max_new=max_new)


def test_cache_past_32_bits(backend):
    """A plane of over 4 GiB: the pages in use are its last ones."""
    page, hk, d, n = 256, 8, 128, 1000
    pages = (5 << 30) // (page * hk * d * 2)
    k, v = (torch.zeros((pages, hk, page, d), dtype=torch.bfloat16, device="cuda:0") for _ in range(2))
    b = Batch("bf16", 8, hk, d, page, [1, 30], [n, 300], seed=16)
    want, tol = b.want()
    small = b.k.shape[0]
    k[pages - small:], v[pages - small:] = b.k.to("cuda:0"), b.v.to("cuda:0")
    table = torch.from_numpy(np.where(b.table >= 0, b.table + pages - small, -1).astype(np.int32)).to("cuda:0")
    q, out = b.q.to("cuda:0"), torch.empty((31, 8, d), dtype=torch.bfloat16, device="cuda:0")
    start, lens = torch.from_numpy(b.start).to("cuda:0"), torch.tensor(b.kv, dtype=torch.int32, device="cuda:0")
    kv = tcb_amd.KVCache(tcb_amd.BF16, pages, page, hk, d, k.data_ptr(), v.data_ptr())
    torch.cuda.synchronize()
    backend.Attention(kv, q.data_ptr(), 8 * d, out.data_ptr(), 8 * d, 31, 8, 2, start.data_ptr(), lens.data_ptr(), table.data_ptr(), b.most, 30)
    backend.ctx.sync()
    assert (np.abs(out.float().cpu().numpy() - want) <= tol).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv_heads,dim,page", [(4, 1, 128, 16), (8, 8, 64, 32), (6, 2, 96, 16), (2, 1, 256, 64)])
@pytest.mark.parametrize("prefix", [1, 31, 64, 333])
def test_shared_prefix(backend, dtype, heads, kv_heads, dim, page, prefix):
    print(dtype, heads, kv_heads, dim, page, prefix, flush=True)
    Batch(dtype, heads, kv_heads, dim, page, [1] * 9, [1, 2, 16, 17, 40, 64, 65, 100, 7], prefix, seed=17).check(backend)
    Batch(dtype, heads, kv_heads, dim, page, [3, 1, 0, 45, 2], [3, 20, 30, 60, 2], prefix, seed=18).check(backend)


def test_shared_prefix_of_a_large_batch(backend):
    b = Batch("bf16", 8, 2, 128, 32, [2] * 70, [2 + (7 * i) % 50 for i in range(70)], 1500, seed=19)
    first = b.check(backend)
    assert np.array_equal(first, b.run(backend))
    Batch("f16", 8, 2, 128, 32, [1] * 3, [1, 5, 9], 5000, seed=20).check(backend)
    b = Batch("bf16", 8, 2, 128, 32, [2, 1], [1, 0], 100, seed=21)  # tokens without a key of their own: the prefix alone
    b.check(backend)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_long_shared_prefix(backend, dtype, dim):
    """The prefix's rows fill tiles of their own and its keys are cut; own parts of one token, of several, of a prompt."""
    for new, kv, prefix in (([1] * 40, [1 + 13 * i % 200 for i in range(40)], 3001), ([3] * 20, [3 + i for i in range(20)], 777),
                            ([1, 150, 2, 1], [40, 150, 300, 1], 2000), ([2], [70], 4097)):
        print(dtype, dim, new[:4], prefix, flush=True)
        b = Batch(dtype, 8, 2, dim, 32, new, kv, prefix, seed=35)
        got = check_whole(backend, b)
        assert np.array_equal(got, b.run(backend))


def test_shared_prefix_equals_whole_tables(backend):
    """The same keys through trhip_attn, with tables that name the prefix's pages first (it ends at a page's end)."""
    page, prefix = 16, 96
    b = Batch("f16", 8, 4, 64, page, [1, 20, 2], [33, 20, 70], prefix, seed=22)
    shared, (want, tol) = b.run(backend), b.want()
    w = Batch.__new__(Batch)
    w.__dict__.update(b.__dict__)
    w.table = np.concatenate([np.tile(b.prefix_table[:prefix // page], (3, 1)), b.table], 1).astype(np.int32)
    w.most, w.kv, w.prefix = w.table.shape[1], [n + prefix for n in b.kv], 0
    assert (np.abs(w.run(backend) - shared) <= 2 * tol).all()


def test_replayed_graph_follows_the_lengths(backend):
    """A captured call reads the lengths, tables and rows of the moment; every replay equals the eager call."""
    L, ctx, dev = _lib.lib(), backend.ctx, "cuda:0"
    b = Batch("bf16", 8, 2, 128, 16, [1, 1, 1], [700, 300, 900], seed=23, poison=False)
    k, v, q = b.k.to(dev), b.v.to(dev), b.q.to(dev)
    out, eager = (torch.zeros((3, 8, 128), dtype=torch.bfloat16, device=dev) for _ in range(2))
    start, lens, table = torch.from_numpy(b.start).to(dev), torch.tensor(b.kv, dtype=torch.int32, device=dev), torch.from_numpy(b.table).to(dev)
    kv = tcb_amd.KVCache(tcb_amd.BF16, k.shape[0], 16, 2, 128, k.data_ptr(), v.data_ptr())

    def call(to):
        backend.Attention(kv, q.data_ptr(), 1024, to.data_ptr(), 1024, 3, 8, 3, start.data_ptr(), lens.data_ptr(), table.data_ptr(), b.most, 1)

    torch.cuda.synchronize()
    call(eager)
    ctx.sync()
    assert L.trhip_graph_begin(ctx.h) == 0
    call(out)
    graph = ctypes.c_void_p()
    assert L.trhip_graph_end(ctx.h, ctypes.byref(graph)) == 0
    for step in range(4):
        lens.copy_(torch.tensor([max(1, n - 211 * step) for n in b.kv], dtype=torch.int32))
        q.mul_(-0.9)
        torch.cuda.synchronize()
        call(eager)
        assert L.trhip_graph_launch(ctx.h, graph) == 0
        ctx.sync()
        assert torch.equal(out, eager)
    assert L.trhip_graph_destroy(graph) == 0


@pytest.mark.parametrize("new,kv,prefix", [([40, 1, 90, 1], [1500, 3000, 400, 7], 0), ([50], [6000], 0), ([1, 1, 2], [40, 300, 9], 2000),
                                           ([9, 30, 1, 60], [40, 300, 9, 61], 777)])
def test_replayed_graph_of_every_launch(backend, new, kv, prefix):
    """Prompts beside tokens, a chunk in joined pieces, few and many rows behind a prefix: captured, then replayed with other
    lengths and rows between eager calls."""
    L, ctx, dev = _lib.lib(), backend.ctx, "cuda:0"
    b = Batch("f16", 8, 2, 128, 16, new, kv, prefix=prefix, seed=38, poison=False)
    k, v, q = b.k.to(dev), b.v.to(dev), b.q.to(dev)
    out, eager = (torch.zeros((b.tokens, 8, 128), dtype=torch.float16, device=dev) for _ in range(2))
    start, lens, table = torch.from_numpy(b.start).to(dev), torch.tensor(b.kv, dtype=torch.int32, device=dev), torch.from_numpy(b.table).to(dev)
    lead = torch.from_numpy(b.prefix_table).to(dev)
    cache = tcb_amd.KVCache(tcb_amd.F16, k.shape[0], 16, 2, 128, k.data_ptr(), v.data_ptr())

    def call(to):
        args = (cache, q.data_ptr(), 1024, to.data_ptr(), 1024, b.tokens, 8, len(new), start.data_ptr(), lens.data_ptr(), table.data_ptr(), b.most)
        if prefix:
            backend.AttentionShared(*args, lead.data_ptr(), prefix, max_new=max(new))
        else:
            backend.Attention(*args, max_new=max(new))

    torch.cuda.synchronize()
    call(eager)
    ctx.sync()
    assert L.trhip_graph_begin(ctx.h) == 0
    call(out)
    graph = ctypes.c_void_p()
    assert L.trhip_graph_end(ctx.h, ctypes.byref(graph)) == 0
    for step in range(4):
        lens.copy_(torch.tensor([max(n, m - 317 * step) for n, m in zip(new, kv)], dtype=torch.int32))
        q.mul_(-0.9)
        out.fill_(5.0)
        torch.cuda.synchronize()
        call(eager)
        assert L.trhip_graph_launch(ctx.h, graph) == 0
        ctx.sync()
        assert torch.equal(out, eager)
    assert L.trhip_graph_destroy(graph) == 0


def test_refusals(backend):
    x = torch.zeros(4096, dtype=torch.int32, device="cuda:0")
    a = x.data_ptr()

    def kv(**c):
        f = dict(dtype=tcb_amd.BF16, pages=2, page=16, heads=2, dim=64, k=a, v=a)
        f.update(c)
        return tcb_amd.KVCache(**f)

    def attn(cache=None, **c):
        f = dict(q=a, q_stride=256, out=a, out_stride=256, tokens=1, heads=4, nreq=1, q_start=a, kv_len=a, table=a, max_pages=1, max_new=1,
                 window=0, sinks=0, scale=0.1)
        f.update(c)
        backend.Attention(cache or kv(), **f)

    def refused(code, f, *args, **c):
        with pytest.raises(TrhipError) as e:
            f(*args, **c)
        assert e.value.code == code and e.value.detail

    for c in (dict(page=8), dict(page=48), dict(page=8192), dict(heads=0), dict(pages=-1), dict(pages=2 ** 31), dict(k=0), dict(v=a + 8)):
        refused(_lib.ERR_INVALID, attn, kv(**c))
    for c in (dict(dtype=tcb_amd.F32), dict(dim=4), dict(dim=100), dict(dim=264)):
        refused(_lib.ERR_UNSUPPORTED, attn, kv(**c))
    for c in (dict(heads=3), dict(heads=0), dict(tokens=-1), dict(nreq=-1), dict(max_pages=-1), dict(max_new=-1), dict(window=-1),
              dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=0), dict(out=0),
              dict(q_start=0), dict(kv_len=0), dict(table=0), dict(q=a + 1), dict(out=a + 1), dict(q_stride=255), dict(out_stride=0),
              dict(tokens=2 ** 30), dict(max_pages=2 ** 28), dict(window=2 ** 31)):
        refused(_lib.ERR_INVALID, attn, **c)
    with pytest.raises(TrhipError):
        backend.AttentionShared(kv(), a, 256, a, 256, 1, 4, 1, a, a, a, 1, 0, 5)
    with pytest.raises(TrhipError):
        backend.AttentionShared(kv(), a, 256, a, 256, 1, 4, 1, a, a, a, 1, a, -5)
    assert _lib.lib().trhip_attn(backend.ctx.h, None, None, 0, None, 0, 0, 1, 0, None, None, None, 0, 0, 0, 0, 1.0) == _lib.ERR_INVALID
    attn(tokens=0, q=0, out=0)
    attn(nreq=0, q=0, out=0)
