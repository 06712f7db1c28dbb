"""Attention over the 4-bit cache (trhip_kv4_attn) against the float64 form in paged_ref.py, on the values that the cache stands for."""
import ctypes
import threading

import numpy as np
import pytest
import torch

import kv4_ref as K4
import paged_ref as R
import tcb_amd
from tcb_amd import TrhipError, _lib

pytestmark = pytest.mark.gpu
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"bf16": tcb_amd.BF16, "f16": tcb_amd.F16}
DEV = "cuda:0"


class Batch:
    """A step's inputs: shuffled pages; every place that no request holds has all codes 15 and scale NaN, every page entry past a
    request's is out of range."""

    def __init__(self, dtype, heads, kv_heads, dim, page, new, kv, seed=0, spare=2, poison=True, size=1.0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.heads, self.kv_heads, self.dim, self.page = dtype, heads, kv_heads, dim, page
        self.new, self.kv = list(new), list(kv)
        counts = [-(-max(n, 0) // page) for n in self.kv]
        total = sum(counts) + spare
        order = torch.randperm(total, generator=g).tolist()
        self.most = max(counts + [1])
        self.table = np.full((len(self.kv), self.most), -7, np.int32)
        at = 0
        for i, c in enumerate(counts):
            self.table[i, :c] = order[at:at + c]
            at += c
        self.codes, self.scales = [], []
        keep = np.zeros((total, page), bool)
        for i, n in enumerate(self.kv):
            for j in range(n):
                keep[self.table[i, j // page], j % page] = True
        for which in range(2):
            c, d = K4.quantize((torch.randn((total, kv_heads, page, dim), generator=g) * size).numpy())
            if poison:
                c = np.where(keep[:, None, :, None], c, 15).astype(np.uint8)
                d = np.where(keep[:, None, :, None], d, np.float16("nan"))
            self.codes.append(c), self.scales.append(d)
        self.tokens = sum(self.new)
        self.start = np.concatenate([[0], np.cumsum(self.new)]).astype(np.int32)
        self.q = torch.randn((max(self.tokens, 1), heads, dim), generator=g).to(TORCH[dtype])

    def values(self):
        with np.errstate(invalid="ignore"):
            return [np.where(np.isfinite(np.repeat(d, 32, -1)), K4.values(c, d), np.nan) for c, d in zip(self.codes, self.scales)]

    def planes(self):
        return [torch.from_numpy(K4.pack(c, d, w)).to(DEV) for c, d, w in zip(self.codes, self.scales, (False, True))]

    def wide_table(self):
        tiles = (self.tokens * self.heads // self.kv_heads // 16 + len(self.kv)) * self.kv_heads
        most = max(self.most, 2 ** 27 // (tiles * self.dim * self.page) + 2)
        return np.concatenate([self.table, np.full((len(self.kv), most - self.most), -7, np.int32)], 1)

    def run(self, tb, window=0, sinks=0, scale=None, max_new=None, pad=0, shift=0, out_pad=0, out_shift=0, wide=False):
        """The operator's rows as float32 [tokens, heads, dim]; pad, shift: elements between rows and in front; wide: a table so wide that
        the call counts as a large one, whose long requests' keys are opened first."""
        width = self.heads * self.dim
        q = torch.zeros(shift + self.tokens * (width + pad) + 8, dtype=TORCH[self.dtype], device=DEV)
        rows = q[shift:shift + self.tokens * (width + pad)].view(self.tokens, width + pad)
        rows[:, :width] = self.q[:self.tokens].reshape(self.tokens, width).to(DEV)
        out = torch.full((out_shift + self.tokens * (width + out_pad) + 8,), 7.0, dtype=TORCH[self.dtype], device=DEV)
        k, v = self.planes()
        start, lens = torch.from_numpy(self.start).to(DEV), torch.tensor(self.kv, dtype=torch.int32, device=DEV)
        table = self.wide_table() if wide else self.table
        most, table = table.shape[1], torch.from_numpy(table).to(DEV)
        kv = tcb_amd.KV4Cache(k.shape[0], self.page, self.kv_heads, self.dim, k.data_ptr(), v.data_ptr())
        max_new = max(self.new) if max_new is None else max_new
        torch.cuda.synchronize()
        tb.KV4Attention(kv, q.data_ptr() + 2 * shift, CODE[self.dtype], width + pad, out.data_ptr() + 2 * out_shift, width + out_pad, self.tokens, self.heads,
                        len(self.kv), start.data_ptr(), lens.data_ptr(), table.data_ptr(), most, max_new=max_new, window=window, sinks=sinks, scale=scale)
        tb.ctx.sync()
        whole = out[out_shift:out_shift + self.tokens * (width + out_pad)].view(self.tokens, width + out_pad)
        assert (whole[:, width:] == 7.0).all() and (out[:out_shift] == 7.0).all() and (out[out_shift + whole.numel():] == 7.0).all()
        return whole[:, :width].float().cpu().numpy().reshape(self.tokens, self.heads, self.dim)

    def want(self, window=0, sinks=0, scale=None):
        scale = self.dim ** -0.5 if scale is None else scale
        outs, tols = [], []
        k, v = self.values()
        for i, (n, m) in enumerate(zip(self.new, self.kv)):
            q = self.q[self.start[i]:self.start[i + 1]].float().numpy()
            kk, vv = (R.rows_of(c, self.table[i], m, self.page) for c in (k, v))
            o, spread, reach = R.attend(q, kk, vv, m - n, scale, window, sinks)
            outs.append(o)
            largest = np.abs(np.nan_to_num(vv)).max(initial=0.0)
            tols.append(K4.bound(self.dtype, self.dim, m, n * (self.heads // self.kv_heads) > 96, o, spread, reach, largest))
        return np.concatenate(outs), np.concatenate(tols)

    def check(self, tb, window=0, sinks=0, scale=None, wide=False, **how):
        """Twice, where there are long requests: as a small call and as a large one."""
        if not wide and not window and max(self.new) * self.heads // self.kv_heads > 96:
            self.check(tb, window, sinks, scale, True, **how)
        got = self.run(tb, window, sinks, scale, wide=wide, **how)
        want, tol = self.want(window, sinks, scale)
        off = np.abs(got - want) - tol
        assert np.isfinite(want).all()
        assert np.isfinite(got).all(), "%d values are not finite" % (~np.isfinite(got)).sum()
        worst = np.unravel_index(np.argmax(off), off.shape)
        assert off.max() <= 0, "at %s: got %r want %r, allowed %r" % (worst, got[worst], want[worst], tol[worst])
        return got


HEADS = [(1, 1), (4, 1), (8, 8), (10, 2), (12, 4), (17, 1), (33, 1), (40, 1)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
@pytest.mark.parametrize("page", [16, 64])
def test_tokens(backend, dtype, dim, page):
    """One token a request: lengths around tiles, pages and pieces, no key but its own, a long one."""
    for heads, kv_heads in ([(4, 1), (10, 2)] if dim != 128 else HEADS):
        print(dtype, dim, page, heads, kv_heads, flush=True)
        lens = [1, 2, 15, 16, 17, 31, 32, 33, 63, 65, 127, 128, 129, 300, 1025]
        Batch(dtype, heads, kv_heads, dim, page, [1] * len(lens), lens, seed=dim + page).check(backend)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_long_histories(backend, dtype):
    """Keys cut into many pieces; the sizes' hints too large and too small."""
    for lens, hint in [([20000], 1), ([9000, 4000, 1, 7777], 1), ([5000, 3000], 0), ([5000, 3000], 700)]:
        print(dtype, lens, hint, flush=True)
        Batch(dtype, 8, 2, 128, 32, [1] * len(lens), lens, seed=3).check(backend, max_new=hint)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 96, 128, 256])
def test_few_tokens(backend, dtype, dim):
    """Chunks of a few tokens: rows around tiles of 16, 32 and the border to the kernel of many rows."""
    for heads, kv_heads, new in [(4, 1, [3, 4, 5, 8, 9, 1]), (8, 2, [23, 24, 25, 1, 0, 2]), (3, 3, [15, 16, 17, 33, 95, 97]), (20, 1, [1, 2, 4, 5])]:
        kv = [n + a for n, a in zip(new, [0, 300, 17, 64, 5, 130])]
        print(dtype, dim, heads, new, flush=True)
        Batch(dtype, heads, kv_heads, dim, 16, new, kv, seed=dim).check(backend)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 192, 256])
def test_prompts(backend, dtype, dim):
    """Whole prompts and chunks behind a history, beside tokens."""
    for heads, kv_heads, new, kv in [(4, 2, [200, 1, 131], [200, 50, 400]), (2, 2, [300], [300]), (6, 1, [64, 65, 1, 1], [64, 1000, 77, 3])]:
        print(dtype, dim, heads, new, kv, flush=True)
        Batch(dtype, heads, kv_heads, dim, 32, new, kv, seed=dim + 1).check(backend)


@pytest.mark.parametrize("hint", [0, 1, 5, 40, 1000])
def test_wrong_hints(backend, hint):
    Batch("bf16", 8, 2, 64, 16, [150, 1, 7, 30], [400, 33, 90, 31], seed=2).check(backend, max_new=hint)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(1, 0), (16, 4), (33, 1), (100, 0), (64, 70), (500, 17), (1, 200)])
def test_windows(backend, dtype, window, sinks):
    """Tokens, chunks and prompts; keys outside the window and the first ones are never read where whole pages of them are."""
    lens, new = [1, 30, 65, 129, 700, 1500, 400], [1, 1, 1, 20, 1, 1, 300]
    b = Batch(dtype, 8, 2, 64, 16, new, lens, seed=window)
    b.check(backend, window, sinks)
    Batch(dtype, 4, 1, 128, 64, new, lens, seed=window).check(backend, window, sinks)
    for i, (n, m) in enumerate(zip(new, lens)):  # entries of pages that nobody sees may hold anything
        for j in range(b.most):
            seen = any(R.visible(p, key, window, sinks) for p in range(m - n, m) for key in range(16 * j, 16 * j + 16))
            b.table[i, j] = b.table[i, j] if seen else 2 ** 31 - 1 - j
    b2 = b.run(backend, window, sinks)
    for i, (n, m) in enumerate(zip(new, lens)):
        b.table[i] = np.where(b.table[i] > 10 ** 6, 0, b.table[i])
    want, tol = b.want(window, sinks)
    assert (np.abs(b2 - want) <= tol).all()


@pytest.mark.parametrize("dtype,window,sinks", [("bf16", 1, 0), ("f16", 33, 5), ("bf16", 100, 0), ("f16", 100, 70), ("bf16", 500, 17), ("f16", 2000, 4)])
def test_windows_of_large_calls(backend, dtype, window, sinks):
    """Windows over prompts whose keys are opened first (some of their tokens are compared). What no token of a request sees is not finite, and
    page entries there are out of range."""
    new, lens = [1300, 1, 900, 1300, 40], [1300, 50, 1500, 2205, 90]
    b = Batch(dtype, 32, 8, 128, 16, new, lens, seed=window)
    clean = [c.copy() for c in b.scales]
    table = b.table.copy()
    for i, (n, m) in enumerate(zip(new, lens)):
        for j in range(sinks, max(m - n - window + 1, 0)):
            for d in b.scales:
                d[table[i, j // 16], :, j % 16] = np.float16("nan")
        for j in range(-(-sinks // 16), max(m - n - window + 1, 0) // 16):
            b.table[i, j] = 2 ** 31 - 1 - j
    got = b.run(backend, window, sinks)
    b.scales, b.table = clean, table
    k, v = b.values()
    for i, (n, m) in enumerate(zip(new, lens)):
        kk, vv = (R.rows_of(c, table[i], m, 16) for c in (k, v))
        for t in sorted({0, min(1, n - 1), max(n - 2, 0), n - 1, window % n, (window + 1) % n} | set(range(7, n, 211))):
            q = b.q[b.start[i] + t:b.start[i] + t + 1].float().numpy()
            o, spread, reach = R.attend(q, kk, vv, m - n + t, 128 ** -0.5, window, sinks)
            tol = K4.bound(dtype, 128, m, n * 4 > 96, o, spread, reach, np.abs(np.nan_to_num(vv)).max())
            assert (np.abs(got[b.start[i] + t] - o[0]) <= tol[0]).all(), (i, t)


def test_tokens_that_see_nothing(backend):
    """More tokens than keys: the first rows are zeros. Requests without tokens, without keys."""
    for new, kv in [([3, 1], [2, 0]), ([40, 0, 2], [5, 9, 0]), ([200], [100]), ([1], [-4])]:
        want, tol = Batch("bf16", 8, 2, 64, 16, new, [max(n, 0) for n in kv]).want()
        for wide in (False, True):
            got = Batch("bf16", 8, 2, 64, 16, new, kv).run(backend, wide=wide)
            assert (np.abs(got - want) <= tol).all()
            at = 0
            for n, m in zip(new, kv):
                assert (got[at:at + max(0, n - max(m, 0))] == 0).all()
                at += n


def test_rows_outside_every_request(backend):
    """Rows before, behind and between the requests stay as they are."""
    for n in (1, 200):
        c = Batch("bf16", 4, 1, 64, 16, [2, n, 2], [20, n + 30, 7])
        want, tol = c.want()
        c.table, c.kv = c.table[[0, 2]], [c.kv[0], c.kv[2]]
        c.start = np.array([0, 2, 2 + n + 2], np.int32)  # the second request takes the tokens in between as its own first ones
        for wide in (False, True):
            off = np.abs(c.run(backend, wide=wide) - want) - tol  # (its last two tokens see what they saw, by another kernel where there are many)
            assert off[:2].max() <= 0 and off[-2:].max() <= 0
        c.table, c.kv, c.start = c.table[:1], c.kv[:1], np.array([0, 2], np.int32)
        for wide in (False, True):
            assert (c.run(backend, wide=wide)[2:] == 7).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_strides_and_alignment(backend, dtype):
    for pad, shift, out_pad, out_shift in [(256, 0, 0, 0), (1, 0, 0, 0), (0, 3, 0, 1), (5, 1, 3, 2), (8, 8, 4, 4), (0, 0, 2, 2)]:
        for new, kv in [([1, 1], [100, 33]), ([9, 150], [40, 160])]:
            Batch(dtype, 8, 2, 96, 16, new, kv, seed=pad).check(backend, pad=pad, shift=shift, out_pad=out_pad, out_shift=out_shift)


def test_pages_out_of_range(backend):
    """An entry out of range reads as keys and values of 0."""
    for new, kv in [([1, 1], [100, 64]), ([120, 3], [150, 64])]:
        b = Batch("bf16", 4, 1, 64, 16, new, kv, poison=False)
        z = b.codes[0].shape[0]
        for i in range(2):
            b.codes[i] = np.concatenate([b.codes[i], np.full_like(b.codes[i][:1], 8)])
            b.scales[i] = np.concatenate([b.scales[i], np.zeros_like(b.scales[i][:1])])
        b.table[0, 2] = b.table[1, 0] = z
        want, tol = b.want()
        for i in range(2):
            b.codes[i], b.scales[i] = b.codes[i][:-1], b.scales[i][:-1]
        for bad in (z, -1, 2 ** 31 - 1, -2 ** 31):
            b.table[0, 2] = b.table[1, 0] = bad
            for wide in (False, True):
                assert (np.abs(b.run(backend, wide=wide) - want) <= tol).all()


@pytest.mark.parametrize("new,kv", [([1, 1, 1], [70, 40, 333]), ([30, 1, 5], [70, 40, 333]), ([300, 1, 120], [350, 40, 120])])
def test_blocks_that_are_not_finite(backend, new, kv):
    """A value's block with scale NaN or Inf: NaN in its elements for every token that sees it, nothing for the others; a key's: the whole
    row of the heads that read it."""
    for window, sinks, wide in ((0, 0, False), (0, 0, True), (50, 3, False)):
        for which in range(2):
            b = Batch("bf16", 8, 2, 96, 16, new, kv, seed=4)
            hit = []
            for i, j, head, block, bad in [(0, 33, 0, 1, "nan"), (0, kv[0] - 1, 1, 0, "inf"), (1, 0, 1, 2, "-inf"), (2, 100, 0, 0, "nan")]:
                b.scales[which][b.table[i, j // 16], head, j % 16, block] = np.float16(bad)
                hit.append((i, j, head, block))
            want = np.zeros((b.tokens, 8, 96), bool)
            for i, j, head, block in hit:
                for t in range(new[i]):
                    if R.visible(kv[i] - new[i] + t, j, window, sinks):
                        a = slice(None) if which == 0 else slice(32 * block, 32 * block + 32)
                        want[b.start[i] + t, 4 * head:4 * head + 4, a] = True
            got = b.run(backend, window, sinks, wide=wide)
            assert np.array_equal(np.isnan(got), want) and not np.isinf(got).any()
            for i, j, head, block in hit:
                b.scales[which][b.table[i, j // 16], head, j % 16, block] = 0
            ref, tol = b.want(window, sinks)
            clean = ~want
            if which == 1:  # (a key of zeros would still take weight)
                assert (np.abs(got - ref)[clean] <= tol[clean]).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_scales_that_append_does_not_write(backend, dtype):
    """Scales of eleven bits. Values are then (c - 8) d in 15 bits: exact in requests of few rows, rounded once in long ones, by half a step, keys
    and values alike (a key's rounding moves its score by half a step of its absolute sum)."""
    b = Batch(dtype, 8, 2, 96, 32, [1, 3, 40, 130], [70, 333, 300, 513], seed=21, size=0.5)
    rng = np.random.default_rng(2)
    b.scales = [np.where(np.isnan(d), d, (d.astype(np.float64) * (1 + rng.random(d.shape) / 16)).astype(np.float16)) for d in b.scales]
    want, tol = b.want()
    k, v = b.values()
    for i, (n, m) in enumerate(zip(b.new, b.kv)):
        if n * 4 > 96:
            kk, vv = (R.rows_of(c, b.table[i], m, b.page) for c in (k, v))
            _, spread, reach = R.attend(b.q[b.start[i]:b.start[i + 1]].float().numpy(), kk, vv, m - n, b.dim ** -0.5)
            half = K4.HALF[dtype]
            tol[b.start[i]:b.start[i + 1]] += (1 + half) * half * spread * (1 + 2 * reach)
    for wide in (False, True):
        assert (np.abs(b.run(backend, wide=wide) - want) <= tol).all()


def test_sizes_of_values(backend):
    """Values from f16's smallest scales to its largest, growing and falling along the keys: weights times scales must neither
    overflow nor vanish."""
    for dtype in ("bf16", "f16"):
        for new in (1, 6, 130):
            for size in (2.0 ** -18, 1e-3, 1.0, 1000.0, 60000.0):
                b = Batch(dtype, 4, 1, 64, 16, [new], [400], seed=int(size) % 7)
                c, d = K4.quantize((torch.randn(b.codes[1].shape, generator=torch.Generator().manual_seed(1)) * size / 4).numpy())
                live = np.isfinite(b.scales[1])
                b.codes[1], b.scales[1] = c, np.where(live, d, b.scales[1])
                if size * 4 < 65504 or dtype == "bf16":
                    b.check(backend)
            for up in (True, False):
                b = Batch(dtype, 4, 1, 64, 16, [new], [600], seed=8)
                for j in range(600):
                    e = (j if up else 599 - j) / 600 * 22 - 14
                    at = (b.table[0, j // 16], slice(None), j % 16)
                    x = b.values()[1][at] if j == 0 else None
                    d = b.scales[1][at].astype(np.float64) * 2.0 ** np.floor(e)
                    b.scales[1][at] = np.clip(d, -7936, 7936).astype(np.float16)
                b.check(backend)


def test_small_weights_behind_a_key_that_outweighs_them(backend):
    """One key 12 to 24 nats above the rest, with values of 0: the rest's sum is the result."""
    for dtype in ("bf16", "f16"):
        for new in (1, 5):
            for gap in (12.0, 17.4, 24.0):
                b = Batch(dtype, 2, 1, 64, 16, [new], [3000], seed=5, poison=False)
                b.codes[0][:], b.scales[0][:] = 8, np.float16(0)
                at = (b.table[0, 0], 0, 3)
                b.codes[0][at], b.scales[0][at[0], 0, 3] = 8, np.float16(0)
                b.codes[0][at[0], 0, 3, 0], b.scales[0][at[0], 0, 3, 0] = 0, np.float16(-1.0)  # element 0 is 8
                b.codes[1][at], b.scales[1][at[0], 0, 3] = 8, np.float16(0)
                b.q[:] = 0
                b.q[..., 0] = 1.0
                b.check(backend, scale=gap / 8)


def test_far_scores(backend):
    """Large scores, next to each other and far apart; scales of the softmax from tiny to large."""
    for dtype in ("bf16", "f16"):
        for new in (1, 7, 140):
            for scale in (1e-20, 1e-3, 1.0, 30.0):
                b = Batch(dtype, 4, 1, 64, 16, [new], [300], seed=9)
                want, _ = b.want(scale=scale)
                _, tol = b.want(scale=scale)
                for wide in (False, True):
                    assert (np.abs(b.run(backend, scale=scale, wide=wide) - want) <= np.minimum(tol, 50)).all()
            b = Batch(dtype, 4, 1, 64, 16, [new], [300], seed=10)
            b.q = (b.q.float() * 1000).to(TORCH[dtype])
            want, tol = b.want()
            for wide in (False, True):
                got = b.run(backend, wide=wide)
                assert np.isfinite(got).all() and (np.abs(got - want) <= np.minimum(tol, 50)).all()


def test_q_of_any_size(backend):
    """q from 1e-30 to 1e30 in bf16 (scores made of the same size by the scale), zeros, and very different elements in one row."""
    for e in (-30, -10, 10, 25):
        b = Batch("bf16", 4, 1, 64, 16, [1, 4], [100, 130], seed=11)
        b.q = (b.q.float() * 10.0 ** e).to(torch.bfloat16)
        b.check(backend, scale=float(0.125 * 10.0 ** -e))
    b = Batch("bf16", 4, 1, 64, 16, [1, 4], [100, 130], seed=11)
    b.q[..., ::3] = 0
    b.q[..., 1] *= 2.0 ** -20
    b.q[0] = 0
    b.check(backend)


def test_q_that_is_not_finite(backend):
    """A NaN in a row of q is NaN in that head's row, and nowhere else."""
    for new, kv, wide in (([2, 1], [50, 20], False), ([60, 1], [70, 20], False), ([60, 1], [70, 20], True)):
        b = Batch("bf16", 8, 2, 64, 16, new, kv, seed=12)
        clean = b.run(backend, wide=wide)
        b.q[1, 3, 5] = float("nan")
        got = b.run(backend, wide=wide)
        want = np.zeros(got.shape, bool)
        want[1, 3] = True
        assert np.array_equal(np.isnan(got), want) and np.array_equal(got[~want], clean[~want])


def test_cache_past_32_bits(backend):
    """Planes of over 4 GiB, the keys in their last pages; tokens and a prompt."""
    pages, page, heads, dim = 1000, 4096, 8, 256
    k, v = (torch.zeros((pages, heads, page // 16, 9 * dim), dtype=torch.uint8, device=DEV) for _ in range(2))
    assert k.numel() > 1 << 32
    small = Batch("bf16", 8, 8, dim, 16, [1, 40], [50, 60], seed=13)
    c = [K4.pack(a, s, w) for a, s, w in zip(small.codes, small.scales, (False, True))]
    for plane, tiles in zip((k, v), c):
        for i, n in enumerate((50, 60)):
            for j in range(-(-n // 16)):
                plane[pages - 1 - i, :, j] = torch.from_numpy(tiles[small.table[i, j], :, 0]).to(DEV)
    kv = tcb_amd.KV4Cache(pages, page, heads, dim, k.data_ptr(), v.data_ptr())
    table = torch.tensor([[pages - 1], [pages - 2]], dtype=torch.int32, device=DEV)
    q, out = small.q.to(DEV), torch.empty((41, 8 * dim), dtype=torch.bfloat16, device=DEV)
    start, lens = torch.from_numpy(small.start).to(DEV), torch.tensor([50, 60], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    backend.KV4Attention(kv, q.data_ptr(), tcb_amd.BF16, 8 * dim, out.data_ptr(), 8 * dim, 41, 8, 2, start.data_ptr(), lens.data_ptr(), table.data_ptr(), 1, max_new=40)
    backend.ctx.sync()
    want, tol = small.want()
    assert (np.abs(out.float().cpu().numpy().reshape(41, 8, dim) - want) <= tol).all()


def test_starts_and_lengths_of_any_kind(backend):
    """Starts out of order, negative, past the tokens; lengths past the table: nothing is read or written out of range."""
    b = Batch("bf16", 8, 2, 64, 16, [1, 4, 9, 150], [40, 60, 9, 160], seed=14, poison=False)
    b.table = np.where(b.table < 0, 0, b.table)
    start, kv = b.start.copy(), list(b.kv)
    for wide in (False, True):
        good = b.run(backend, wide=wide)
        for bad in ([0, -5, 400, 3, 164], [164, 14, 5, 1, 0], [2 ** 31 - 1, -2 ** 31, 7, 0, 2 ** 31 - 1], [0, 164, 0, 164, 0]):
            b.start = np.array(bad, np.int32)
            b.run(backend, wide=wide)
        b.start, b.kv = start, [2 ** 31 - 1, -2 ** 31, 10 ** 6, 161]
        b.run(backend, wide=wide)
        b.kv = kv
        assert np.array_equal(b.run(backend, wide=wide), good)


def test_captured(backend):
    """A replayed graph follows lengths, starts, tables and rows, with other work and another graph of the same context in between."""
    lib = _lib.lib()
    graphs = []
    for new, kv, wide in (([1] * 6, [100, 7, 33, 1, 900, 64], False), ([120, 1, 7], [130, 40, 300], False), ([120, 1, 7], [130, 40, 300], True)):
        b = Batch("bf16", 8, 2, 128, 16, new, kv, seed=15)
        b.table = b.wide_table() if wide else b.table
        b.most = b.table.shape[1]
        k, v = b.planes()
        q = torch.zeros((b.tokens, 8 * 128), dtype=torch.bfloat16, device=DEV)
        out = torch.zeros_like(q)
        start, lens, table = (torch.zeros(s, dtype=torch.int32, device=DEV) for s in ((len(new) + 1,), (len(new),), b.table.shape))
        cache = tcb_amd.KV4Cache(k.shape[0], 16, 2, 128, k.data_ptr(), v.data_ptr())

        def step(cache=cache, q=q, out=out, start=start, lens=lens, table=table, b=b, new=new):
            backend.KV4Attention(cache, q.data_ptr(), tcb_amd.BF16, 1024, out.data_ptr(), 1024, b.tokens, 8, len(new), start.data_ptr(), lens.data_ptr(),
                                 table.data_ptr(), b.most, max_new=max(new))
        torch.cuda.synchronize()
        step()
        g = ctypes.c_void_p()
        assert lib.trhip_graph_begin(backend.ctx.h) == 0
        step()
        assert lib.trhip_graph_end(backend.ctx.h, ctypes.byref(g)) == 0
        graphs.append((b, g, q, out, start, lens, table, (k, v)))
    for i in range(4):
        for b, g, q, out, start, lens, table, _ in graphs:
            keep = list(b.kv)
            b.kv = [max(n, m - 3 * i) for n, m in zip(b.new, b.kv)]
            b.q = torch.randn(b.q.shape, generator=torch.Generator().manual_seed(i)).to(torch.bfloat16)
            q.copy_(b.q.view(b.tokens, -1)), start.copy_(torch.from_numpy(b.start)), lens.copy_(torch.tensor(b.kv)), table.copy_(torch.from_numpy(b.table))
            torch.cuda.synchronize()
            assert lib.trhip_graph_launch(backend.ctx.h, g) == 0
            backend.ctx.sync()
            want, tol = b.want()
            assert (np.abs(out.float().cpu().numpy().reshape(want.shape) - want) <= tol).all(), i
            b.kv = keep
        Batch("f16", 4, 1, 64, 16, [1, 30], [2000, 30], seed=i).check(backend)
    for t in graphs:
        assert lib.trhip_graph_destroy(t[1]) == 0


def test_two_contexts_at_once():
    """Two contexts on two threads, each with its own workspaces."""
    wrong = []

    def work(seed):
        tb = tcb_amd.QuantBackend(0)
        try:
            b = Batch("bf16", 8, 2, 128, 16, [1, 1, 50, 130], [3000, 70, 60, 700], seed=seed)
            want, tol = b.want()
            for i in range(10):
                if not (np.abs(b.run(tb, wide=i % 2 == 0) - want) <= tol).all():
                    wrong.append(seed)
        except Exception as e:  # (a thread's exception is not seen otherwise)
            wrong.append(e)
        tb.close()
    threads = [threading.Thread(target=work, args=(s,)) for s in (1, 2)]
    [t.start() for t in threads], [t.join() for t in threads]
    assert not wrong


def test_same_bits_every_time(backend):
    b = Batch("f16", 8, 2, 128, 16, [1, 1, 30, 1], [9000, 70, 60, 2000], seed=16)
    for wide in (False, True):
        first = b.run(backend, wide=wide)
        for _ in range(5):
            assert np.array_equal(b.run(backend, wide=wide), first)


def test_refusals(backend):
    x, i = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    p, n = x.data_ptr(), i.data_ptr()
    cache = dict(pages=2, page=16, heads=2, dim=64, k=p, v=p + (1 << 15))
    good = dict(q=p, qtype=tcb_amd.BF16, q_stride=256, out=p + 4096, out_stride=256, tokens=2, heads=4, nreq=1, q_start=n, kv_len=n, table=n, max_pages=2)

    def refused(code=_lib.ERR_INVALID, kv={}, **change):
        with pytest.raises(TrhipError) as e:
            backend.KV4Attention(tcb_amd.KV4Cache(**{**cache, **kv}), **{**good, **change})
        assert e.value.code == code
    refused(_lib.ERR_UNSUPPORTED, qtype=tcb_amd.F32)
    refused(_lib.ERR_UNSUPPORTED, kv=dict(dim=80))
    refused(kv=dict(page=8))
    refused(kv=dict(k=p + 8))
    refused(heads=3)
    refused(heads=0)
    refused(tokens=-1)
    refused(tokens=2 ** 31 // 4)
    refused(nreq=-1)
    refused(max_pages=-1)
    refused(max_pages=2 ** 27)
    refused(window=-1)
    refused(window=2 ** 31)
    refused(sinks=-1)
    refused(sinks=2 ** 31)
    refused(max_new=-1)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(scale=scale)
    refused(q_stride=255)
    refused(out_stride=255)
    for name in ("q", "out", "q_start", "kv_len", "table"):
        refused(**{name: 0})
    refused(q=p + 1)
    refused(out=p + 1)
    backend.KV4Attention(tcb_amd.KV4Cache(**cache), **{**good, "tokens": 0})
    backend.KV4Attention(tcb_amd.KV4Cache(**cache), **{**good, "nreq": 0})
