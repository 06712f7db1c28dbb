"""Sampling (trhip_sample) against the definition in 64 bits."""
import ctypes
import math
import threading

import numpy as np
import pytest
import torch

import tcb_amd
from tcb_amd import TrhipError, _lib

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": tcb_amd.F32, "bf16": tcb_amd.BF16, "f16": tcb_amd.F16}
DEV = "cuda:0"
CLOSE = 1e-12  # of the sum: nearer to a border than this, either side is right


def choose(x, t, k, p, low, u):
    """(token, logprob, whether a border is so close that 64 bits do not decide) of one row. (Sums in 80 bits: a hundred thousand additions
    to about 1 would each round by 2^-54, all in one direction where they are equal.)"""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, math.nan, False
    if not t > 0:
        return int(order[0]), 0.0, False
    if 0 < k < len(order):
        order = order[:k]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == x[order[0]], 1.0, np.exp((x[order] - x[order[0]]) / t)).astype(np.longdouble)
    close, n = False, len(order)
    if p < 1:
        run = np.cumsum(w)
        goal = p * run[-1]
        n = max(1, min(n, int(np.searchsorted(run, goal, side="left")) + 1))
        close = bool((np.abs(run - goal) <= CLOSE * run[-1]).any())
    if low > 0:
        n = min(n, max(1, int((w >= min(low, 1.0)).sum())))
        close = close or bool((np.abs(w - min(low, 1.0)) <= CLOSE)[1:].any() and low < 1)
    keep = np.sort(order[:n])
    where = {i: y for i, y in zip(order[:n].tolist(), w[:n].tolist())}
    w = np.array([where[i] for i in keep.tolist()])
    run = np.cumsum(w)
    goal = max(u, 0.0) * run[-1] if u == u else np.longdouble(0)
    over = np.nonzero(run > goal)[0]
    at = int(over[0]) if len(over) else int(np.nonzero(w > 0)[0][-1])
    if 0 < u < 1:
        close = close or bool((np.abs(run - goal) <= CLOSE * run[-1]).any())
    return int(keep[at]), math.log(w[at] / run[-1]) if w[at] > 0 else -math.inf, close


def sample(tb, x, u, t=None, k=None, p=None, low=None, pad=0, shift=0, logprob=True):
    rows, vocab = x.shape
    buf = torch.full((shift + rows * (vocab + pad) + 8,), 1e4, dtype=x.dtype, device=DEV)
    buf[shift:shift + rows * (vocab + pad)].view(rows, vocab + pad)[:, :vocab] = x.to(DEV)
    f = [None if a is None else torch.tensor(a, dtype=d, device=DEV) for a, d in ((t, torch.float32), (k, torch.int32), (p, torch.float32), (low, torch.float32), (u, torch.float32))]
    token, lp = torch.full((rows + 2,), 77, dtype=torch.int32, device=DEV), torch.full((rows + 2,), 77.0, device=DEV)
    torch.cuda.synchronize()
    a = [None if y is None else y.data_ptr() for y in f]
    io = {v: CODE[n] for n, v in TORCH.items()}[x.dtype]
    tb.Sample(buf.data_ptr() + shift * buf.element_size(), io, vocab + pad, rows, vocab, a[4], token.data_ptr() + 4, lp.data_ptr() + 4 if logprob else None,
              temperature=a[0], top_k=a[1], top_p=a[2], min_p=a[3])
    tb.ctx.sync()
    token, lp = token.cpu().numpy(), lp.cpu().numpy()
    assert token[0] == token[-1] == 77 and lp[0] == lp[-1] == 77
    return token[1:-1], lp[1:-1]


def check(tb, x, u, t=None, k=None, p=None, low=None, **how):
    """x [rows, vocab] (torch, on the CPU); settings: lists of one value a row, or None."""
    token, lp = sample(tb, x, u, t, k, p, low, **how)
    y = x.double().numpy()
    near = 0
    for r in range(len(y)):
        f = lambda a, d: d if a is None else float(np.float32(a[r]))  # noqa: E731
        want, log, close = choose(y[r], f(t, 1.0), 0 if k is None else k[r], f(p, 1.0), f(low, 0.0), float(np.float32(u[r])))
        if close:
            near += 1
            continue
        assert token[r] == want, (r, token[r], want, f(t, 1.0), k and k[r], p and p[r], low and low[r], u[r])
        if math.isnan(log):
            assert math.isnan(lp[r])
        else:  # rounded once, from 64 bits
            assert lp[r] == log or abs(lp[r] - log) <= 2.0 ** -23 * abs(log) + 1e-11, (r, lp[r], log)
    assert near <= len(y) // 4 + 1


def zipf(rows, vocab, seed, steep=(1.1, 2.3)):
    g = torch.Generator().manual_seed(seed)
    a = torch.linspace(*steep, rows)
    return torch.stack([10 - a[r] * (torch.randperm(vocab, generator=g) + 1.0).log() + 0.3 * torch.randn(vocab, generator=g) for r in range(rows)])


def settings(rows, seed):
    rng = np.random.default_rng(seed)
    t = rng.choice([0.0, 0.3, 0.7, 1.0, 1.0, 1.7, 5.0], rows).tolist()
    k = rng.choice([0, 0, 1, 2, 5, 40, 300, 5000, 10 ** 6], rows).tolist()
    p = rng.choice([1.0, 0.0, 0.1, 0.5, 0.9, 0.95, 0.999, 1.5], rows).tolist()
    low = rng.choice([0.0, 0.0, 0.01, 0.1, 0.5, 1.0], rows).tolist()
    return t, k, p, low, rng.random(rows).astype(np.float32).tolist()


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("vocab", [1, 2, 3, 63, 64, 65, 255, 1000, 1023, 1024, 1025, 4097, 8191, 32000, 50257, 128256, 151936])
def test_settings(backend, dtype, vocab):
    """Every mix of settings, peaked and flat rows; in 16 bits many logits are equal."""
    rows = 48 if vocab < 20000 else 24
    print(dtype, vocab, flush=True)
    x = zipf(rows, vocab, vocab).to(TORCH[dtype])
    t, k, p, low, u = settings(rows, vocab)
    check(backend, x, u, t, k, p, low)
    check(backend, x, u)
    check(backend, x, u, t=t)
    check(backend, x, u, k=k)
    check(backend, x, u, p=p)
    check(backend, x, u, low=low)
    check(backend, x, u, t, p=p)


@pytest.mark.parametrize("vocab", [700, 9000, 128256])
def test_flat_rows(backend, vocab):
    """Rows where nearly everything is kept, and rows of a few equal values (ties at every border, by index)."""
    g = torch.Generator().manual_seed(vocab)
    for x in (torch.zeros((16, vocab)), torch.randn((16, vocab), generator=g) * 0.01, torch.randint(0, 3, (16, vocab), generator=g).float(),
              torch.randn((16, vocab), generator=g), torch.randn((16, vocab), generator=g) * 3):
        t, k, p, low, u = settings(16, vocab + 1)
        check(backend, x, u, [max(a, 0.2) for a in t], k, p, low)
        check(backend, x, u, p=[0.3 + 0.04 * i for i in range(16)])
        check(backend, x, u, k=[1 + (vocab // 2 * i) // 9 for i in range(16)])
        check(backend, x.to(torch.bfloat16), u, k=[3 + 97 * i for i in range(16)], p=[0.99] * 16)


def test_ties_at_the_cut_of_top_k(backend):
    """Large entries in few stripes and many equal ones at the border of top_k, then top_p among them: the lowest indexes of the equal ones."""
    g, vocab, rows = torch.Generator().manual_seed(12), 60000, 24
    x = torch.randn((rows, vocab), generator=g)
    for r in range(rows):
        at = 256 * (r * 7 % 200)
        x[r, at:at + 700] = 5 + torch.rand(700, generator=g)  # more in a workgroup than its share
        x[r, torch.randperm(vocab, generator=g)[:3000]] = 4.5
    x[:, 0] = 9
    k, p = [300 + 60 * r for r in range(rows)], [0.5 + 0.02 * r for r in range(rows)]
    u = torch.rand(rows, generator=g).tolist()
    check(backend, x, u, k=k)
    check(backend, x, u, k=k, p=p)
    check(backend, x, u, k=k, p=[0.999] * rows, low=[0.001 * r for r in range(rows)])
    check(backend, x, u, p=p)
    check(backend, x.bfloat16(), u, k=k, p=p)
    check(backend, x.bfloat16(), u, p=p)


def test_around_zero(backend):
    """Cuts at -0, 0 and the smallest numbers, many of each; and rows of nothing but negative or positive values."""
    g = torch.Generator().manual_seed(4)
    some = torch.tensor([-1.0, -1e-38, -1e-45, -0.0, 0.0, 1e-45, 1e-38, 1.0])
    for vocab in (300, 9000, 130000):
        x = some[torch.randint(0, 8, (12, vocab), generator=g)]
        u = [(2 * i + 1) / 24 for i in range(12)]
        check(backend, x, u, k=[1 + vocab * i // 12 for i in range(12)])
        check(backend, x, u, p=[0.05 + 0.08 * i for i in range(12)])
        check(backend, x, u, k=[1 + vocab * (i + 1) // 13 for i in range(12)], p=[0.97 - 0.08 * i for i in range(12)])
        y = torch.randn((12, vocab), generator=g) * 0.5
        for z in (y - 40.0, y + 40.0, y * 1e-3, y * 1e-41):
            check(backend, z, u, p=[0.05 + 0.08 * i for i in range(12)])
            check(backend, z, u, k=[1 + vocab * i // 12 for i in range(12)], low=[0.1] * 12)


def test_order_of_the_rows_values(backend):
    """The largest first, last, in the middle; falling and rising rows; only one entry of weight."""
    for vocab in (100, 5000, 70000):
        up = torch.linspace(-30, 30, vocab)
        one = torch.full((vocab,), -200.0)
        one[vocab // 3] = 50.0
        x = torch.stack([up, up.flip(0), one, up[torch.randperm(vocab, generator=torch.Generator().manual_seed(1))]])
        for u in (0.0, 0.3, 0.999999):
            for k, p in ((None, None), ([7] * 4, None), (None, [0.9] * 4), ([50] * 4, [0.5] * 4), ([vocab - 1] * 4, [0.99999] * 4)):
                check(backend, x, [u] * 4, k=k, p=p)


def test_borders_of_u(backend):
    """u of 0 takes the first that is kept, of 1 and above the last with weight, below 0 and NaN are 0."""
    x = torch.tensor([[-800.0, 1.0, 2.0, float("-inf"), 0.5, -900.0]])
    for u, want in ((0.0, 1), (-1.0, 1), (float("nan"), 1), (1.0, 4), (2.0, 4), (float("inf"), 4)):
        token, lp = sample(backend, x, [u])
        assert token[0] == want and abs(lp[0] - math.log(math.exp(x[0, want]) / (math.e + math.e ** 2 + math.e ** 0.5))) < 1e-6
    token, _ = sample(backend, torch.tensor([[-5.0, 1.0, 2.0, -4.0]]), [0.0], k=[2])
    assert token[0] == 1
    # a weight of e^-700 counts where u is 0
    token, lp = sample(backend, torch.tensor([[-700.0, 0.0]]), [0.0])
    assert token[0] == 0 and abs(lp[0] + 700) < 1e-3


def test_values_that_are_not_finite(backend):
    inf, nan = float("inf"), float("nan")
    rows = [[nan, 1.0, nan, 2.0], [-inf] * 4, [nan] * 4, [nan, -inf, nan, -inf], [inf, 0.0, inf, 3.0], [-inf, -inf, -5.0, nan], [3.4e38, -3.4e38, 0.0, -0.0],
            [-0.0, 0.0, -0.0, 0.0]]
    x = torch.tensor(rows)
    for u in (0.0, 0.49, 0.51, 0.999):
        for kw in ({}, dict(k=[1] * 8), dict(p=[0.6] * 8), dict(low=[0.5] * 8), dict(k=[3] * 8, p=[0.9] * 8), dict(t=[0.0] * 8), dict(t=[nan] * 8), dict(t=[-1.0] * 8),
                   dict(t=[1e-40] * 8), dict(t=[1e30] * 8), dict(p=[nan] * 8), dict(low=[nan] * 8), dict(p=[-1.0] * 8), dict(k=[-3] * 8)):
            check(backend, x, [u] * 8, **kw)
    x = torch.cat([x.repeat(1, 1000), x], 1)
    for kw in ({}, dict(k=[5] * 8), dict(p=[0.5] * 8), dict(low=[0.5] * 8)):
        check(backend, x, [0.7] * 8, **kw)


@pytest.mark.parametrize("dtype", ["f32", "f16"])
def test_temperatures_of_any_size(backend, dtype):
    """Infinite ones, the largest and the smallest, with logits that are infinite too: entries of +Inf are alone where there are some."""
    g, ts = torch.Generator().manual_seed(8), [float("inf"), 3e38, 1e38, 1e30, 1e-30, 1e-38, 1e-45]
    for vocab in (300, 9000, 128256):
        x = (torch.randn((3 * len(ts), vocab), generator=g) * 3).to(TORCH[dtype])
        x[1::3, 5] = x[1::3, vocab // 2] = float("inf")
        x[1::3, 9] = x[2::3, 7] = float("-inf")
        x[2::3, ::2] = 0.0
        rows = len(x)
        u, t = torch.rand(rows, generator=g).tolist(), [a for a in ts for _ in range(3)]
        alone = x.float()
        alone[1::3] = torch.where(alone[1::3] == float("inf"), 0.0, float("-inf"))
        alone = alone.double().numpy()
        for k, p in (([0] * rows, [1.0] * rows), ([0] * rows, [0.6] * rows), ([50] * rows, [0.6] * rows), ([2000] * rows, [0.9] * rows)):
            token, lp = sample(backend, x, u, t, k, p)
            for r in range(rows):
                want, log, close = choose(alone[r], float(np.float32(t[r])), k[r], float(np.float32(p[r])), 0.0, float(np.float32(u[r])))
                assert close or (token[r] == want and abs(lp[r] - log) <= 2.0 ** -23 * abs(log) + 1e-11), (vocab, t[r], k[r], p[r], r % 3, token[r], want)


def test_sums_of_many_small_weights(backend):
    """One large logit, then tens of thousands of equal small ones at several heights: borders of top_p among them, where each weighs some
    1e-9 of the sum (a rounding of each to a common unit would be off by whole entries)."""
    g, vocab, rows = torch.Generator().manual_seed(4), 128256, 48
    x = torch.full((rows, vocab), -40.0)
    for h, heights in enumerate(([-20.53, -20.61, -20.74, -20.87, -20.95, -21.02], [-24.1, -24.4, -25.3, -26.2, -26.9, -27.7])):
        for i, y in enumerate(heights):
            x[h::2, 20000 * i:20000 * (i + 1)] = y
    x = x[:, torch.randperm(vocab, generator=g)]
    x[:, 77] = 0.0
    w = torch.exp(x.double())
    tail = (w.sum(1) - 1) / w.sum(1)
    p = (1 - tail * torch.linspace(0.02, 0.98, rows, dtype=torch.float64)).float()
    u = (1 - tail * torch.rand(rows, generator=g).double()).float()
    check(backend, x, u.tolist(), p=p.tolist())
    check(backend, x, u.tolist(), k=[110000 - 300 * r for r in range(rows)], p=p.tolist())
    check(backend, x + 5, [0.999] * rows, t=[3.0] * rows, p=torch.linspace(0.4, 0.97, rows).tolist())
    check(backend, x + 5, [0.999] * rows, t=[3.0] * rows, k=[110000 - 300 * r for r in range(rows)], p=torch.linspace(0.4, 0.97, rows).tolist())


def test_no_temperature_is_the_first_largest(backend):
    x = torch.tensor([[1.0, 5.0, 5.0, 2.0], [5.0, 5.0, 5.0, 5.0], [-9.0, -8.0, -8.0, -8.0]])
    token, lp = sample(backend, x, [0.9] * 3, t=[0.0] * 3, k=[3] * 3, p=[0.99] * 3)
    assert token.tolist() == [1, 0, 1] and (lp == 0).all()
    big = torch.zeros((2, 100000))
    big[0, 77777] = big[0, 99999] = 1.0
    token, _ = sample(backend, big, [0.9] * 2, t=[0.0] * 2)
    assert token.tolist() == [77777, 0]


def test_strides_and_alignment(backend):
    for dtype in TORCH:
        for vocab, pad, shift in [(1000, 24, 0), (1001, 0, 0), (1001, 0, 1), (5003, 7, 3), (128256, 1, 0), (33000, 0, 5), (128, 8, 2)]:
            x = zipf(6, vocab, 5).to(TORCH[dtype])
            t, k, p, low, u = settings(6, pad + shift)
            check(backend, x, u, t, k, p, low, pad=pad, shift=shift)


def test_many_rows(backend):
    for rows, vocab in [(256, 2000), (1000, 300), (300, 40000)]:
        x = zipf(rows, vocab, rows)
        t, k, p, low, u = settings(rows, rows)
        check(backend, x, u, t, k, p, low)


def test_large_vocabulary(backend):
    x = zipf(2, 3_000_001, 8)
    check(backend, x, [0.4, 0.8], k=[100, 0], p=[1.0, 0.9])
    check(backend, x, [0.4, 0.8])


def test_frequencies(backend):
    """Over many random numbers, tokens come as often as their weights say (within five standard deviations)."""
    x = torch.tensor([[0.0, 1.0, 2.0, 1.5, -1.0, 0.7]]).repeat(4096, 1)
    u = np.random.default_rng(0).random(4096).astype(np.float32)
    token, lp = sample(backend, x, u.tolist())
    w = torch.softmax(x[0].double(), 0).numpy()
    n = np.bincount(token, minlength=6)
    assert (np.abs(n - 4096 * w) <= 5 * np.sqrt(4096 * w * (1 - w))).all()
    assert np.abs(lp - np.log(w)[token]).max() < 1e-6


def test_without_logprob_and_repeatable(backend):
    x = zipf(20, 30000, 3)
    t, k, p, low, u = settings(20, 9)
    a, lp = sample(backend, x, u, t, k, p, low)
    for _ in range(3):
        b, lq = sample(backend, x, u, t, k, p, low)
        assert np.array_equal(a, b) and np.array_equal(lp, lq, equal_nan=True)
    b, lq = sample(backend, x, u, t, k, p, low, logprob=False)
    assert np.array_equal(a, b) and (lq == 77).all()


def test_captured(backend):
    """A replayed graph follows logits, settings and numbers; other work in between does not disturb it."""
    rows, vocab = 5, 33333
    x = torch.zeros((rows, vocab), device=DEV)
    t, p, low, u = (torch.zeros(rows, device=DEV) for _ in range(4))
    k, token, lp = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(rows, device=DEV)

    def step():
        backend.Sample(x.data_ptr(), tcb_amd.F32, vocab, rows, vocab, u.data_ptr(), token.data_ptr(), lp.data_ptr(), temperature=t.data_ptr(),
                       top_k=k.data_ptr(), top_p=p.data_ptr(), min_p=low.data_ptr())
    torch.cuda.synchronize()
    step()
    lib, g = _lib.lib(), ctypes.c_void_p()
    assert lib.trhip_graph_begin(backend.ctx.h) == 0
    step()
    assert lib.trhip_graph_end(backend.ctx.h, ctypes.byref(g)) == 0
    for i in range(5):
        y = zipf(rows, vocab, 50 + i, (0.2, 2.0))
        s = settings(rows, i)
        x.copy_(y)
        for d, v in zip((t, k, p, low, u), s):
            d.copy_(torch.tensor(v, dtype=d.dtype))
        torch.cuda.synchronize()
        assert lib.trhip_graph_launch(backend.ctx.h, g) == 0
        backend.ctx.sync()
        got = token.cpu().numpy()
        for r in range(rows):
            want, _, close = choose(y[r].numpy(), s[0][r], s[1][r], float(np.float32(s[2][r])), float(np.float32(s[3][r])), s[4][r])
            assert close or got[r] == want
        check(backend, zipf(40, 9000, i), [0.5] * 40)
    assert lib.trhip_graph_destroy(g) == 0


def test_two_contexts_at_once():
    """Two contexts on two threads, each with its own workspaces."""
    x, wrong = zipf(24, 50257, 3), []
    t, k, p, low, u = settings(24, 17)
    want = [choose(x[r].double().numpy(), *(float(np.float32(a[r])) if a is not k else a[r] for a in (t, k, p, low, u))) for r in range(24)]

    def work():
        tb = tcb_amd.QuantBackend(0)
        try:
            for _ in range(8):
                token, _ = sample(tb, x, u, t, k, p, low)
                wrong.extend(r for r in range(24) if not want[r][2] and token[r] != want[r][0])
        except Exception as e:  # (a thread's exception is not seen otherwise)
            wrong.append(e)
        tb.close()
    threads = [threading.Thread(target=work) for _ in range(2)]
    [a.start() for a in threads], [a.join() for a in threads]
    assert not wrong


def test_refusals(backend):
    x, i = torch.zeros(4096, device=DEV), torch.zeros(8, dtype=torch.int32, device=DEV)
    p = x.data_ptr()
    good = dict(logits=p, ltype=tcb_amd.F32, stride=100, rows=2, vocab=100, u=p, token=i.data_ptr())

    def refused(**change):
        with pytest.raises(TrhipError) as e:
            backend.Sample(**{**good, **change})
        assert e.value.code == _lib.ERR_INVALID
    refused(rows=-1)
    refused(vocab=-1)
    refused(vocab=0)
    refused(vocab=(1 << 24) + 1, stride=1 << 25)
    refused(rows=(1 << 20) + 1)
    refused(stride=99)
    refused(ltype=4)
    refused(logits=0)
    refused(u=0)
    refused(token=0)
    refused(logits=p + 2)
    refused(logits=p + 1, ltype=tcb_amd.F16)
    backend.Sample(**{**good, "rows": 0, "logits": 0, "u": 0, "token": 0})
