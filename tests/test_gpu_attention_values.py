"""Attention over a paged cache at scores, weights and values far from the ordinary (trhip_attn, trhip_attn_shared)."""
import math

import numpy as np
import pytest
import torch

import tcb_amd

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"bf16": tcb_amd.BF16, "f16": tcb_amd.F16}


class Case:
    """One request (or `reqs` of them over the same keys) of `new` tokens and `kv` keys, one kv head; k and v [kv, dim], q [new, heads, dim].
    The first `prefix` of the keys are shared ones (trhip_attn_shared)."""

    def __init__(self, dtype, heads, dim, new, kv, prefix=0, reqs=1, page=16):
        self.dtype, self.heads, self.dim, self.new, self.kv, self.prefix, self.reqs, self.page = dtype, heads, dim, new, kv, prefix, reqs, page
        t = TORCH[dtype]
        self.k, self.v = (torch.zeros((kv, dim), dtype=t) for _ in range(2))
        self.q = torch.zeros((new, heads, dim), dtype=t)

    def run(self, tb, scale, max_new=None, window=0, sinks=0):
        """Rows of the last request, float64 [new, heads, dim]."""
        t, page, own = TORCH[self.dtype], self.page, self.kv - self.prefix
        lead, pages = -(-self.prefix // page), -(-own // page)
        planes = []
        for rows in (self.k, self.v):
            x = torch.full(((lead + pages) * page, self.dim), float("nan"), dtype=t)
            x[:self.prefix], x[lead * page:lead * page + own] = rows[:self.prefix], rows[self.prefix:]
            planes.append(x.view(lead + pages, 1, page, self.dim).to(DEV))
        n, tokens = self.reqs, self.new * self.reqs
        q = self.q.repeat(n, 1, 1).contiguous().to(DEV)
        out = torch.full((tokens, self.heads, self.dim), 7.0, dtype=t, device=DEV)
        start = torch.arange(n + 1, dtype=torch.int32, device=DEV) * self.new
        lens = torch.full((n,), own, dtype=torch.int32, device=DEV)
        first = torch.arange(lead, dtype=torch.int32, device=DEV)
        table = (torch.arange(pages, dtype=torch.int32, device=DEV) + lead).repeat(n, 1).contiguous()
        kv = tcb_amd.KVCache(CODE[self.dtype], lead + pages, page, 1, self.dim, planes[0].data_ptr(), planes[1].data_ptr())
        width = self.heads * self.dim
        args = (kv, q.data_ptr(), width, out.data_ptr(), width, tokens, self.heads, n, start.data_ptr(), lens.data_ptr(), table.data_ptr(), max(pages, 1))
        max_new = self.new if max_new is None else max_new
        torch.cuda.synchronize()
        if self.prefix:
            tb.AttentionShared(*args, first.data_ptr(), self.prefix, max_new=max_new, scale=scale)
        else:
            tb.Attention(*args, max_new=max_new, window=window, sinks=sinks, scale=scale)
        tb.ctx.sync()
        return out[tokens - self.new:].double().cpu().numpy()

    def want(self, scale):
        """The formula in float64."""
        k, v, q = self.k.double().numpy(), self.v.double().numpy(), self.q.double().numpy()
        out = np.zeros((self.new, self.heads, self.dim))
        for t in range(self.new):
            see = self.kv - self.new + t + 1
            s = scale * (q[t] @ k[:see].T)
            e = np.exp(s - s.max(1, keepdims=True))
            out[t] = (e @ v[:see]) / e.sum(1, keepdims=True)
        return out


# (heads, tokens): a single token, a few rows, a prompt of rows; the kernels of few and of many rows
FORMS = [(4, 1), (8, 12), (4, 60)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads,new", FORMS)
def test_far_scores_one_step_apart(backend, dtype, dim, heads, new):
    """Scores of 2^27 + 16 and 2^27 + 32, neighbours in fp32: the later key's weight is 2^16 of the earlier one's, past the largest f16,
    and the whole answer."""
    print(dtype, dim, heads, new, flush=True)
    c = Case(dtype, heads, dim, new, 400 + new)
    c.q[:, :, 0], c.q[:, :, 1] = 2.0 ** 14, 4.0
    c.v[:] = torch.randn((c.kv, dim), generator=torch.Generator().manual_seed(dim)).to(c.v.dtype)
    for first, then in ((0, 128), (5, 384), (70, 130)):
        c.k[:] = 0
        c.k[first, 0], c.k[first, 1] = 2.0 ** 13, 4.0
        c.k[then, 0], c.k[then, 1] = 2.0 ** 13, 8.0
        got = c.run(backend, math.log(2.0))
        # (its weight is 1 - 2^-16; one rounding of the output, bf16's 2^-9, and 2^-16 of the other value)
        want = c.v[then].double().numpy()
        assert np.isfinite(got).all()
        assert (np.abs(got - want) <= 2.0 ** -9 * np.abs(want) + 2.0 ** -15 * np.abs(c.v.double().numpy()).max()).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("reqs", [1, 40])
@pytest.mark.parametrize("scale", [1e-38, 1e-45])
def test_smallest_scales(backend, dtype, reqs, scale):
    """All weights are equal: the mean over a shared prefix and the own keys behind it, whichever kernels have the two."""
    c = Case(dtype, 4, 128, 1, 400, prefix=300, reqs=reqs)
    g = torch.Generator().manual_seed(reqs)
    c.q[:], c.k[:] = (torch.randn(x.shape, generator=g).to(x.dtype) for x in (c.q, c.k))
    c.v[:300], c.v[300:] = 1.0, 5.0
    got = c.run(backend, scale)
    assert (np.abs(got - 2.0) <= 2.0 ** -8).all()  # (the mean is 2 and representable: half a unit of bf16 below it)


def dominated(heads, dim, new, kv, prefix, reqs, gap, at, seed):
    """f16: one key `gap` nats above all others, with values of 0; the others' scores are equal up to 0.5, their values about 1."""
    c = Case("f16", heads, dim, new, kv, prefix=prefix, reqs=reqs)
    g = torch.Generator().manual_seed(seed)
    c.q[:, :, 0] = 1.0
    c.k[:, 0] = 0.5 * torch.rand(kv, generator=g)
    c.v[:] = (1.0 + 0.5 * torch.randn((kv, dim), generator=g)).half()
    c.k[at, 0], c.v[at] = gap, 0.0
    return c


def formula(c):
    """(out, spread) of the formula in float64 on the device, scale 1: spread = sum_j e_j |v_j| / sum_j e_j."""
    k, v = c.k.to(DEV).double(), c.v.to(DEV).double()
    s = c.q.to(DEV).double().view(c.new * c.heads, c.dim) @ k.t().contiguous()
    see = torch.arange(c.kv, device=DEV) <= (torch.arange(c.new, device=DEV) + c.kv - c.new).repeat_interleave(c.heads).unsqueeze(1)
    e = torch.softmax(s.masked_fill(~see, -math.inf), 1)
    return [(e @ x).view(c.new, c.heads, c.dim).cpu().numpy() for x in (v, v.abs())]


@pytest.mark.parametrize("gap", [10.0, 17.4, 22.0, 30.0])
@pytest.mark.parametrize("heads,dim,new,kv,prefix,reqs,at", [
    (4, 128, 1, 131071, 0, 1, 0), (8, 64, 1, 30001, 0, 1, 17000), (4, 256, 1, 20000, 0, 3, 19999), (1, 96, 20, 9000, 0, 1, 5),
    (4, 128, 1, 20300, 20000, 1, 3), (4, 128, 1, 6000, 0, 500, 0), (4, 64, 1, 3000, 0, 700, 100), (2, 256, 1, 3000, 0, 300, 7)])
def test_small_weights_of_tokens(backend, gap, heads, dim, new, kv, prefix, reqs, at):
    """The output is what the small weights leave. Two 16-bit terms lose 2^-18 of a weight (they are on a grid of 2^-24 where a block's
    largest is 2^-7 at least), sums in fp32 2^-24 a term in numerator and denominator, exp2 and the divide 2^-20, the output's rounding
    2^-11; 31 keys beside the large one are held to 2^-31 of it."""
    print(gap, heads, dim, new, kv, prefix, flush=True)
    c = dominated(heads, dim, new, kv, prefix, reqs, gap, at, 1)
    got, (want, spread) = c.run(backend, 1.0), formula(c)
    tol = 2.0 ** -11 * np.abs(want) + spread * (2.0 ** -18 + 2 * kv * 2.0 ** -24 + 2.0 ** -20) + 32 * 2.0 ** -31 * np.abs(c.v.double().numpy()).max() + 2.0 ** -25
    off = np.abs(got - want)
    assert (off <= tol).all(), (off.max(), np.abs(want).max(), (off / tol).max())


@pytest.mark.parametrize("gap", [10.0, 17.4, 19.0])
@pytest.mark.parametrize("heads,dim,new,kv,prefix,reqs,at", [
    (4, 128, 60, 131071, 0, 1, 0), (4, 64, 60, 30001, 0, 1, 17000), (4, 256, 30, 20000, 0, 1, 5), (8, 128, 30, 250, 0, 1, 5), (4, 128, 1, 20300, 20000, 40, 3),
    (4, 128, 60, 6000, 0, 300, 0), (4, 64, 60, 3000, 0, 300, 300), (2, 256, 60, 3000, 0, 300, 300),
    (4, 256, 1, 9300, 9000, 40, 8000)])
def test_small_weights_of_many_rows(backend, gap, heads, dim, new, kv, prefix, reqs, at):
    """As above with weights rounded once: 2^-11 of a weight, or 2^-31 of the row's largest where that is more."""
    print(gap, heads, dim, new, kv, prefix, flush=True)
    c = dominated(heads, dim, new, kv, prefix, reqs, gap, at, 2)
    got, (want, spread) = c.run(backend, 1.0), formula(c)
    most = np.abs(c.v.double().numpy()).max()
    tol = 2.0 ** -11 * np.abs(want) + spread * (2.0 ** -11 + 2 * kv * 2.0 ** -24 + 2.0 ** -20) + kv * 2.0 ** -31 * most + 2.0 ** -25
    off = np.abs(got - want)
    assert (off <= tol).all(), (off.max(), np.abs(want).max(), (off / tol).max())


def test_small_and_large_blocks_in_turn(backend):
    """f16: every other block of a wave's keys 20 to 40 bits below the ones between them, of both kinds first: references go up and down."""
    for heads, new, step in ((4, 1, 128), (4, 1, 32), (4, 60, 64)):
        c = Case("f16", heads, 128, new, 6000)
        g = torch.Generator().manual_seed(step)
        c.q[:, :, 0] = 1.0
        j = torch.arange(c.kv)
        for first in (0, 1):
            print(heads, new, step, first, flush=True)
            low = (j // step) % 2 == first
            c.k[:, 0] = torch.where(low, -14.0 - 14.0 * torch.rand(c.kv, generator=g), torch.rand(c.kv, generator=g)).half()
            c.v[:] = torch.where(low.unsqueeze(1), 60000.0, 0.5).half() * (1 + torch.rand((c.kv, 128), generator=g)).half().clamp(max=1.0)
            got, (want, spread) = c.run(backend, 1.0), formula(c)
            one = 2.0 ** -11 if new > 1 else 2.0 ** -18
            tol = 2.0 ** -11 * np.abs(want) + spread * (one + 2 * c.kv * 2.0 ** -24 + 2.0 ** -20) + 2.0 ** -25
            tol += 60000 * 2.0 ** -31 * (1.0 if new > 1 else 2.0 ** -8)  # (a few large weights among each block's, and what 2^-31 of them is)
            assert (np.abs(got - want) <= tol).all(), (np.abs(got - want) / tol).max()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("steps", [(0, -200, -190, -178, -160, -300, -15, -280), (-3000, -2900, 0, -2900, -2950, -60, -80, -2000),
                                   (0, -3e6, -2e6, -70, -3e6, -90, -3e6, -10), (-3e6, -2.5e6, -3e6, 5, -3e6, -60, -2e6, 0)])
def test_references_that_fall_and_rise(backend, dtype, steps):
    """Blocks of one score each (powers of two), far below the largest and rising again, in the order one wave takes them: whole tiles and
    pieces, few rows and many. The sums stay finite and hold the largest blocks."""
    t = TORCH[dtype]
    for heads, new, reqs in ((4, 1, 500), (4, 1, 1), (4, 60, 300), (4, 60, 1)):
        print(dtype, steps, heads, new, reqs, flush=True)
        c = Case(dtype, heads, 64, new, 128 * len(steps) + 70, reqs=reqs)
        far = max(abs(x) for x in steps) > 6e4
        c.q[:, :, 0] = 1024.0 if far else 1.0
        score = torch.tensor(steps, dtype=torch.float64).repeat_interleave(128).repeat(2)[:c.kv]
        c.k[:, 0] = (score / c.q[0, 0, 0].double()).to(t)
        c.v[:] = torch.randn((c.kv, 64), generator=torch.Generator().manual_seed(3)).to(t)
        got, want = c.run(backend, math.log(2.0)), c.want(math.log(2.0))
        # equal weights within a block: 2^-9 (a weight, the output), fp32 sums, 2^-4 of a far score's unit between blocks more than 5 apart
        tol = 2.0 ** -8 * np.abs(c.v.double().numpy()).max()
        assert np.isfinite(got).all() and (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("new,max_new", [([1, 199], 100), ([20, 60, 40], 40), ([1] + [0] * 29 + [119], 4000)])
def test_a_wrong_hint_keeps_a_short_requests_weights(backend, dtype, new, max_new):
    """Weights midway between two 16-bit numbers, all rounded the same way: with two terms the output is the rounded formula's, with one it is
    off by more. A request of up to 96 rows gets two, also where max_new says that all requests are longer ones."""
    from test_gpu_attention import Batch
    b = Batch(dtype, 4, 1, 128, 16, new, [2000] + [max(n, 1) for n in new[1:]], seed=41, poison=False)
    b.q[:], b.k[:], b.v[:] = 0, 0, 1
    b.q[:, :, 0] = 1.0
    s = -0.99609375 if dtype == "bf16" else -0.99951171875  # 2^s is 0.00136 above 0.5 (bf16 steps 0.0039), 0.000169 (f16 0.00049)
    for j in range(2000):
        b.k[b.table[0, j // 16], 0, j % 16, 0] = s
    b.k[b.table[0, 3], 0, 5, 0] = 0.0
    b.v[b.table[0, 3], 0, 5] = 0.0  # (its weight is 1)
    got = b.run(backend, scale=math.log(2.0), max_new=max_new)[0]
    u, w = (2.0 ** -9, 2000 - new[0]) if dtype == "bf16" else (2.0 ** -12, 2000 - new[0])
    want = w * 2.0 ** s / (1 + w * 2.0 ** s)
    print(dtype, new, got[0, 0], want, flush=True)
    assert (np.abs(got - want) <= u * want + 2.0 ** -15).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,dim,new,kv,prefix,reqs", [
    (4, 128, 1, 300, 0, 1), (8, 64, 3, 5000, 0, 1), (4, 256, 1, 900, 0, 300), (4, 72, 20, 2000, 0, 3), (4, 128, 60, 200, 0, 1), (4, 128, 200, 1500, 0, 1),
    (4, 128, 30, 9000, 0, 1), (2, 256, 100, 700, 0, 1), (4, 128, 1, 1100, 1000, 1), (4, 128, 2, 1100, 1000, 40), (4, 64, 40, 640, 600, 2)])
def test_values_that_are_not_finite_and_seen(backend, dtype, heads, dim, new, kv, prefix, reqs):
    """A visible value that is not finite makes its element NaN, that one alone, in every row that sees it and in no other: in blocks that all
    rows see and in others, in pieces, behind a prefix, with weights that are far below a 16-bit number."""
    t, inf = TORCH[dtype], float("inf")
    c = Case(dtype, heads, dim, new, kv, prefix=prefix, reqs=reqs)
    g = torch.Generator().manual_seed(kv)
    c.q[:], c.k[:], c.v[:] = (torch.randn(x.shape, generator=g).to(t) for x in (c.q, c.k, c.v))
    spots = [(3, 0, inf), (kv // 2, 1, -inf), (5, 2, float("nan")), (0, 3, inf), (kv - new - 1, 3, -inf), (kv // 3, dim - 1, -inf), (kv - 1, 5, inf),
             (kv - new, 6, -inf), (kv - 1 - new // 2, 7, float("nan"))]
    for low in (False, True):
        print(dtype, heads, dim, new, kv, prefix, reqs, low, flush=True)
        if low:  # the weights of those keys that all rows see are 2^-60 of the others' and less
            c.q[:, :, 4], c.k[:, 4] = 8.0, 0.0
            for j, _, _ in spots:
                c.k[j, 4] = -64.0 if j < kv - new else 0.0
        scale = 0.25 if low else dim ** -0.5
        clean, v = c.run(backend, scale), c.v.clone()
        odd = np.zeros(clean.shape, bool)
        for j, d, x in spots:
            c.v[j, d] = x
            odd[[i for i in range(new) if j <= kv - new + i], :, d] = True
        got = c.run(backend, scale)
        c.v = v
        assert np.isfinite(clean).all() and np.array_equal(np.isnan(got), odd) and np.isfinite(got[~odd]).all()
        assert np.abs(got[~odd] - clean[~odd]).max() <= 2.0 ** -7 * np.abs(clean).max()


def test_values_that_are_not_finite_in_a_window(backend):
    """As above where a window and first tokens decide who sees them."""
    inf = float("inf")
    for dtype, heads, dim, new, kv in (("bf16", 4, 128, 1, 700), ("f16", 4, 128, 60, 700), ("bf16", 2, 256, 80, 900), ("f16", 4, 64, 20, 500)):
        print(dtype, dim, new, kv, flush=True)
        c = Case(dtype, heads, dim, new, kv)
        g = torch.Generator().manual_seed(kv)
        c.q[:], c.k[:], c.v[:] = (torch.randn(x.shape, generator=g).to(c.k.dtype) for x in (c.q, c.k, c.v))
        window, sinks = 100, 5
        clean = c.run(backend, dim ** -0.5, window=window, sinks=sinks)
        odd = np.zeros(clean.shape, bool)
        for j, d, x in ((2, 0, inf), (5, 1, inf), (kv - new - 70, 2, -inf), (kv - new - 99, 3, inf), (kv - new - 100, 4, inf), (4, 2, -inf), (kv - new, 6, inf)):
            c.v[j, d] = x
            odd[[i for i in range(new) if j <= kv - new + i and (kv - new + i - window < j or j < sinks)], :, d] = True
        got = c.run(backend, dim ** -0.5, window=window, sinks=sinks)
        assert np.array_equal(np.isnan(got), odd) and np.isfinite(got[~odd]).all()
        assert np.abs(got[~odd] - clean[~odd]).max() <= 2.0 ** -7 * np.abs(clean).max()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_values_that_are_not_finite_in_mixed_batches(backend, dtype, dim):
    """Prompts beside tokens, whose kernels share a launch: each row has its own request's, of its own kv head."""
    from test_gpu_attention import Batch
    for new, kv in (([1, 200, 1, 40], [300, 260, 5000, 700]), ([200, 1], [200, 37]), ([150, 0, 12], [9000, 3, 12])):
        print(dtype, dim, new, kv, flush=True)
        b = Batch(dtype, 8, 2, dim, 16, new, kv, seed=44)
        clean = b.run(backend)
        odd = np.zeros(clean.shape, bool)
        for i, n in enumerate(kv):
            for j, d, x in ((0, 8 * i + 1, float("inf")), (n // 2, 8 * i + 2, float("-inf")), (n - 1, 8 * i + 3, float("inf")), (n // 3, 8 * i + 4, float("nan"))):
                b.v[b.table[i, j // 16], 1, j % 16, d] = x
                odd[[b.start[i] + t for t in range(new[i]) if j <= n - new[i] + t], 4:, d] = True
        got = b.run(backend)
        assert np.array_equal(np.isnan(got), odd) and np.isfinite(got[~odd]).all()
        assert np.abs(got[~odd] - clean[~odd]).max() <= 2.0 ** -7 * np.abs(clean[~odd]).max()
