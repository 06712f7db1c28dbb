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
