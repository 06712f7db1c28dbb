"""Sampling with u of 1 and above: the last kept entry whose weight is not 0, however the sums before it were rounded."""
import numpy as np
import pytest
import torch

from test_gpu_sample import choose, sample, zipf

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [70, 700, 5000, 50257])
def test_the_last_entry(backend, vocab):
    """Rows of many weights and, in their last entries, ones that are too small to change the sum."""
    rows = 32
    x = zipf(rows, vocab, vocab)
    x[:, vocab - vocab // 5:] = -40.0 - torch.rand((rows, vocab - (vocab - vocab // 5)), generator=torch.Generator().manual_seed(1))
    # (every entry, the largest 400 or 2000, and by a share of the largest: kept entries in the row's end among them)
    for kw in (dict(), dict(k=[vocab // 2 + 1] * rows), dict(k=[min(2000, vocab - 3)] * rows), dict(low=[1e-25] * rows), dict(k=[60] * rows),
               dict(p=[0.999999] * rows), dict(k=[vocab - 2] * rows, p=[0.9999] * rows)):
        for u in (1.0, 3.5, float("inf")):
            token, lp = sample(backend, x, [u] * rows, **kw)
            for r in range(rows):
                want, log, close = choose(x[r].double().numpy(), 1.0, kw.get("k", [0] * rows)[r], float(np.float32(kw.get("p", [1.0] * rows)[r])),
                                          float(np.float32(kw.get("low", [0.0] * rows)[r])), u)
                assert close or (token[r] == want and abs(lp[r] - log) <= 2.0 ** -23 * abs(log) + 1e-11), (vocab, kw, u, r, token[r], want)
