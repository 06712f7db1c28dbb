"""Sampling where weights fall out of 64 bits' range: the first and the last entry whose weight is not 0 (the oracle's too)."""
import numpy as np
import pytest
import torch

from test_gpu_sample import choose, sample

pytestmark = pytest.mark.gpu
STRIPE = 256


def rows(stripes, last):
    """A row whose largest entry is 0, whose outermost stripes (the last ones, or the first) hold entries at -747 alone (e^-747 is 0 in 64 bits), beside
    entries at -744 (which have weight) in other stripes."""
    x = torch.full((1, stripes * STRIPE), float("-inf"))
    at = torch.arange(stripes) * STRIPE
    x[0, (stripes // 2) * STRIPE + 17] = 0.0
    for s in range(stripes // 4, 3 * stripes // 4):
        x[0, at[s] + 5 + s % 200] = -744.0
    quarter = slice(3 * stripes // 4 * STRIPE, None) if last else slice(0, stripes // 4 * STRIPE)
    x[0, quarter] = -747.0
    return x


@pytest.mark.parametrize("stripes", [4, 40, 80, 501, 1200])
@pytest.mark.parametrize("t", [1.0, 0.25])
def test_outermost_entries_without_weight(backend, stripes, t):
    for last in (True, False):
        x = rows(stripes, last) * t
        for u in (0.0, 1e-45, 0.5, 1.0, 7.0, float("inf")):
            want, log, _ = choose(x[0].double().numpy(), t, 0, 1.0, 0.0, u)
            token, lp = sample(backend, x, [u], [t])
            assert token[0] == want, (stripes, last, u, token[0], want)
            assert abs(lp[0] - log) <= 2.0 ** -23 * abs(log) + 1e-11


@pytest.mark.parametrize("t", [0.004, 0.01])
def test_low_temperatures(backend, t):
    """Ordinary logits whose weights at this temperature reach from 1 to far below what 64 bits hold."""
    g = torch.Generator().manual_seed(2)
    for vocab in (3000, 20480, 128256):
        x = torch.randn((6, vocab), generator=g) * 1.1 - 3.3
        x[:, vocab // 2] = 0.0
        for u in (0.0, 1.0):
            token, _ = sample(backend, x, [u] * 6, [t] * 6)
            for r in range(6):
                y = x[r].double().numpy()
                y = (y - y.max()) / float(np.float32(t))
                at = token[r]
                # weights below 2^-1074 are 0; nearer to that than a rounding either is right
                some = np.nonzero(y > -745.2)[0]
                assert y[at] > -745.2 and (some[0] <= at if u == 0 else some[-1] >= at), (vocab, r, u)
                sure = np.nonzero(y > -744.5)[0]
                assert at <= sure[0] if u == 0 else at >= sure[-1], (vocab, r, u)
