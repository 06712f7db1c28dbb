"""Attention over the 4-bit cache: scales that are not finite are found beside the largest finite ones."""
import numpy as np
import pytest

import paged_ref as R
from test_gpu_kv4_attention import Batch

pytestmark = pytest.mark.gpu


def sees(b, i, t, j, window, sinks):
    return R.visible(b.kv[i] - b.new[i] + t, j, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("first", [7936.0, 32768.0, 40000.0, 65504.0, -65504.0])
def test_infinite_scales_behind_the_largest(backend, dtype, first):
    """A large scale, then in a later block an infinite one: NaN in its elements where it is seen, nothing where it is hidden. The first block of
    32 keys a token sees is the fifth's wave's, and the ninth's."""
    sinks = 100
    for bad in (np.inf, -np.inf, np.nan):
        for lens, place, window in (([140], 133, 0), ([140], 139, 0), ([140], 141, 0), ([300], 257, 0), ([300], 147, 150), ([300], 160, 139), ([300], 161, 139)):
            b = Batch(dtype, 4, 1, 96, 16, [1], lens, seed=5, poison=False)
            seen = sees(b, 0, 0, place, window, sinks)
            for j in range(32):  # (first tokens, which stay visible)
                b.scales[1][b.table[0, j // 16], 0, j % 16] = np.float16(first)
            b.codes[1][b.table[0, place // 16], 0, place % 16] = 8
            b.scales[1][b.table[0, place // 16], 0, place % 16, 1] = 0
            want, tol = b.want(window, sinks)
            b.scales[1][b.table[0, place // 16], 0, place % 16, 1] = np.float16(bad)
            got = b.run(backend, window, sinks)
            nan = np.zeros(got.shape, bool)
            nan[..., 32:64] = seen
            assert np.array_equal(np.isnan(got), nan), (bad, lens, place, window)
            # (f16: such results pass its range)
            fits = ~nan & (np.abs(want) + tol < 65504 if dtype == "f16" else True)
            assert (np.abs(got - want)[fits] <= tol[fits]).all(), (bad, lens, place, window)
