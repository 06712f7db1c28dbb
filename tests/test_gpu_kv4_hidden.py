"""Attention over the 4-bit cache: what a token's mask hides does not change a bit of its result, whatever scales the places have, and
scales that are not finite are found beside the largest finite ones."""
import numpy as np
import pytest

import kv4_ref as K4
import paged_ref as R
from test_gpu_kv4_attention import Batch

pytestmark = pytest.mark.gpu


def sees(b, i, t, j, window, sinks):
    return R.visible(b.kv[i] - b.new[i] + t, j, window, sinks)


def loud_run(b, backend, loud, scale, window, sinks, **how):
    """Rows with the places `loud` [(request, place)] at this scale in both planes (codes anything), and with zeros there."""
    rng = np.random.default_rng(7)
    got, kept = [], [c.copy() for c in b.codes + b.scales]
    for quiet in (True, False):
        for which in range(2):
            for i, j in loud:
                at = (b.table[i, j // b.page], slice(None), j % b.page)
                shape = b.codes[which][at].shape
                b.codes[which][at] = 8 if quiet else rng.integers(0, 16, shape)
                b.scales[which][at] = 0 if quiet else np.float16(scale) * rng.choice([-1, 1], b.scales[which][at].shape)
        got.append(b.run(backend, window, sinks, **how))
        if quiet:
            want, tol = b.want(window, sinks)
    b.codes, b.scales = kept[:2], kept[2:]
    return got[0], got[1], want, tol


def check(b, backend, loud, scale, window=0, sinks=0, **how):
    """The rows that see none of the loud places: the same bits, and right."""
    quiet, got, want, tol = loud_run(b, backend, loud, scale, window, sinks, **how)
    some = 0
    for i, n in enumerate(b.new):
        for t in range(n):
            if not any(r == i and sees(b, i, t, j, window, sinks) for r, j in loud):
                at, some = b.start[i] + t, some + 1
                assert (np.abs(quiet[at] - want[at]) <= tol[at]).all(), (i, t)
                assert np.array_equal(got[at], quiet[at]), (i, t, scale, np.abs(got[at] - quiet[at]).max())
    assert some


LOUD = [65504.0, 40000.0, 7936.0, 1.0, np.inf]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("size", [1.0, 0.01, 1e-4])
def test_places_behind_the_last_key(backend, dtype, size):
    """Lengths of every place in a page: the rest of the last page holds anything."""
    kv = list(range(1, 41)) + [63, 64, 65, 129, 143, 300, 1025]
    for dim, heads, kv_heads in ((64, 4, 2), (128, 8, 2), (256, 2, 2)):
        b = Batch(dtype, heads, kv_heads, dim, 16, [1] * len(kv), kv, seed=dim, poison=False, size=size)
        loud = [(i, j) for i, n in enumerate(kv) for j in range(n, -(-n // 16) * 16)]
        for scale in LOUD:
            print(dtype, size, dim, scale, flush=True)
            check(b, backend, loud, scale)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("window,sinks", [(21, 0), (5, 3), (100, 17)])
def test_places_before_the_window(backend, dtype, window, sinks):
    """The places between the first tokens and the window of every token."""
    kv, new = [30, 55, 128, 300, 700], [1, 1, 3, 1, 24]
    for size in (1.0, 1e-3):
        b = Batch(dtype, 8, 2, 96, 16, new, kv, seed=window, poison=False, size=size)
        loud = [(i, j) for i, n in enumerate(kv) for j in range(n) if not any(sees(b, i, t, j, window, sinks) for t in range(new[i]))]
        for scale in LOUD:
            print(dtype, size, scale, flush=True)
            check(b, backend, loud, scale, window, sinks)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_tokens_of_the_same_request(backend, dtype):
    """What the later tokens of a request see and the earlier ones do not, in the same tile of rows; with a window what the earlier ones
    see and the later ones do not."""
    for new, kv in (([4, 2], [4, 90]), ([7, 12], [40, 300]), ([24], [500])):
        for size in (1.0, 1e-3):
            b = Batch(dtype, 8, 2, 64, 16, new, kv, seed=len(new), poison=False, size=size)
            for scale in LOUD:
                print(dtype, new, size, scale, flush=True)
                check(b, backend, [(i, m - 1) for i, m in enumerate(kv)], scale)
                if min(kv) > 60:
                    check(b, backend, [(i, m - n - 9) for i, (n, m) in enumerate(zip(new, kv))], scale, 10, 0)
                    check(b, backend, [(i, m - n - 9) for i, (n, m) in enumerate(zip(new, kv))] + [(0, 1)], scale, 10, 1)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_prompts(backend, dtype):
    """More rows than the kernel of few rows takes, read as they are and with their keys opened: places behind the last key."""
    b = Batch(dtype, 8, 2, 64, 16, [70, 1, 130], [70, 21, 333], seed=3, poison=False, size=0.01)
    loud = [(i, j) for i, n in enumerate(b.kv) for j in range(n, -(-n // 16) * 16)]
    for scale in LOUD:
        for hint in (1, 130):
            for wide in (False, True):
                check(b, backend, loud, scale, max_new=hint, wide=wide)


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
