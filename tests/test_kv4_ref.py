"""The 4-bit cache's plain form holds what the header says of it (no device)."""
import numpy as np
import pytest

import kv4_ref as R


def test_values_are_exact_in_16_bits():
    rng = np.random.default_rng(1)
    x = rng.standard_normal((500, 64)) * 2.0 ** rng.integers(-30, 20, (500, 1))
    c, d = R.quantize(x)
    v = R.values(c, d)
    assert np.array_equal(v.astype(np.float16).astype(np.float64), v)
    b = v.astype(np.float32).view(np.uint32)
    assert not (b & 0xFFFF).any()  # bf16


def test_error_of_a_block():
    """Half a step inside, a quarter of a step at the largest element, a step and a quarter at the far end of the other sign."""
    x = np.random.default_rng(2).standard_normal((2000, 32))
    c, d = R.quantize(x)
    d = d.astype(np.float64)
    q = x / d
    off = np.abs(q - (c.astype(np.float64) - 8))
    assert off[np.abs(q) <= 7.5].max() <= 0.5 and off.max() <= 1.26
    assert np.array_equal(np.abs(x).argmax(1), np.abs(q).argmax(1)) and (q.min(1) >= -8.26).all() and (q.min(1) <= -7.74).all()


@pytest.mark.parametrize("dim", [32, 96, 256])
def test_pack_touches_every_bit_once(dim):
    codes = np.full((1, 1, 16, dim), 15, np.uint8)
    d = np.full((1, 1, 16, dim // 32), -1.0, np.float16)
    for value in (False, True):
        plane = R.pack(codes, d, value)
        assert (plane[..., :8 * dim] == 255).all() and (plane[..., 8 * dim:].reshape(-1, 2) == (0, 0xBC)).all()
        assert plane.shape[-1] == 9 * dim
