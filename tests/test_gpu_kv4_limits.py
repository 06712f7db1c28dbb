"""Attention over the 4-bit cache at the ends of what a call may have."""
import numpy as np
import pytest
import torch

import kv4_ref as K4
import paged_ref as R
import tcb_amd
from tcb_amd import TrhipError, _lib
from test_gpu_kv4_attention import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_more_rows_than_a_launch_has(backend):
    """Refused before anything is launched: 2^24 tiles of rows, by tokens and by requests."""
    x, i = torch.zeros(1 << 16, dtype=torch.uint8, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    p, n = x.data_ptr(), i.data_ptr()
    for heads, kv_heads, tokens, nreq in ((1, 1, 1 << 28, 1), (32, 8, 1 << 23, 1), (8, 8, 1 << 21, 1 << 21)):
        assert (tokens * heads // kv_heads // 16 + nreq) * kv_heads >= 1 << 24  # (or it would be launched, on arrays that are not there)
        kv = tcb_amd.KV4Cache(2, 16, kv_heads, 64, p, p + (1 << 15))
        with pytest.raises(TrhipError) as e:
            backend.KV4Attention(kv, p, tcb_amd.BF16, heads * 64, p, heads * 64, tokens, heads, nreq, n, n, n, 2, max_new=1)
        assert e.value.code == _lib.ERR_INVALID and "too many rows" in str(e.value)


@pytest.mark.parametrize("e", [1e10, 5e12])
@pytest.mark.parametrize("new", [1, 5])
def test_large_scales_of_the_softmax(backend, e, new):
    """Rows of q near 1e30 over keys near 1e-6, and a scale that brings their products to 1e34 and more: within fp32, while the factor between q's
    operands and the scores is not."""
    b = Batch("bf16", 4, 1, 64, 16, [new], [30], seed=4, poison=False)
    b.codes[0], b.scales[0] = K4.quantize((torch.randn(b.codes[0].shape, generator=torch.Generator().manual_seed(2)) * 1e-6).numpy())
    b.q = (b.q.float() * 1e30).to(torch.bfloat16)
    scale = float(np.float32(e))
    k, v = b.values()
    kk, vv = (R.rows_of(c, b.table[0], 30, 16) for c in (k, v))
    got = b.run(backend, scale=scale)
    for t in range(new):
        for a in range(4):
            s = scale * (kk[:30 - new + t + 1, 0] @ b.q[t, a].double().numpy())
            order = np.argsort(-s)
            # one key has all the weight: the next score is further below than an fp32 sum may be off
            assert abs(s).max() < 3e38 and s[order[0]] - s[order[1]] > 64 * 64 * 2.0 ** -24 * abs(s).max()
            want = vv[order[0], 0]
            assert (np.abs(got[t, a] - want) <= 2.0 ** -8 * np.abs(want)).all(), (t, a)
