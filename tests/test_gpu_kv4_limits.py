"""Attention over the 4-bit cache at the ends of what a call may have."""
import pytest
import torch

import tcb_amd
from tcb_amd import TrhipError, _lib

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
