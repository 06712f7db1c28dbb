"""Sizes at the edges of what the attention calls take: refused, or served (trhip_attn, trhip_attn_shared)."""
import numpy as np
import pytest
import torch

import tcb_amd
from tcb_amd import TrhipError, _lib
from test_gpu_attention import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page", [16, 4096])
def test_longest_tables(backend, page):
    """max_pages * page of 2^31 - 4096 and more is refused: a length rounded up to whole blocks would not fit 32 bits. Just below it is served."""
    x = torch.zeros(16384, dtype=torch.float32, device="cuda:0")
    a = x.data_ptr()
    kv = tcb_amd.KVCache(tcb_amd.BF16, 1, page, 1, 8, a, a)
    most = (2 ** 31 - 4096) // page
    for pages in (most, most + 1, 2 ** 31 // page - 1):
        for call, more in ((backend.Attention, ()), (backend.AttentionShared, (a, 3))):
            with pytest.raises(TrhipError) as e:
                call(kv, a, 8, a + 64, 8, 1, 1, 1, a + 128, a + 192, a, pages, *more, max_new=1)
            assert e.value.code == _lib.ERR_INVALID and "2^31" in e.value.detail
    b = Batch("bf16", 4, 2, 64, page, [1], [40], seed=50)
    want, tol = b.want()
    b.most = most - 1  # one request: the table's row is as long as it is
    assert (np.abs(b.run(backend) - want) <= tol).all()
