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


def test_starts_out_of_order(backend):
    """Starts that fall, overlap or pass the tokens: nothing is written but out's rows of the batch, and the next call is right."""
    dev, h, d = "cuda:0", 8, 128
    good = Batch("bf16", h, 2, d, 16, [1, 90, 2], [300, 500, 40], seed=60)
    want = good.run(backend)
    for start in ([0, 60, 20, 93], [93, 0, 93, 0], [-5, 50, 2 ** 31 - 1, 7], [40, 30, 20, 10], [0, 93, 0, 93], [-2 ** 31, 2 ** 31 - 1, -1, 2 ** 31 - 1]):
        for prefix, window in ((0, 0), (0, 50), (70, 0)):
            for max_new in (1, 30, 93):
                print(start, prefix, window, max_new, flush=True)
                b = Batch("bf16", h, 2, d, 16, [1, 90, 2], [300, 500, 40], prefix=prefix, seed=61)
                b.start = np.array(start, np.int32)
                b.run(backend, window=window, max_new=max_new)  # (checks what lies around out's rows)
    assert np.array_equal(good.run(backend), want)


def test_lengths_of_any_sign(backend):
    """Negative lengths hold no keys, lengths past the table are cut to it."""
    b = Batch("f16", 4, 2, 64, 16, [1, 3, 100], [32, 32, 112], seed=62, poison=False)
    b.table[:, :] = b.table[2, :]
    b.kv = [-1, -2 ** 31, 2 ** 31 - 1]
    got = b.run(backend)
    assert (got[:4] == 0).all()
    b.kv = [0, 0, 16 * b.most]
    assert np.array_equal(got, b.run(backend))


def test_contexts_and_threads(backend):
    """Two contexts on threads of their own, each with its stream, workspace and counters: every call gives what it gives alone."""
    import threading
    batches = [Batch("bf16", 8, 2, 128, 16, [1] * 5, [9000, 300, 4000, 17, 800], seed=63), Batch("bf16", 8, 2, 128, 16, [150, 1, 3], [3000, 700, 20], seed=64),
               Batch("f16", 8, 2, 128, 16, [2] * 20, [30 + i for i in range(20)], prefix=2000, seed=65)]
    want = [b.run(backend) for b in batches]
    tbs, wrong = [tcb_amd.QuantBackend(0) for _ in range(2)], []

    def work(tb, order):
        for turn in range(6):
            for i in order:
                if not np.array_equal(batches[i].run(tb), want[i]):
                    wrong.append((order, turn, i))

    threads = [threading.Thread(target=work, args=(tb, order)) for tb, order in zip(tbs, ((0, 1, 2), (2, 0, 1)))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for tb in tbs:
        tb.close()
    assert not wrong
