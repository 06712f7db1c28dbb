"""Page tables where requests are refused or page numbers are out of range: pages taken, slots (trhip_page_tables)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def run(tb, page, old, add, free, table, nslots):
    """(table, q_start, kv_len, slots, used) of one call."""
    ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (old, add, free)]
    tab = torch.from_numpy(table).to(DEV)
    outs = [torch.full((m,), 12345, dtype=torch.int32, device=DEV) for m in (len(old) + 1, len(old), nslots, 1)]
    torch.cuda.synchronize()
    tb.PageTables(len(old), page, ints[0].data_ptr(), ints[1].data_ptr(), ints[2].data_ptr(), len(free), tab.data_ptr(), table.shape[1],
                  *(o.data_ptr() for o in outs[:3]), nslots, outs[3].data_ptr())
    tb.ctx.sync()
    return (tab.cpu().numpy(),) + tuple(o.cpu().numpy() for o in outs)


def serve(page, old, add, free, table):
    """Request after request: (table, kv_len, slots, pages taken from the free list)."""
    table, taken, gone, kv_len, slots = table.copy(), 0, 0, [], []
    for i, (o, a) in enumerate(zip(old, add)):
        have, need = -(-o // page), -(-(o + a) // page)
        grow = need - have if need <= table.shape[1] else 0
        ok = need <= table.shape[1] and (grow == 0 or gone + grow <= len(free))
        gone += grow  # what a refused request could not have counts against the requests after it
        if ok and grow:
            table[i, have:need] = free[taken:taken + grow]
            taken += grow
        kv_len.append(o + a if ok else o)
        slots += [int(table[i, p // page]) * page + p % page if ok else -1 for p in range(o, o + a)]
    return table, kv_len, slots, taken


@pytest.mark.parametrize("old,add,nfree,most", [
    ([10, 30, 5, 16, 8], [200, 5, 100, 20, 2], 5, 8),  # a table too short, then the free pages used up, then no page needed
    ([0, 3], [40, 2], 2, 8),                           # the only request that needs pages is refused
    ([0, 3, 0, 3], [40, 2, 16, 2], 2, 8),
    ([5] * 700, [17, 3] * 350, 200, 4),                # two chunks of requests
    ([16, 0] * 40, [0, 20] * 40, 33, 4),
    ([0] * 3, [20] * 3, 0, 4),
])
def test_pages_taken(backend, old, add, nfree, most):
    """used is the number of pages taken from the front of the free list: what the table's new entries hold, never more than there are."""
    print(old[:5], add[:5], nfree, most, flush=True)
    page, sizes = 16, [-(-o // 16) for o in old]
    pool = np.random.default_rng(1).permutation(sum(sizes) + nfree).astype(np.int32)
    table = np.full((len(old), most), -1, np.int32)
    at = 0
    for i, n in enumerate(sizes):
        table[i, :n] = pool[at:at + n]
        at += n
    free = pool[at:]
    want = serve(page, old, add, free, table)
    got = run(backend, page, old, add, free.tolist(), table, len(want[2]) + 2)
    assert np.array_equal(got[0], want[0]) and got[2].tolist() == want[1] and got[3].tolist() == want[2] + [-1, -1]
    assert got[1].tolist() == [0] + np.cumsum(add).tolist()
    assert got[4][0] == want[3] == (got[0] != table).sum() <= nfree
    assert set(got[0][got[0] != table].tolist()) == set(free[:got[4][0]].tolist())


@pytest.mark.parametrize("page", [16, 4096])
def test_page_numbers_out_of_range(backend, page):
    """A page number whose slots do not fit 32 bits, or a negative one, gives no slot: never another page's (from the free list, from a table)."""
    last = (2 ** 31 - 1) // page  # of the highest page whose slots fit
    numbers = [2 ** 32 // page if page > 16 else 2 ** 28, last, last + 1, -1, -2 ** 31, 2 ** 31 - 1, 3]
    for free in (True, False):
        print(page, free, flush=True)
        n = len(numbers)
        old, table = [0 if free else 1] * n, np.full((n, 2), 5, np.int32)
        if not free:
            table[:, 0] = numbers
        got = run(backend, page, old, [2] * n, numbers if free else [], table, 2 * n)
        want = []
        for x in numbers:
            first = x * page + (0 if free else 1)
            want += [first + i if 0 <= first + i < 2 ** 31 else -1 for i in range(2)]
        assert got[3].tolist() == want
        assert got[4][0] == (n if free else 0)


def test_a_refused_request_holds_up_those_that_need_pages(backend):
    """For want of pages: the requests behind it that need one are refused too. By its table's width: nobody else is."""
    table = np.full((4, 4), -1, np.int32)
    table[3, 0] = 9
    kv_len, slots = run(backend, 16, [0, 0, 0, 3], [10, 60, 5, 2], [1, 2, 3], table, 77)[2:4]
    assert kv_len.tolist() == [10, 0, 0, 5] and slots.tolist() == list(range(16, 26)) + [-1] * 65 + [9 * 16 + 3, 9 * 16 + 4]
    kv_len, slots = run(backend, 16, [0, 0, 0, 3], [10, 65, 5, 2], [1, 2, 3], table, 82)[2:4]
    assert kv_len.tolist() == [10, 0, 5, 5]
    assert slots.tolist() == list(range(16, 26)) + [-1] * 65 + list(range(32, 37)) + [9 * 16 + 3, 9 * 16 + 4]
