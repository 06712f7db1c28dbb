"""Page tables and cache append (trhip_page_tables, trhip_kv_append) against plain forms."""
import ctypes

import numpy as np
import pytest
import torch

import paged_ref as R
import tcb_amd
from tcb_amd import TrhipError, _lib

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": tcb_amd.F32, "bf16": tcb_amd.BF16, "f16": tcb_amd.F16}
DEV = "cuda:0"


def run_tables(tb, page, old, add, free, table, nslots):
    n = len(old)
    ints = [torch.tensor(x, dtype=torch.int32, device=DEV) for x in (old, add, free)]
    tab = torch.from_numpy(table).to(DEV)
    outs = [torch.full((m + 1,), 12345, dtype=torch.int32, device=DEV) for m in (n + 1, n, nslots, 1)]
    torch.cuda.synchronize()
    tb.PageTables(n, page, ints[0].data_ptr(), ints[1].data_ptr(), ints[2].data_ptr(), len(free), tab.data_ptr(), table.shape[1],
                  outs[0].data_ptr(), outs[1].data_ptr(), outs[2].data_ptr(), nslots, outs[3].data_ptr())
    tb.ctx.sync()
    got = [o.cpu().numpy() for o in outs]
    assert all(g[-1] == 12345 for g in got)
    return (tab.cpu().numpy(),) + tuple(g[:-1] for g in got)


def check_tables(tb, page, old, add, nfree, most, nslots=None, seed=0):
    rng = np.random.default_rng(seed)
    have = [-(-max(o, 0) // page) for o in old]
    pool = rng.permutation(sum(have) + nfree + 5).astype(np.int32)
    table = np.full((len(old), most), -1, np.int32)
    at = 0
    for i, h in enumerate(have):
        h = min(h, most)
        table[i, :h] = pool[at:at + h]
        at += h
    free = pool[at:at + nfree]
    nslots = sum(max(a, 0) for a in add) + 3 if nslots is None else nslots
    got = run_tables(tb, page, old, add, free, table, nslots)
    want = R.page_tables(page, old, add, free, table, nslots)
    for g, w, name in zip(got, want, ("table", "q_start", "kv_len", "slots", "used")):
        assert np.array_equal(g, np.asarray(w).reshape(g.shape)), name
    return want


@pytest.mark.parametrize("page", [16, 32, 256, 4096])
def test_tables(backend, page):
    check_tables(backend, page, [0], [1], 1, 1)
    check_tables(backend, page, [0, 0, 0], [0, 0, 0], 0, 2)
    check_tables(backend, page, [page - 1, page, page + 1, 5 * page, 0, 3], [1, 1, 1, 0, 3 * page, 1], 20, 9)
    check_tables(backend, page, [7, 0, 100], [2000, 1, 5001], 700, 600)
    check_tables(backend, page, [-5, 9, -1], [4, -3, 0], 4, 3)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 255, 256, 257, 1023, 1025, 2500])
def test_tables_of_many_requests(backend, n):
    rng = np.random.default_rng(n)
    old, add = rng.integers(0, 90, n).tolist(), rng.integers(0, 60, n).tolist()
    check_tables(backend, 16, old, add, 5 * n, 12, seed=n)
    check_tables(backend, 16, old, [1] * n, n, 12, seed=n)


def test_requests_that_do_not_fit(backend):
    """The table too short, the free pages used up: refused alone; one that needs no fresh page is still served."""
    want = check_tables(backend, 16, [10, 30, 5, 16, 8], [200, 5, 100, 20, 2], 5, 8)
    assert (want[3] == -1).any() and want[2][4] == 10
    check_tables(backend, 16, [0] * 40, [20] * 40, 33, 4)
    check_tables(backend, 16, [0] * 3, [20] * 3, 0, 4)
    check_tables(backend, 16, [0] * 3, [20] * 3, 10, 1)
    check_tables(backend, 16, [5] * 600, [17] * 600, 700, 4)


def test_lengths_past_32_bits_together(backend):
    """Lengths whose sums pass 2^31 and 2^32: those requests do not fit, and what stands before them is served."""
    for huge in ([2 ** 31 - 1] * 2, [2 ** 31 - 1] * 5, [2 ** 30] * 3):
        old, add = [7, 3] + [0] * len(huge) + [9], [30, 1] + huge + [5]
        have = [1, 1] + [0] * len(huge) + [1]
        table = np.full((len(old), 6), -1, np.int32)
        table[:, 0] = np.arange(len(old))
        free = np.arange(100, 120, dtype=np.int32)
        got = run_tables(backend, 16, old, add, free, table.copy(), 60)
        want = table.copy()
        want[0, 1:3] = [100, 101]
        assert np.array_equal(got[0], want) and got[4][0] == 2
        assert got[2][:2].tolist() == [37, 4] and got[2][2:-1].tolist() == [0] * len(huge)
        assert got[1][:3].tolist() == [0, 30, 31] and (np.diff(got[1].astype(np.int64)) >= 0).all()
        slots = [p % 16 + 16 * [0, 100, 101][p // 16] for p in range(7, 37)] + [16 + 3]
        assert got[3].tolist() == slots + [-1] * (60 - len(slots))


@pytest.mark.parametrize("nslots", [0, 1, 50, 5000])
def test_slots_shorter_or_longer_than_the_step(backend, nslots):
    check_tables(backend, 16, [3, 50, 0], [40, 1, 70], 30, 10, nslots)


def test_no_requests(backend):
    got = run_tables(backend, 16, [], [], [], np.zeros((0, 4), np.int32), 6)
    assert got[1].tolist() == [0] and (got[3] == -1).all() and got[4][0] == 0


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("src", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("heads,dim,page", [(1, 8, 16), (2, 64, 16), (8, 128, 32), (3, 96, 64), (1, 256, 128)])
def test_append(backend, dtype, src, heads, dim, page):
    for tokens, pad, shift in ((1, 0, 0), (5, 8, 8), (33, 3, 1), (700, 2 * heads * dim, 0)):
        print(dtype, src, heads, dim, page, tokens, flush=True)
        pages = -(-tokens // page) + 3
        g = torch.Generator().manual_seed(tokens)
        width = heads * dim
        rows = torch.randn(shift + tokens * (2 * width + pad), generator=g) * 10.0 ** torch.randint(-6, 6, (1,), generator=g).item()
        rows[shift] = float("nan")
        rows[shift + 1] = float("inf")
        rows[shift + 2] = -70000.0
        rows[shift + 3] = 1e-6
        rows = rows.to(TORCH[src]).to(DEV)
        slots = torch.randperm(pages * page, generator=g)[:tokens].to(torch.int32)
        if tokens > 4:
            slots[2], slots[4] = -1, pages * page
        k, v = (torch.full((pages, heads, page, dim), 5.0, dtype=TORCH[dtype], device=DEV) for _ in range(2))
        kv = tcb_amd.KVCache(CODE[dtype], pages, page, heads, dim, k.data_ptr(), v.data_ptr())
        e, dslots = rows.element_size(), slots.to(DEV)
        torch.cuda.synchronize()
        backend.KVAppend(kv, tokens, rows.data_ptr() + shift * e, rows.data_ptr() + (shift + width) * e, CODE[src], 2 * width + pad, dslots.data_ptr())
        backend.ctx.sync()
        view = rows[shift:].view(tokens, 2 * width + pad).float().to(TORCH[dtype]).cpu()
        for plane, at in ((k, 0), (v, width)):
            want = torch.full((pages, heads, page, dim), 5.0, dtype=TORCH[dtype])
            for t, s in enumerate(slots.tolist()):
                if 0 <= s < pages * page:
                    want[s // page, :, s % page] = view[t, at:at + width].view(heads, dim)
            got, nan = plane.cpu(), torch.isnan(want)
            assert torch.equal(torch.isnan(got), nan)
            assert torch.equal(got.masked_fill(nan, 0).view(torch.int16), want.masked_fill(nan, 0).view(torch.int16))


def test_new_cache(backend):
    kv = backend.NewKVCache(tcb_amd.F16, 3, 16, 2, 64)
    rows = torch.randn((4, 256), device=DEV, dtype=torch.float16)
    slots = torch.tensor([47, 0, 16, 20], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    backend.KVAppend(kv, 4, rows.data_ptr(), rows.data_ptr() + 256, tcb_amd.F16, 256, slots.data_ptr())
    got = kv.v.download(np.float16, 3 * 2 * 16 * 64).reshape(3, 2, 16, 64)
    want = rows.cpu().numpy()
    for t, s in enumerate((47, 0, 16, 20)):
        assert np.array_equal(got[s // 16, :, s % 16].reshape(-1), want[t, 128:])
    kv.release()


def test_replayed_step(backend):
    """Tables and append captured together; every replay takes the step's lengths and rows."""
    L, ctx, n, page = _lib.lib(), backend.ctx, 5, 16
    old = torch.tensor([0, 15, 16, 40, 7], dtype=torch.int32, device=DEV)
    add = torch.ones(n, dtype=torch.int32, device=DEV)
    free = torch.arange(20, 40, dtype=torch.int32, device=DEV)
    table = torch.arange(n * 4, dtype=torch.int32, device=DEV).view(n, 4).contiguous()
    q_start, kv_len, slots, used = (torch.zeros(m, dtype=torch.int32, device=DEV) for m in (n + 1, n, 8, 1))
    kv = backend.NewKVCache(tcb_amd.BF16, 40, page, 1, 64)
    rows = torch.zeros((8, 128), dtype=torch.float32, device=DEV)
    torch.cuda.synchronize()
    kv.k.fill(0), kv.v.fill(0)

    def step():
        backend.PageTables(n, page, old.data_ptr(), add.data_ptr(), free.data_ptr(), 20, table.data_ptr(), 4, q_start.data_ptr(),
                           kv_len.data_ptr(), slots.data_ptr(), 8, used.data_ptr())
        backend.KVAppend(kv, 8, rows.data_ptr(), rows.data_ptr() + 256, tcb_amd.F32, 128, slots.data_ptr())

    assert L.trhip_graph_begin(ctx.h) == 0
    step()
    graph = ctypes.c_void_p()
    assert L.trhip_graph_end(ctx.h, ctypes.byref(graph)) == 0
    plane = np.zeros((40, page, 64), np.float32)
    for turn in range(5):
        rows.copy_(torch.arange(8 * 128, device=DEV).view(8, 128) % 97 + turn)
        torch.cuda.synchronize()
        before, o = table.cpu().numpy(), old.cpu().numpy()
        assert L.trhip_graph_launch(ctx.h, graph) == 0
        ctx.sync()
        want = R.page_tables(page, o, [1] * n, free.cpu().numpy(), before, 8)
        assert np.array_equal(table.cpu().numpy(), want[0]) and np.array_equal(slots.cpu().numpy(), want[3])
        assert np.array_equal(kv_len.cpu().numpy(), want[2]) and used.item() == want[4]
        for t, s in enumerate(want[3]):
            if s >= 0:
                plane[s // page, s % page] = rows[t, :64].cpu().numpy()
        bits = kv.k.download(np.uint16, 40 * page * 64).astype(np.uint32) << 16
        assert np.array_equal(bits.view(np.float32).reshape(plane.shape), plane)
        old.copy_(kv_len)
        torch.cuda.synchronize()
    assert L.trhip_graph_destroy(graph) == 0
    kv.release()


def test_refusals(backend):
    x = torch.zeros(64, dtype=torch.int32, device=DEV)
    a = [x.data_ptr() + 64 * i for i in range(4)]

    def refused(f, *args):
        with pytest.raises(TrhipError) as e:
            f(*args)
        assert e.value.code in (_lib.ERR_INVALID, _lib.ERR_UNSUPPORTED) and e.value.detail

    good = [1, 16, a[0], a[0], a[0], 1, a[1], 1, a[2], a[3], a[3] + 16, 1, a[3] + 32]
    for at, bad in ((0, -1), (0, 2 ** 31), (1, 0), (1, 24), (1, 8), (1, 8192), (2, 0), (3, 0), (4, 0), (5, -1), (6, 0), (7, -1), (8, 0), (9, 0),
                    (9, a[0]), (8, a[0]), (10, 0), (11, -1), (11, 2 ** 31), (12, 0)):
        refused(backend.PageTables, *(good[:at] + [bad] + good[at + 1:]))

    def kv(**c):
        f = dict(dtype=tcb_amd.BF16, pages=1, page=16, heads=1, dim=8, k=a[0], v=a[0])
        f.update(c)
        return tcb_amd.KVCache(**f)

    good = [kv(), 1, a[0], a[0], tcb_amd.F32, 8, a[0]]
    for at, bad in ((0, kv(dtype=tcb_amd.F32)), (0, kv(page=20)), (0, kv(dim=12)), (0, kv(k=0)), (0, kv(v=a[0] + 2)), (1, -1), (2, 0), (3, 0),
                    (4, 7), (5, 7), (6, 0), (2, a[0] + 2), (3, a[0] + 1)):
        refused(backend.KVAppend, *(good[:at] + [bad] + good[at + 1:]))
    backend.KVAppend(kv(), 0, 0, 0, tcb_amd.F32, 8, 0)
