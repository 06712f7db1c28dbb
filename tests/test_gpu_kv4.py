"""The 4-bit paged cache (trhip_kv4_append, trhip_kv4_read) against its plain form."""
import numpy as np
import pytest
import torch

import kv4_ref as R
import tcb_amd
from tcb_amd import TrhipError, _lib

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": tcb_amd.F32, "bf16": tcb_amd.BF16, "f16": tcb_amd.F16}
DEV = "cuda:0"


def new_cache(pages, page, heads, dim, fill=0xA5):
    k, v = (torch.full((pages, heads, page // 16, 9 * dim), fill, dtype=torch.uint8, device=DEV) for _ in range(2))
    return tcb_amd.KV4Cache(pages, page, heads, dim, k.data_ptr(), v.data_ptr()), k, v


def append(tb, kv, rows, dtype, slots, stride=None, shift=0):
    """rows [2, tokens, heads, dim] (torch, on the CPU) to slots; stride, shift in elements. Returns the rows as float64."""
    n, width = rows.shape[1], kv.heads * kv.dim
    stride = width if stride is None else stride
    src = [torch.full((shift + n * stride + 8,), 3.0, dtype=TORCH[dtype], device=DEV) for _ in range(2)]
    for s, r in zip(src, rows):
        s[shift:shift + n * stride].view(n, stride)[:, :width] = r.reshape(n, width).to(TORCH[dtype]).to(DEV)
    at = torch.tensor(slots, dtype=torch.int32, device=DEV)
    e = src[0].element_size() * shift
    torch.cuda.synchronize()
    tb.KV4Append(kv, n, src[0].data_ptr() + e, src[1].data_ptr() + e, CODE[dtype], stride, at.data_ptr())
    tb.ctx.sync()
    return rows.to(TORCH[dtype]).double().numpy()


def want_planes(kv, rows, slots, fill=0xA5):
    """Both planes as append leaves them, from planes of `fill` bytes."""
    planes = []
    for which in range(2):
        codes = np.full((kv.pages, kv.heads, kv.page, kv.dim), 0, np.uint8)
        d = np.zeros((kv.pages, kv.heads, kv.page, kv.dim // 32), np.float16)
        mine = np.zeros((kv.pages, kv.page), bool)
        c, s = R.quantize(rows[which])
        for t, slot in enumerate(slots):
            if 0 <= slot < kv.pages * kv.page:
                codes[slot // kv.page, :, slot % kv.page], d[slot // kv.page, :, slot % kv.page] = c[t], s[t]
                mine[slot // kv.page, slot % kv.page] = True
        p = R.pack(codes, d, which == 1)
        full = R.pack(np.where(mine[:, None, :, None], 15, 0).astype(np.uint8) * np.ones_like(codes),
                      np.where(mine[:, None, :, None], np.frombuffer(b"\xff\xff", np.float16), np.float16(0)) * np.ones_like(d), which == 1)
        # (bits of places that were written; the scale's mask by its own bits)
        mask = full.copy()
        sm = np.zeros(d.shape, np.uint16)
        sm[np.broadcast_to(mine[:, None, :, None], d.shape)] = 0xFFFF
        mask[..., 8 * kv.dim:] = R.pack(np.zeros_like(codes), sm.view(np.float16), which == 1)[..., 8 * kv.dim:]
        planes.append(np.where(mask > 0, (p & mask) | (fill & ~mask), fill).astype(np.uint8))
    return planes


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 64, 96, 128, 160, 192, 224, 256])
def test_append(backend, dtype, dim):
    """Bytes of both planes, those of other places untouched: pages, places in any order, slots out of range, strides, misaligned rows."""
    g = torch.Generator().manual_seed(dim)
    for page, heads, tokens, pad, shift in [(16, 1, 1, 0, 0), (32, 3, 37, 0, 0), (64, 2, 50, 5, 1), (16, 8, 16, 64, 8), (128, 5, 130, 3, 3)]:
        print(dtype, dim, page, heads, tokens, flush=True)
        kv, k, v = new_cache(4, page, heads, dim)
        rows = torch.randn((2, tokens, heads, dim), generator=g) * 3
        slots = torch.randperm(4 * page, generator=g)[:tokens].tolist() if 4 * page >= tokens else list(range(4 * page)) + [-1] * (tokens - 4 * page)
        slots = slots + [] if tokens < 3 else slots[:-2] + [-1, 4 * page]
        x = append(backend, kv, rows, dtype, slots, heads * dim + pad, shift)
        for got, want in zip((k, v), want_planes(kv, x, slots)):
            assert np.array_equal(got.cpu().numpy(), want)


def test_append_whole_pieces(backend):
    """Slots in a row, from anywhere, across pages: what a prompt brings."""
    for dim, start, tokens in [(128, 0, 64), (64, 3, 61), (128, 13, 7), (256, 17, 30), (96, 15, 2), (128, 4, 4), (128, 60, 68)]:
        kv, k, v = new_cache(8, 16, 2, dim)
        rows = torch.randn((2, tokens, 2, dim), generator=torch.Generator().manual_seed(tokens))
        order = [5, 2, 7, 0, 1, 6, 3, 4]
        slots = [order[(start + t) // 16] * 16 + (start + t) % 16 for t in range(tokens)]
        for dtype in ("bf16", "f32"):
            x = append(backend, kv, rows, dtype, slots)
            for got, want in zip((k, v), want_planes(kv, x, slots)):
                assert np.array_equal(got.cpu().numpy(), want), (dim, start, tokens, dtype)


def hard_blocks():
    """Blocks [n, 32] where the rules bite: ties of size and of rounding, borders next to them, zeros, the ends of f16, what is not finite."""
    rng = np.random.default_rng(5)
    out = [np.zeros(32), -np.zeros(32), np.full(32, 1.0), np.full(32, -1.0)]
    x = rng.standard_normal(32)
    x[7], x[20] = 4.0, -4.0  # the first decides the sign
    out += [x, -x]
    for d in (1.0, 0.3125, 2.0 ** -14, 2.0 ** -20, 7936.0, -1.0, -0.3125):  # exact halves, and one step beside them
        h = np.concatenate([[-8.0], np.arange(-7.5, 7.6, 1.0), np.arange(-7, 8)]) * d
        out += [h, np.nextafter(h.astype(np.float32), np.float32(1e9)).astype(np.float64), np.nextafter(h.astype(np.float32), np.float32(-1e9)).astype(np.float64)]
        out[-1][0] = out[-2][0] = h[0]
    for m in (33.0, 33.0 * 8 / 32, 16.5 * 8, 16.25 * 8, 17.5 * 8, 31.5 * 8, 31.75 * 8):  # the scale's own ties
        out.append(np.concatenate([[m], rng.uniform(-m, m, 31)]))
    for e in range(-34, 20, 2):
        out.append(rng.standard_normal(32) * 2.0 ** e)
    out += [rng.standard_normal(32) * 1e5, rng.standard_normal(32) * 1e30, np.full(32, 63488.0), np.full(32, -65504.0), np.full(32, 1e-40)]
    for bad in (np.inf, -np.inf, np.nan):
        x = rng.standard_normal(32)
        x[rng.integers(32)] = bad
        out.append(x)
    return np.stack(out)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_hard_blocks(backend, dtype):
    b = torch.from_numpy(hard_blocks().astype(np.float32))
    n = b.shape[0]
    kv, k, v = new_cache(-(-n // 16), 16, 1, 32)
    rows = torch.stack([b, b.flip(1)]).view(2, n, 1, 32)
    slots = list(range(n))
    x = append(backend, kv, rows, dtype, slots)
    for got, want in zip((k, v), want_planes(kv, x, slots)):
        assert np.array_equal(got.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("dim", [32, 96, 128, 256])
def test_read(backend, dtype, dim):
    """What was appended comes back as the values it stands for; slots out of range leave their rows alone."""
    for page, heads, tokens, pad, shift in [(16, 1, 1, 0, 0), (32, 3, 37, 0, 0), (64, 2, 50, 5, 1), (16, 8, 33, 64, 8)]:
        kv, k, v = new_cache(4, page, heads, dim)
        rows = torch.randn((2, tokens, heads, dim), generator=torch.Generator().manual_seed(page)) * 5
        rows[0, 0, 0, 3], rows[1, tokens // 2, heads - 1, 31] = float("nan"), float("-inf")
        slots = (torch.randperm(4 * page)[:tokens]).tolist()
        x = append(backend, kv, rows, "f32", slots)
        ask = list(slots)
        if tokens > 3:
            ask[2], ask[-1] = -5, 4 * page
        width, stride = heads * dim, heads * dim + pad
        back = [torch.full((shift + tokens * stride + 8,), 7.0, dtype=TORCH[dtype], device=DEV) for _ in range(2)]
        at = torch.tensor(ask, dtype=torch.int32, device=DEV)
        e = back[0].element_size() * shift
        torch.cuda.synchronize()
        backend.KV4Read(kv, tokens, back[0].data_ptr() + e, back[1].data_ptr() + e, CODE[dtype], stride, at.data_ptr())
        backend.ctx.sync()
        for which in range(2):
            want = R.values(*R.quantize(x[which])).reshape(tokens, width)
            got = back[which].cpu()
            body = got[shift:shift + tokens * stride].view(tokens, stride)
            assert (got[:shift] == 7).all() and (got[shift + tokens * stride:] == 7).all() and (body[:, width:] == 7).all()
            for t in range(tokens):
                w = want[t] if 0 <= ask[t] < 4 * page else np.full(width, 7.0)
                assert np.array_equal(body[t, :width].double().numpy(), w, equal_nan=True), t


def test_read_of_any_scale(backend):
    """Scales that append does not write: eleven bits, infinite ones; rounded once to the type asked for."""
    rng = np.random.default_rng(3)
    codes = rng.integers(0, 16, (1, 1, 16, 32)).astype(np.uint8)
    d = np.array([0x3C01, 0x7BFF, 0xFBFF, 0x0001, 0x7C00, 0xFC00, 0x7E00, 0x3555, 0x8003, 0x1234, 0x6BCD, 0x0, 0x8000, 0x4321, 0xB00B, 0x3FFF], np.uint16)
    d = d.view(np.float16).reshape(1, 1, 16, 1)
    planes = [torch.from_numpy(R.pack(codes, d, w)).to(DEV) for w in (False, True)]
    kv = tcb_amd.KV4Cache(1, 16, 1, 32, planes[0].data_ptr(), planes[1].data_ptr())
    at = torch.arange(16, dtype=torch.int32, device=DEV)
    for dtype in TORCH:
        back = torch.empty((2, 16, 32), dtype=TORCH[dtype], device=DEV)
        torch.cuda.synchronize()
        backend.KV4Read(kv, 16, back[0].data_ptr(), back[1].data_ptr(), CODE[dtype], 32, at.data_ptr())
        backend.ctx.sync()
        with np.errstate(invalid="ignore"):
            want = np.where(np.isfinite(d), R.values(codes, d).reshape(1, 1, 16, 32), np.nan)[0, 0]
        want = torch.from_numpy(want).to(TORCH[dtype]).double().numpy()
        for b in back.cpu().double().numpy():
            assert np.array_equal(b, want, equal_nan=True)


def test_same_slot_twice(backend):
    """Two rows for one slot: a mix of both, its neighbours untouched."""
    kv, k, v = new_cache(1, 16, 1, 64)
    rows = torch.randn((2, 2, 1, 64), generator=torch.Generator().manual_seed(1))
    append(backend, kv, rows, "f32", [5, 5])
    keep = want_planes(kv, rows.double().numpy(), [5, -1])
    other = want_planes(kv, rows.double().numpy(), [-1, 5])
    for got, a, b in zip((k, v), keep, other):
        g = got.cpu().numpy()
        same = a == b
        assert np.array_equal(g[same], a[same])


def test_past_32_bits(backend):
    """Planes of over 4 GiB: the last page's places."""
    pages, page, heads, dim = 1000, 4096, 8, 256
    k, v = (torch.empty(tcb_amd.KV4Cache.plane_bytes(pages, page, heads, dim), dtype=torch.uint8, device=DEV) for _ in range(2))
    assert k.numel() > 1 << 32
    kv = tcb_amd.KV4Cache(pages, page, heads, dim, k.data_ptr(), v.data_ptr())
    last = pages * page - 16
    rows = torch.randn((2, 16, heads, dim), generator=torch.Generator().manual_seed(2))
    slots = list(range(last, last + 16))
    x = append(backend, kv, rows, "f32", slots)
    back = torch.empty((2, 16, heads * dim), dtype=torch.float32, device=DEV)
    at = torch.tensor(slots, dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    backend.KV4Read(kv, 16, back[0].data_ptr(), back[1].data_ptr(), tcb_amd.F32, heads * dim, at.data_ptr())
    backend.ctx.sync()
    for which in range(2):
        assert np.array_equal(back[which].cpu().double().numpy(), R.values(*R.quantize(x[which])).reshape(16, -1))


def test_captured(backend):
    """Append and read in a replayed graph follow their rows and slots."""
    kv, k, v = new_cache(4, 16, 2, 128)
    rows = torch.zeros((2, 5, 256), device=DEV)
    at, back = torch.zeros(5, dtype=torch.int32, device=DEV), torch.zeros((2, 5, 256), device=DEV)

    def step():
        backend.KV4Append(kv, 5, rows[0].data_ptr(), rows[1].data_ptr(), tcb_amd.F32, 256, at.data_ptr())
        backend.KV4Read(kv, 5, back[0].data_ptr(), back[1].data_ptr(), tcb_amd.F32, 256, at.data_ptr())
    import ctypes
    lib, g = _lib.lib(), ctypes.c_void_p()
    assert lib.trhip_graph_begin(backend.ctx.h) == 0
    step()
    assert lib.trhip_graph_end(backend.ctx.h, ctypes.byref(g)) == 0
    for i in range(4):
        r = torch.randn((2, 5, 2, 128), generator=torch.Generator().manual_seed(i))
        rows.copy_(r.view(2, 5, 256))
        at.copy_(torch.tensor([3 + i, 20, 21, 40 - i, 63], dtype=torch.int32))
        torch.cuda.synchronize()
        assert lib.trhip_graph_launch(backend.ctx.h, g) == 0
        backend.ctx.sync()
        for which in range(2):
            assert np.array_equal(back[which].cpu().double().numpy(), R.values(*R.quantize(r[which].double().numpy())).reshape(5, 256))
    assert lib.trhip_graph_destroy(g) == 0


def test_refusals(backend):
    k = torch.zeros(1 << 20, dtype=torch.uint8, device=DEV)
    at = torch.zeros(4, dtype=torch.int32, device=DEV)
    p = k.data_ptr()
    good = dict(pages=2, page=16, heads=2, dim=64, k=p, v=p + (1 << 19))

    def refused(code, cache={}, tokens=1, src=p, type=tcb_amd.F32, stride=128, slots=None):
        kv = tcb_amd.KV4Cache(**{**good, **cache})
        for call in (backend.KV4Append, backend.KV4Read):
            with pytest.raises(TrhipError) as e:
                call(kv, tokens, src, p, type, stride, at.data_ptr() if slots is None else slots)
            assert e.value.code == code
    for page in (0, 8, 24, 8192, -16):
        refused(_lib.ERR_INVALID, dict(page=page))
    for dim in (0, 8, 48, 288, -32):
        refused(_lib.ERR_UNSUPPORTED, dict(dim=dim))
    refused(_lib.ERR_INVALID, dict(heads=0))
    refused(_lib.ERR_INVALID, dict(pages=-1))
    refused(_lib.ERR_INVALID, dict(pages=1 << 28))
    refused(_lib.ERR_INVALID, dict(k=0))
    refused(_lib.ERR_INVALID, dict(v=p + 8))
    refused(_lib.ERR_INVALID, tokens=-1)
    refused(_lib.ERR_INVALID, tokens=1 << 31)
    refused(_lib.ERR_INVALID, type=3)
    refused(_lib.ERR_INVALID, stride=127)
    refused(_lib.ERR_INVALID, src=0)
    refused(_lib.ERR_INVALID, src=p + 2)
    refused(_lib.ERR_INVALID, src=p + 1, type=tcb_amd.F16)
    refused(_lib.ERR_INVALID, slots=0)
    kv = tcb_amd.KV4Cache(**good)
    backend.KV4Append(kv, 0, 0, 0, tcb_amd.F32, 128, 0)
    backend.KV4Read(kv, 0, 0, 0, tcb_amd.F32, 128, 0)
    own = backend.NewKV4Cache(2, 16, 2, 64)
    assert own.k.nbytes == 2 * 16 * 2 * 64 * 9 // 16
    own.release()
