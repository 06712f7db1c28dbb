"""Rotary positions (trhip_rope) against the formula in 64 bits and more."""
import ctypes

import numpy as np
import pytest
import torch

import tcb_amd
from tcb_amd import TrhipError, _lib

pytestmark = pytest.mark.gpu
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODE = {"f32": tcb_amd.F32, "bf16": tcb_amd.BF16, "f16": tcb_amd.F16}
HALF = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}  # half a step, relative
LEAST = {"f32": 2.0 ** -150, "bf16": 2.0 ** -134, "f16": 2.0 ** -25}
DEV = "cuda:0"


def pair_axes(pairs, dealt):
    """(axis, place in the axis) of every pair, dealt out as one would by hand."""
    if not dealt:
        return [(a, j) for a, n in enumerate(pairs) for j in range(n)]
    out = []
    for j in range(max(pairs)):
        out += [(a, j) for a, n in enumerate(pairs) if j < n]
    return out


def turned(x, pos, pairs, base, neighbours, dealt, ladders, factors):
    """float64 rows [tokens, heads, dim] and how far fp32 arithmetic may be off (before the output's rounding)."""
    out, tol, total = x.copy(), np.zeros_like(x), sum(pairs)
    for i, (a, j) in enumerate(pair_axes(pairs, dealt)):
        s = np.longdouble(j) / pairs[a] if ladders else np.longdouble(i) / total
        f = np.longdouble(base) ** -s * (np.longdouble(1) if factors is None else np.longdouble(float(factors[i])))
        angle = pos[a].astype(np.longdouble) * f
        c, q = np.cos(angle).astype(np.float64)[:, None], np.sin(angle).astype(np.float64)[:, None]
        e, g = (2 * i, 2 * i + 1) if neighbours else (i, total + i)
        out[..., e], out[..., g] = x[..., e] * c - x[..., g] * q, x[..., e] * q + x[..., g] * c
        # the angle in 64 bits (four roundings of it), then within an eighth of a turn in fp32 (two roundings of up to pi / 4), its
        # series (2^-28, and two roundings of up to 1), and the products and their sum (three)
        off = 4 * 2.0 ** -53 * np.abs(angle).astype(np.float64)[:, None] + 2.0 ** -24 * 1.6 + 2.0 ** -28 + 2 * 2.0 ** -24 + 3 * 2.0 ** -24
        tol[..., e] = tol[..., g] = off * (np.abs(x[..., e]) + np.abs(x[..., g]))
    return out, tol


def check(tb, dtype, tokens, heads, dim, pairs, base=10000.0, neighbours=False, dealt=False, ladders=False, factors=None, far=5000, in_place=False,
          pad=0, shift=0, out_pad=0, out_shift=0, pos_pad=0, rows=None, pos=None, seed=0):
    g = torch.Generator().manual_seed(seed + dim + tokens)
    width = heads * dim
    x = (torch.randn((tokens, heads, dim), generator=g) if rows is None else rows).to(TORCH[dtype])
    pos = torch.randint(-far, far + 1, (len(pairs), tokens), generator=g, dtype=torch.int32) if pos is None else pos
    src = torch.full((shift + tokens * (width + pad) + 8,), 3.0, dtype=TORCH[dtype], device=DEV)
    src[shift:shift + tokens * (width + pad)].view(tokens, width + pad)[:, :width] = x.view(tokens, width).to(DEV)
    if in_place:
        out, out_pad, out_shift = src, pad, shift
    else:
        out = torch.full((out_shift + tokens * (width + out_pad) + 8,), 3.0, dtype=TORCH[dtype], device=DEV)
    where = torch.zeros((len(pairs), tokens + pos_pad), dtype=torch.int32, device=DEV)
    where[:, :tokens] = pos.to(DEV)
    fac = None if factors is None else torch.tensor(factors, dtype=torch.float32, device=DEV)
    spec = tcb_amd.RopeSpec(pairs, base, neighbours, dealt, ladders, None if fac is None else fac.data_ptr())
    e = src.element_size()
    torch.cuda.synchronize()
    tb.Rope(spec, src.data_ptr() + e * shift, width + pad, out.data_ptr() + e * out_shift, width + out_pad, CODE[dtype], tokens, heads, dim,
            where.data_ptr(), tokens + pos_pad)
    tb.ctx.sync()
    got = out.cpu()
    body = got[out_shift:out_shift + tokens * (width + out_pad)].view(tokens, width + out_pad)
    assert (got[:out_shift] == 3).all() and (got[out_shift + body.numel():] == 3).all() and (body[:, width:] == 3).all()
    got = body[:, :width].double().numpy().reshape(tokens, heads, dim)
    want, tol = turned(x.double().numpy(), pos.numpy(), pairs, base, neighbours, dealt, ladders, None if fac is None else fac.cpu().numpy())
    tol = tol + HALF[dtype] * (np.abs(want) + tol) + LEAST[dtype]
    bad = np.abs(got - want) - tol
    worst = np.unravel_index(np.argmax(bad), bad.shape)
    assert bad.max() <= 0, "at %s: got %r want %r, allowed %r" % (worst, got[worst], want[worst], tol[worst])
    rest = got[..., 2 * sum(pairs):]
    assert np.array_equal(rest, x.double().numpy()[..., 2 * sum(pairs):])


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("neighbours", [False, True])
def test_one_axis(backend, dtype, neighbours):
    for dim, n in [(2, 1), (4, 1), (64, 32), (96, 48), (128, 64), (128, 16), (128, 37), (80, 40), (200, 99), (256, 128), (512, 256), (1024, 5), (34, 17)]:
        for tokens, heads in [(1, 1), (3, 5), (17, 40), (130, 2)]:
            print(dtype, neighbours, dim, n, tokens, heads, flush=True)
            check(backend, dtype, tokens, heads, dim, [n], neighbours=neighbours)


@pytest.mark.parametrize("dealt", [False, True])
@pytest.mark.parametrize("ladders", [False, True])
@pytest.mark.parametrize("neighbours", [False, True])
def test_axes(backend, neighbours, ladders, dealt):
    for dim, pairs in [(128, [16, 24, 24]), (128, [24, 20, 20]), (64, [16, 16]), (96, [10, 7, 20, 11]), (128, [0, 5, 0, 6]), (72, [12, 12, 12]), (64, [1, 0])]:
        for dtype in ("f32", "bf16"):
            check(backend, dtype, 50, 3, dim, pairs, 1e6, neighbours, dealt, ladders)
            check(backend, dtype, 9, 2, dim, pairs, 500.0, neighbours, dealt, ladders, factors=np.linspace(1.5, -0.125, sum(pairs)))


def test_far_positions(backend):
    """Positions of any size: the angle of one step is as good at 2^31 as at 0."""
    pos = torch.tensor([[0, 1, -1, 2 ** 20, 2 ** 24 + 1, -(2 ** 30) - 1, 2 ** 31 - 1, -(2 ** 31)]], dtype=torch.int32)
    for base in (10000.0, 1e7, 1.0, 0.5, 1e-3):
        check(backend, "f32", 8, 3, 128, [64], base, pos=pos)


def test_octants(backend):
    """A quarter of a turn in 64 steps, several times round, both ways."""
    pos = torch.arange(-700, 701, dtype=torch.int32).view(1, -1)
    check(backend, "f32", pos.shape[1], 1, 2, [1], factors=[np.float32(np.pi / 128)], pos=pos)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
def test_rows_of_a_merged_product(backend, dtype):
    """In place and not, strides and starts of every alignment."""
    for pad, shift, out_pad, out_shift in [(0, 0, 0, 0), (512, 0, 0, 0), (8, 8, 0, 4), (3, 0, 5, 0), (0, 1, 0, 0), (0, 0, 1, 3), (4, 2, 2, 6)]:
        for dim, pairs in [(128, [64]), (128, [20]), (96, [16, 8, 8]), (34, [17])]:
            for neighbours in (False, True):
                check(backend, dtype, 33, 5, dim, pairs, neighbours=neighbours, pad=pad, shift=shift, out_pad=out_pad, out_shift=out_shift, pos_pad=7)
                check(backend, dtype, 33, 5, dim, pairs, neighbours=neighbours, pad=pad, shift=shift, in_place=True)


def test_many_tokens(backend):
    check(backend, "bf16", 3001, 40, 128, [24, 20, 20], 1e6, dealt=True, far=20000)
    check(backend, "f32", 2500, 9, 64, [32], far=100000, in_place=True, pad=128)


def test_more_tokens_than_a_launch_has(backend):
    """Small rows of more than 2^26 tokens, in place and to other rows."""
    n = (1 << 26) + 5
    pos = (torch.arange(n, dtype=torch.int32, device=DEV) * 7919) % 100003
    x = torch.ones((n, 2), dtype=torch.float16, device=DEV)
    x[:, 1] = 0.5
    out = torch.zeros((n, 4), dtype=torch.float16, device=DEV)
    torch.cuda.synchronize()
    spec = tcb_amd.RopeSpec((1,))
    backend.Rope(spec, x.data_ptr(), 2, out.data_ptr(), 4, tcb_amd.F16, n, 1, 2, pos.data_ptr(), n)
    backend.Rope(spec, x.data_ptr(), 2, x.data_ptr(), 2, tcb_amd.F16, n, 1, 2, pos.data_ptr(), n)
    backend.ctx.sync()
    assert torch.equal(out[:, :2], x) and not out[:, 2:].any()
    for a in range(0, n, 1 << 23):
        t = pos[a:a + (1 << 23)].double()
        c, s = torch.cos(t), torch.sin(t)
        want = torch.stack([c - 0.5 * s, s + 0.5 * c], 1)
        # half a step of f16 (of values up to 1.2), and the arithmetic's 2^-20
        assert ((x[a:a + (1 << 23)].double() - want).abs() <= 2.0 ** -11 * want.abs() + 2.0 ** -20).all(), a


def test_values_that_are_not_finite(backend):
    """A NaN or an infinity stays in its pair; elements behind the pairs keep their bits."""
    for dtype in ("f32", "bf16", "f16"):
        x = torch.randn((4, 2, 96)).to(TORCH[dtype])
        x[1, 0, 3], x[2, 1, 70], x[3, 0, 95] = float("nan"), float("inf"), float("nan")
        src, out = x.to(DEV), torch.empty_like(x, device=DEV)
        pos = torch.tensor([[1, 2, 3, 4]], dtype=torch.int32, device=DEV)
        torch.cuda.synchronize()
        backend.Rope(tcb_amd.RopeSpec([40]), src.data_ptr(), 192, out.data_ptr(), 192, CODE[dtype], 4, 2, 96, pos.data_ptr(), 4)
        backend.ctx.sync()
        bad = ~torch.isfinite(out.cpu().float())
        want = torch.zeros_like(bad)
        want[1, 0, 3] = want[1, 0, 43] = want[2, 1, 70] = want[2, 1, 30] = want[3, 0, 95] = True
        assert torch.equal(bad, want)
        bits = torch.int32 if dtype == "f32" else torch.int16
        assert torch.equal(out.cpu()[..., 80:].contiguous().view(bits), x[..., 80:].contiguous().view(bits))


def test_captured(backend):
    """A replayed graph follows rows, positions and factors."""
    x, out = torch.zeros((6, 256), device=DEV), torch.zeros((6, 256), device=DEV)
    pos, fac = torch.zeros((2, 6), dtype=torch.int32, device=DEV), torch.ones(64, device=DEV)
    spec = tcb_amd.RopeSpec([40, 24], 1e5, factors=fac.data_ptr())
    lib, g = _lib.lib(), ctypes.c_void_p()
    assert lib.trhip_graph_begin(backend.ctx.h) == 0
    backend.Rope(spec, x.data_ptr(), 256, out.data_ptr(), 256, tcb_amd.F32, 6, 2, 128, pos.data_ptr(), 6)
    assert lib.trhip_graph_end(backend.ctx.h, ctypes.byref(g)) == 0
    del spec
    for i in range(3):
        x.copy_(torch.randn((6, 256))), pos.copy_(torch.randint(0, 1000, (2, 6))), fac.fill_(1.0 + i)
        torch.cuda.synchronize()
        assert lib.trhip_graph_launch(backend.ctx.h, g) == 0
        backend.ctx.sync()
        want, tol = turned(x.cpu().double().numpy().reshape(6, 2, 128), pos.cpu().numpy(), [40, 24], 1e5, False, False, False, fac.cpu().numpy())
        assert (np.abs(out.cpu().double().numpy().reshape(6, 2, 128) - want) <= tol + HALF["f32"] * (np.abs(want) + tol) + 1e-45).all()
    assert lib.trhip_graph_destroy(g) == 0


def test_refusals(backend):
    x, pos = torch.zeros(4096, device=DEV), torch.zeros(64, dtype=torch.int32, device=DEV)
    p = x.data_ptr()
    good = dict(x=p, x_stride=256, out=p + 8192, out_stride=256, xtype=tcb_amd.F32, tokens=2, heads=2, dim=128, pos=pos.data_ptr(), pos_stride=2)

    def refused(code=_lib.ERR_INVALID, spec=None, **change):
        with pytest.raises(TrhipError) as e:
            backend.Rope(tcb_amd.RopeSpec([64]) if spec is None else spec, **{**good, **change})
        assert e.value.code == code
    for pairs in ([0], [65], [40, 25], [-1, 5], [300]):
        refused(spec=tcb_amd.RopeSpec(pairs))
    for base in (0.0, -1.0, float("inf"), float("nan")):
        refused(spec=tcb_amd.RopeSpec([64], base))
    bad = tcb_amd.RopeSpec([64])
    for axes in (0, 5, -1):
        bad.c.axes = axes
        refused(spec=bad)
    bad.c.axes, bad.c.flags = 1, 8
    refused(spec=bad)
    refused(spec=tcb_amd.RopeSpec([64], factors=p + 2))
    refused(spec=tcb_amd.RopeSpec([32, 32]), pos_stride=1)
    for dim in (0, 127, 1026, -2):
        refused(_lib.ERR_UNSUPPORTED, dim=dim)
    refused(tokens=-1)
    refused(tokens=1 << 31)
    refused(heads=0)
    refused(xtype=7)
    refused(x_stride=255)
    refused(out_stride=255)
    refused(x=0)
    refused(out=0)
    refused(pos=0)
    refused(x=p + 2)
    refused(out=p + 1, xtype=tcb_amd.F16)
    refused(out=p, out_stride=512)
    with pytest.raises(ValueError):
        tcb_amd.RopeSpec([])
    with pytest.raises(ValueError):
        tcb_amd.RopeSpec([1] * 5)
    backend.Rope(tcb_amd.RopeSpec([64]), 0, 256, 0, 256, tcb_amd.F32, 0, 2, 128, 0, 0)
