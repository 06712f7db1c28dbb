"""Rotary positions at the ends of what a call may have."""
import numpy as np
import pytest
import torch

import tcb_amd
from test_gpu_rope import check

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_more_tokens_than_a_launch_has_one_by_one(backend):
    """Rows whose items fill a workgroup, so that each token has one: past 2^23 tokens, in place, not aligned to 16 bytes."""
    n, heads, dim = (1 << 23) + 5, 9, 64
    width = heads * dim
    buf = torch.empty(1 + n * width, dtype=torch.float16, device=DEV)
    g = torch.Generator(device=DEV).manual_seed(1)
    some = torch.randn((4099, width), generator=g, device=DEV).half()
    rows = buf[1:].view(n, width)
    for a in range(0, n, 4099):
        rows[a:a + 4099] = some[:min(4099, n - a)]
    pos = (torch.arange(n, dtype=torch.int32, device=DEV) * 7919) % 100003
    torch.cuda.synchronize()
    backend.Rope(tcb_amd.RopeSpec((32,)), rows.data_ptr(), width, rows.data_ptr(), width, tcb_amd.F16, n, heads, dim, pos.data_ptr(), n)
    backend.ctx.sync()
    f = torch.tensor([10000.0 ** (-i / 32) for i in range(32)], dtype=torch.float64, device=DEV)
    for a in list(range(0, n, 4099 * 64)) + [(1 << 23) // 4099 * 4099]:  # (the last of these has the border in it)
        m = min(4099, n - a)
        x, t = some[:m].double().view(m, heads, dim), pos[a:a + m].double()[:, None, None] * f
        c, s = torch.cos(t), torch.sin(t)
        want = torch.cat([x[..., :32] * c - x[..., 32:] * s, x[..., :32] * s + x[..., 32:] * c], -1)
        # half a step of f16, and the arithmetic's 2^-20 of values of up to 10
        got = rows[a:a + m].double().view(m, heads, dim)
        assert ((got - want).abs() <= 2.0 ** -11 * want.abs() + 10 * 2.0 ** -20 + 2.0 ** -25).all(), a


@pytest.mark.parametrize("base", [1e301, np.finfo(np.float64).max])
def test_the_largest_bases(backend, base):
    """Any finite base is one."""
    check(backend, "f32", 33, 2, 64, [32], float(base), pos=torch.arange(33, dtype=torch.int32).view(1, -1) * 977)
