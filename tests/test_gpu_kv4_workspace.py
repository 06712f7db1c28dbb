"""Attention over the 4-bit cache where there is no memory to open a prompt's keys: the requests are read as they are."""
import ctypes

import numpy as np
import pytest

import tcb_amd
from tcb_amd import TrhipError, _lib
from tcb_amd._lib import KNOB_WORKSPACE
from test_gpu_kv4_attention import Batch

pytestmark = pytest.mark.gpu


def batch(dtype, heads=8, kv_heads=2, pages=4000):
    """Two long requests beside short ones, tables of so many pages that both's opened planes take over 64 MiB."""
    b = Batch(dtype, heads, kv_heads, 128, 16, [70, 1, 130, 3], [300, 40, 513, 77], seed=6)
    b.table = np.concatenate([b.table, np.full((4, pages - b.most), -7, np.int32)], 1)
    b.most = pages
    return b


@pytest.fixture
def tb():
    """A context of its own, whose workspaces are as small as its calls made them."""
    t = tcb_amd.QuantBackend(0)
    yield t
    t.close()


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_no_memory_to_open_keys(tb, dtype):
    lib, b = _lib.lib(), batch(dtype)
    want, tol = b.want()
    as_they_are = b.run(tb, max_new=1)  # (the workspace that this needs, of 37 MiB, is there from now on)
    assert lib.trhip_set_launch_shape(tb.ctx.h, KNOB_WORKSPACE, 64, 0, 0, 0) == 0
    for _ in range(3):
        got = b.run(tb)
        assert (np.abs(got - want) <= tol).all()
        assert np.array_equal(got, as_they_are)
    g, run = ctypes.c_void_p(), tb.KV4Attention

    def captured(*args, **how):
        """The call in a graph, replayed."""
        run(*args, **how)
        assert lib.trhip_graph_begin(tb.ctx.h) == 0
        run(*args, **how)
        assert lib.trhip_graph_end(tb.ctx.h, ctypes.byref(g)) == 0
        for _ in range(3):
            assert lib.trhip_graph_launch(tb.ctx.h, g) == 0
            tb.ctx.sync()
        assert lib.trhip_graph_destroy(g) == 0
    tb.KV4Attention = captured
    assert np.array_equal(b.run(tb), as_they_are)
    tb.KV4Attention = run
    assert lib.trhip_set_launch_shape(tb.ctx.h, KNOB_WORKSPACE, 0, 0, 0, 0) == 0
    opened = b.run(tb)
    assert (np.abs(opened - want) <= tol).all() and not np.array_equal(opened, as_they_are)
    # what there is already is used
    assert lib.trhip_set_launch_shape(tb.ctx.h, KNOB_WORKSPACE, 64, 0, 0, 0) == 0
    assert np.array_equal(b.run(tb), opened)


def test_no_memory_for_partial_results(tb):
    """A call that cannot do without fails, and the next one is not the worse for it."""
    lib, b = _lib.lib(), batch("bf16")
    assert lib.trhip_set_launch_shape(tb.ctx.h, KNOB_WORKSPACE, 1, 0, 0, 0) == 0
    with pytest.raises(TrhipError) as e:
        b.run(tb)
    assert e.value.code == _lib.ERR_OOM
    assert lib.trhip_set_launch_shape(tb.ctx.h, KNOB_WORKSPACE, 0, 0, 0, 0) == 0
    b.check(tb)
    for bad in ((-1, 0, 0, 0), (0, 1, 0, 0), (5, 0, 0, 1)):
        assert lib.trhip_set_launch_shape(tb.ctx.h, KNOB_WORKSPACE, *bad) == _lib.ERR_INVALID
