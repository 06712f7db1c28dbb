"""What QuantBackend's calls for positions, the 4-bit cache and sampling hand to the library (no device: the library is replaced by a
recorder)."""
import ctypes

import pytest

import tcb_amd
from tcb_amd import _lib


class Recorder:
    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return _lib.OK
        return call


class Ctx:
    h = None


@pytest.fixture
def backend(monkeypatch):
    tb, seen = tcb_amd.QuantBackend.__new__(tcb_amd.QuantBackend), Recorder()
    tb.ctx = Ctx()
    monkeypatch.setattr(_lib, "lib", lambda: seen)
    return tb, seen.calls


def plain(args):
    """Pointers as numbers, structures by reference as they are."""
    return [a.value if isinstance(a, ctypes.c_void_p) else a for a in args]


def arguments(name):
    return {n: a for n, _, a in _lib.SIGNATURES}[name]


def test_rope(backend):
    tb, calls = backend
    spec = tcb_amd.RopeSpec((4, 6, 6), base=5e5, neighbours=True, ladders=True, factors=4096)
    tb.Rope(spec, 16, 640, 32, 512, tcb_amd.BF16, 7, 10, 64, 48, 9)
    got = calls["trhip_rope"]
    assert len(got) == len(arguments("trhip_rope")) and got[1] is spec.ref
    assert plain(got[2:]) == [16, 640, 32, 512, tcb_amd.BF16, 7, 10, 64, 48, 9]
    c = spec.c
    assert (c.axes, list(c.pairs), c.base, c.factors) == (3, [4, 6, 6, 0], 5e5, 4096)
    assert c.flags == _lib.ROPE_NEIGHBOURS | _lib.ROPE_LADDERS
    plainest = tcb_amd.RopeSpec((32,)).c
    assert (plainest.axes, plainest.flags, plainest.base, plainest.factors) == (1, 0, 10000.0, None)
    assert tcb_amd.RopeSpec((8, 8), dealt=True).c.flags == _lib.ROPE_DEALT
    for pairs in ((), (1, 1, 1, 1, 1)):
        with pytest.raises(ValueError):
            tcb_amd.RopeSpec(pairs)


def test_cache_rows(backend):
    tb, calls = backend
    kv = tcb_amd.KV4Cache(6, 32, 2, 96, 4096, 8192)
    assert (kv.c.page, kv.c.heads, kv.c.dim, kv.c.pages, kv.c.k, kv.c.v) == (32, 2, 96, 6, 4096, 8192)
    assert kv.plane_bytes(6, 32, 2, 96) == 6 * 32 * 2 * (96 // 2 + 96 // 32 * 2)
    for call, name in ((tb.KV4Append, "trhip_kv4_append"), (tb.KV4Read, "trhip_kv4_read")):
        call(kv, 5, 16, 32, tcb_amd.F32, 200, 48)
        got = calls[name]
        assert len(got) == len(arguments(name)) and got[1] is kv.ref and plain(got[2:]) == [5, 16, 32, tcb_amd.F32, 200, 48]


def test_attention(backend):
    """The same hint as over the 16-bit cache, and the type between q and its stride."""
    tb, calls = backend
    kv = tcb_amd.KV4Cache(6, 32, 2, 64, 4096, 8192)
    for tokens, hint, want in ((700, None, 700), (3, None, 1), (700, 0, 0), (700, 350, 350)):
        tb.KV4Attention(kv, 16, tcb_amd.F16, 256, 32, 512, tokens, 4, 3, 48, 64, 80, 5, max_new=hint, window=9, sinks=2)
        got = calls["trhip_kv4_attn"]
        assert len(got) == len(arguments("trhip_kv4_attn")) and got[1] is kv.ref
        assert plain(got[2:]) == [16, tcb_amd.F16, 256, 32, 512, tokens, 4, 3, 48, 64, 80, 5, want, 9, 2, 64 ** -0.5]
    tb.KV4Attention(kv, 16, tcb_amd.F16, 256, 32, 512, 3, 4, 3, 48, 64, 80, 5, scale=0.5)
    assert calls["trhip_kv4_attn"][-3:] == (0, 0, 0.5)


def test_sample(backend):
    """Settings by name, and what is left out is no array."""
    tb, calls = backend
    tb.Sample(16, tcb_amd.F32, 1024, 4, 1000, 32, 48)
    got = calls["trhip_sample"]
    assert len(got) == len(arguments("trhip_sample"))
    assert plain(got[1:]) == [16, tcb_amd.F32, 1024, 4, 1000, None, None, None, None, 32, 48, None]
    tb.Sample(16, tcb_amd.BF16, 1024, 4, 1000, 32, 48, logprob=64, min_p=80, top_k=96, temperature=112, top_p=128)
    assert plain(calls["trhip_sample"][1:]) == [16, tcb_amd.BF16, 1024, 4, 1000, 112, 96, 128, 80, 32, 48, 64]


def test_structures_match_the_header():
    """Sizes and places of the structures' fields as a C compiler lays them out."""
    import os
    import subprocess
    import tempfile
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    fields = {"trhip_rope_spec": (_lib.RopeSpec, ("axes", "pairs", "flags", "base", "factors")),
              "trhip_kv4": (_lib.KV4, ("page", "heads", "dim", "pages", "k", "v"))}
    lines = ["#include <stddef.h>", "#include <stdio.h>", '#include "trhip.h"', "int main(void) {"]
    for name, (_, names) in fields.items():
        lines += ['printf("%%zu\\n", sizeof(%s));' % name] + ['printf("%%zu\\n", offsetof(%s, %s));' % (name, f) for f in names]
    with tempfile.TemporaryDirectory() as d:
        with open(os.path.join(d, "a.c"), "w") as f:
            f.write("\n".join(lines + ["return 0; }"]))
        subprocess.run(["gcc", "-I", os.path.join(root, "include"), os.path.join(d, "a.c"), "-o", os.path.join(d, "a")], check=True)
        got = [int(x) for x in subprocess.run([os.path.join(d, "a")], check=True, capture_output=True, text=True).stdout.split()]
    want = []
    for c, names in fields.values():
        want += [ctypes.sizeof(c)] + [getattr(c, f).offset for f in names]
    assert got == want
