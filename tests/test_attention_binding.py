"""What QuantBackend's attention calls hand to the library (no device: the library is replaced by a recorder)."""
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


def backend(monkeypatch):
    tb, seen = tcb_amd.QuantBackend.__new__(tcb_amd.QuantBackend), Recorder()
    tb.ctx = Ctx()
    monkeypatch.setattr(_lib, "lib", lambda: seen)
    return tb, seen.calls


KV = dict(dtype=tcb_amd.BF16, pages=4, page=16, heads=2, dim=64, k=4096, v=8192)
ARGS = (16, 256, 32, 256, 700, 4, 3, 48, 64, 80, 5)


def test_no_hint_rules_out_no_kernel(monkeypatch):
    """Without max_new the call says that a request may bring all tokens (0 would send prompts to the kernel of few rows), or one
    where there are no more tokens than requests."""
    tb, calls = backend(monkeypatch)
    tb.Attention(tcb_amd.KVCache(**KV), *ARGS)
    tb.AttentionShared(tcb_amd.KVCache(**KV), *ARGS, 96, 40)
    names = [n for n, _, a in _lib.SIGNATURES if n.startswith("trhip_attn")]
    assert sorted(calls) == sorted(names) == ["trhip_attn", "trhip_attn_shared"]
    assert calls["trhip_attn"][13] == 700 and calls["trhip_attn_shared"][15] == 700
    few = ARGS[:4] + (3,) + ARGS[5:]
    tb.Attention(tcb_amd.KVCache(**KV), *few)
    tb.AttentionShared(tcb_amd.KVCache(**KV), *few, 96, 40)
    assert calls["trhip_attn"][13] == 1 and calls["trhip_attn_shared"][15] == 1


def test_a_hint_is_handed_on(monkeypatch):
    tb, calls = backend(monkeypatch)
    for hint in (0, 1, 350):
        tb.Attention(tcb_amd.KVCache(**KV), *ARGS, max_new=hint, window=9, sinks=2, scale=0.5)
        tb.AttentionShared(tcb_amd.KVCache(**KV), *ARGS, 96, 40, max_new=hint)
        assert calls["trhip_attn"][13:] == (hint, 9, 2, 0.5) and calls["trhip_attn_shared"][15:] == (hint, 64 ** -0.5)
