"""What the windowed attention and the 4-bit cache's entry points refuse, without a
GPU: the C entries before any launch, the Python wrappers before the library."""

import pytest
import torch

from qmoe import _lib, ops

NONE = None
ERR = _lib.QMOE_ERR_INVALID
A = 1 << 20
NAN, INF = float("nan"), float("inf")


def window(l, q=A, k=2 * A, v=3 * A, ctx=4, B=2, S=1, Hq=32, Hkv=4, D=128, S_max=64, max_ctx=64, window=16, sink=4,
           scale=0.1, ws=5 * A, n=A, out=6 * A):
    return l.qmoe_attn_window(q, k, v, ctx, B, S, Hq, Hkv, D, S_max, max_ctx, window, sink, scale, ws, n, out, NONE)


def kv4(l, q=A, k=2 * A, ks=7 * A, v=3 * A, vs=8 * A, ctx=4, B=2, S=1, Hq=32, Hkv=4, D=128, S_max=64, max_ctx=64,
        window=0, sink=0, scale=0.1, ws=5 * A, n=A, out=6 * A):
    return l.qmoe_attn_kv4(q, k, ks, v, vs, ctx, B, S, Hq, Hkv, D, S_max, max_ctx, window, sink, scale, ws, n, out, NONE)


def store(l, k=A, v=2 * A, S_src=16, n=16, starts=NONE, lengths=NONE, B=2, Hkv=4, D=128, S_max=64, k4=3 * A, ks=4,
          v4=5 * A, vs=8):
    return l.qmoe_kv4_store(k, v, S_src, n, starts, lengths, B, Hkv, D, S_max, k4, ks, v4, vs, NONE)


def load(l, k4=A, ks=2, v4=3 * A, vs=4, B=2, Hkv=4, D=128, S_max=64, n=64, k=5 * A, v=6 * A):
    return l.qmoe_kv4_load(k4, ks, v4, vs, B, Hkv, D, S_max, n, k, v, NONE)


def append(l, raw=4, qn=2, kn=2, cos=4, sin=4, max_pos=10, pos=4, slots=4, B=2, S=1, Hq=32, Hkv=4, D=128, S_max=64,
           eps=1e-6, q=2, k4=4, ks=1, v4=8, vs=1):
    return l.qmoe_kv4_append(raw, qn, kn, cos, sin, max_pos, pos, slots, B, S, Hq, Hkv, D, S_max, eps, q, k4, ks, v4, vs,
                             NONE)


REFUSED = [(fn, change, msg) for fn in (window, kv4) for change, msg in [
    (dict(q=NONE), "null pointer"), (dict(k=NONE), "null pointer"), (dict(v=NONE), "null pointer"),
    (dict(ctx=NONE), "null pointer"), (dict(out=NONE), "null pointer"), (dict(D=64), "head_dim"),
    (dict(Hq=30), "Hq % Hkv"), (dict(Hq=68), "Hq / Hkv <= 16"), (dict(Hkv=0), "Hq % Hkv"),
    (dict(Hq=8192, Hkv=4096), "Hkv < 4096"), (dict(B=-1), "bad B/S"), (dict(B=65536), "bad B/S"),
    (dict(S=-1), "bad B/S"), (dict(B=65000, S=3000), "below 2^27"), (dict(S_max=0), "S_max"),
    (dict(S_max=(1 << 22) + 1), "S_max"), (dict(max_ctx=65), "max_ctx"), (dict(max_ctx=-1), "max_ctx"),
    (dict(window=-1), "window"), (dict(sink=-1), "sink"), (dict(scale=0.0), "scale"), (dict(scale=NAN), "scale"),
    (dict(scale=INF), "scale"), (dict(scale=-1.0), "scale"),
    (dict(q=A + 8), "aligned"), (dict(k=2 * A + 8), "aligned"), (dict(v=3 * A + 8), "aligned"),
    (dict(ws=5 * A + 8), "aligned"), (dict(out=6 * A + 8), "aligned"),
    (dict(out=A), "overlaps"), (dict(out=A + 2 * 32 * 256 - 16), "overlaps"), (dict(out=A - 16), "overlaps")]]
REFUSED += [
    (window, dict(window=0), "window must be positive"),
    (kv4, dict(ks=NONE), "null pointer"), (kv4, dict(vs=NONE), "null pointer"), (kv4, dict(ks=7 * A + 8), "aligned"),
    (kv4, dict(vs=8 * A + 8), "aligned"),
    (store, dict(k=NONE), "null pointer"), (store, dict(v=NONE), "null pointer"), (store, dict(k4=NONE), "null"),
    (store, dict(ks=NONE), "null pointer"), (store, dict(v4=NONE), "null"), (store, dict(vs=NONE), "null pointer"),
    (store, dict(D=64), "head_dim"), (store, dict(B=-1), "bad B"), (store, dict(Hkv=0), "bad B"),
    (store, dict(S_max=0), "bad B"), (store, dict(n=-1), "entries"), (store, dict(n=17), "n <= S_src"),
    (store, dict(k=A + 8), "aligned"), (store, dict(v=2 * A + 2), "aligned"), (store, dict(k4=3 * A + 4), "aligned"),
    (store, dict(v4=5 * A + 1), "aligned"), (store, dict(ks=6), "4-byte"), (store, dict(vs=9), "4-byte"), (store, dict(B=60000, Hkv=60000, n=1 << 20, S_src=1 << 20), "entries"),
    (load, dict(k=NONE), "null pointer"), (load, dict(vs=NONE), "null pointer"), (load, dict(D=256), "head_dim"),
    (load, dict(n=65), "n <= S_max"), (load, dict(n=-1), "entries"), (load, dict(k=5 * A + 2), "aligned"),
    (load, dict(k4=A + 4), "aligned"),
    (append, dict(raw=NONE), "null pointer"), (append, dict(qn=NONE), "null pointer"),
    (append, dict(vs=NONE), "null pointer"), (append, dict(D=64), "head_dim"), (append, dict(Hq=6), "head counts"),
    (append, dict(max_pos=0), "max_pos"), (append, dict(B=-1), "bad B"), (append, dict(S_max=0), "bad B"),
    (append, dict(S=-1), "65536"), (append, dict(S=40000), "65536"), (append, dict(k4=6), "4-byte"),
    (append, dict(v4=6), "4-byte"),
]


@pytest.mark.parametrize("fn,change,msg", REFUSED, ids=lambda x: getattr(x, "__name__", None) or str(x)[:40])
def test_c_entries_refuse(fn, change, msg):
    assert fn(_lib.lib(), **change) == ERR
    assert msg in _lib.last_error(), _lib.last_error()


def test_empty_batches_launch_nothing():
    l = _lib.lib()
    for none in (dict(B=0), dict(S=0)):
        assert window(l, q=NONE, k=NONE, v=NONE, ctx=NONE, out=NONE, ws=NONE, n=0, **none) == 0
        assert kv4(l, q=NONE, k=NONE, ks=NONE, v=NONE, vs=NONE, ctx=NONE, out=NONE, ws=NONE, n=0, **none) == 0
        assert append(l, raw=NONE, pos=NONE, slots=NONE, q=NONE, k4=NONE, ks=NONE, v4=NONE, vs=NONE, **none) == 0
    for none in (dict(B=0), dict(n=0)):
        assert store(l, k=NONE, v=NONE, k4=NONE, ks=NONE, v4=NONE, vs=NONE, **none) == 0
        assert load(l, k=NONE, v=NONE, k4=NONE, ks=NONE, v4=NONE, vs=NONE, **none) == 0


def test_workspace_queries():
    l = _lib.lib()
    for fn in (l.qmoe_attn_window_workspace, l.qmoe_attn_kv4_workspace):
        assert fn(0, 1, 32, 4, 128, 100, 4, 1000) == 0
        assert fn(1, 0, 32, 4, 128, 100, 4, 1000) == 0
        assert fn(8, 1, 32, 4, 128, 1 << 62, 1 << 62, 1 << 22) >= 0
        for bad in [(-1, 1, 32, 4, 128, 1, 1, 1), (1, -1, 32, 4, 128, 1, 1, 1), (1, 1, 33, 4, 128, 1, 1, 1),
                    (1, 1, 32, 4, 64, 1, 1, 1), (1, 1, 32, 4, 128, -1, 1, 1), (1, 1, 32, 4, 128, 1, -1, 1),
                    (1, 1, 32, 4, 128, 1, 1, -1), (1, 1, 32, 4, 128, 1, 1, (1 << 22) + 1)]:
            assert fn(*bad) == -1, bad
    assert l.qmoe_attn_window_workspace(1, 1, 32, 4, 128, 0, 0, 1) == -1


def test_workspace_queries_of_every_size():
    """From caches of which nothing is seen on, whatever the batch, the chunk and the window."""
    l = _lib.lib()
    for top in (0, 1, 63, 64, 65, 256, 257, 513, 1024, 1025, 2048, 5000, 1 << 22):
        for B, S in ((1, 1), (3, 5), (2, 100), (1, 700), (64, 1), (300, 1)):
            for window in (1, 512, 1 << 40):
                assert l.qmoe_attn_window_workspace(B, S, 32, 4, 128, window, 3, top) >= 0
                assert l.qmoe_attn_kv4_workspace(B, S, 32, 4, 128, window, 3, top) >= 0
            assert l.qmoe_attn_kv4_workspace(B, S, 32, 4, 128, 0, 0, top) >= 0


def _cache():
    return ops.kv4_cache(2, 4, 64, 128, "cpu")


def test_kv4_cache_shapes():
    k, ks, v, vs = _cache()
    assert k.shape == v.shape == (2, 4, 64, 64) and ks.shape == vs.shape == (2, 4, 64, 4)
    assert k.dtype == ks.dtype == torch.uint8 and not any(bool(t.any()) for t in (k, ks, v, vs))
    assert len({t.data_ptr() for t in (k, ks, v, vs)}) == 4


def test_wrappers_refuse_without_a_gpu():
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)
    i32 = torch.zeros(2, dtype=torch.int32)
    q, k = bf(2, 32, 128), bf(2, 4, 64, 128)
    with pytest.raises(ValueError, match="must be on a GPU"):
        ops.attn_window(q, k, k, i32, 2, 1, 16)
    for window in (0, -1, 1.5, "8", None, 1 << 70):
        with pytest.raises(ValueError, match="window"):
            ops.attn_window(q, k, k, i32, 2, 1, window)
    for sink in (-1, 0.5, None, torch.zeros(2)):
        with pytest.raises(ValueError, match="sink"):
            ops.attn_window(q, k, k, i32, 2, 1, 4, sink)
        with pytest.raises(ValueError, match="sink"):
            ops.attn_kv4(q, _cache(), i32, 2, 1, 4, sink)
    with pytest.raises(ValueError, match="window"):
        ops.attn_kv4(q, _cache(), i32, 2, 1, -1)
    with pytest.raises(ValueError, match="must be on a GPU"):
        ops.attn_kv4(q, _cache(), i32, 2, 1)
    for B in (-1, 2.0, "2", None, 1 << 40):
        with pytest.raises(ValueError, match="B must"):
            ops.attn_window(q, k, k, i32, B, 1, 16)
    for cache in (None, 5, k, (k, k), [k] * 5):
        with pytest.raises(ValueError, match="cache must be"):
            ops.kv4_store(k, k, cache)
        with pytest.raises(ValueError, match="cache must be"):
            ops.kv4_load(cache)
    with pytest.raises(ValueError, match="expected a tensor"):
        ops.kv4_load([1, 2, 3, 4])
    with pytest.raises(ValueError, match="must be on a GPU"):
        ops.kv4_load(_cache())
    with pytest.raises(ValueError, match="S must"):
        ops.kv4_append(q, q, q, q, q, i32, i32, 32, 4, _cache(), 1e-6, S=-1)
    with pytest.raises(ValueError, match="eps"):
        ops.kv4_append(q, q, q, q, q, i32, i32, 32, 4, _cache(), None)
