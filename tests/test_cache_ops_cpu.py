"""What the shared-prefix and bounded-cache entry points refuse, without a GPU:
the C entries before any launch, the Python wrappers before the library."""

import pytest
import torch

from qmoe import _lib, ops

NONE = None
ERR = _lib.QMOE_ERR_INVALID


def shared(l, q=1, kp=1, vp=1, P=8, P_max=8, k=1, v=1, ctx=1, B=2, S=1, Hq=32, Hkv=4, D=128, S_max=64, max_ctx=64,
           scale=0.1, ws=1, n=0, out=1):
    return l.qmoe_attn_shared(q, kp, vp, P, P_max, k, v, ctx, B, S, Hq, Hkv, D, S_max, max_ctx, scale, ws, n, out, NONE)


def prompt(l, q=1, k=1, v=1, B=2, S=4, Hq=32, Hkv=4, D=128, S_max=64, start=0, lengths=NONE, scale=0.1, ws=1, n=0,
           scores=1, out=1):
    return l.qmoe_attn_prefill_scored(q, k, v, B, S, Hq, Hkv, D, S_max, start, lengths, scale, ws, n, scores, out, NONE)


def scored(l, q=1, k=1, v=1, ctx=1, B=2, Hq=32, Hkv=4, D=128, S_max=64, max_ctx=64, scale=0.1, ws=1, n=0, scores=1,
           out=1):
    return l.qmoe_attn_decode_scored(q, k, v, ctx, B, Hq, Hkv, D, S_max, max_ctx, scale, ws, n, scores, out, NONE)


def append(l, raw=1, qn=1, kn=1, cos=1, sin=1, max_pos=10, pos=1, slots=1, B=2, Hq=32, Hkv=4, D=128, S_max=64,
           eps=1e-6, q=1, k=1, v=1, scores=NONE, sp=NONE):
    return l.qmoe_kv_append(raw, qn, kn, cos, sin, max_pos, pos, slots, B, Hq, Hkv, D, S_max, eps, q, k, v, scores, sp,
                            NONE)


def evict(l, k=1, v=2, sc=3, sp=4, ctx=5, B=2, Hkv=4, D=128, S_max=64, budget=32, recent=4, sink=2, ws=6, n=1 << 20,
          S_out=64, k2=1, v2=2, sc2=3, sp2=4):
    return l.qmoe_kv_evict(k, v, sc, sp, ctx, B, Hkv, D, S_max, budget, recent, sink, ws, n, S_out, k2, v2, sc2, sp2,
                           NONE)


NAN, INF = float("nan"), float("inf")
REFUSED = [
    (shared, dict(q=NONE), "null pointer"), (shared, dict(k=NONE), "null pointer"), (shared, dict(ctx=NONE), "null"),
    (shared, dict(out=NONE), "null pointer"), (shared, dict(kp=NONE), "null prefix"),
    (shared, dict(D=64), "head_dim"), (shared, dict(Hq=30), "Hq % Hkv"), (shared, dict(Hq=68), "Hq / Hkv <= 16"),
    (shared, dict(Hkv=0), "Hq % Hkv"), (shared, dict(B=-1), "bad B/S"), (shared, dict(S=-1), "bad B/S"),
    (shared, dict(B=65000, S=3000), "below 2^27"), (shared, dict(S_max=0), "S_max"),
    (shared, dict(S_max=(1 << 22) + 1), "S_max"), (shared, dict(P=9), "P <= P_max"), (shared, dict(P=-1), "0 <= P"),
    (shared, dict(P_max=(1 << 22) + 1), "2^22"), (shared, dict(max_ctx=65), "max_ctx"),
    (shared, dict(max_ctx=-1), "max_ctx"), (shared, dict(scale=0.0), "scale"), (shared, dict(scale=-1.0), "scale"),
    (shared, dict(scale=NAN), "scale"), (shared, dict(scale=INF), "scale"),
    (shared, dict(), "workspace of 0 bytes"), (shared, dict(ws=NONE, n=1 << 30), "workspace"),
    (prompt, dict(q=NONE), "null pointer"), (prompt, dict(scores=NONE), "null pointer"),
    (prompt, dict(D=64), "head_dim"), (prompt, dict(Hq=33), "Hq % Hkv"), (prompt, dict(start=-1), "start"),
    (prompt, dict(start=61), "start + S"), (prompt, dict(scale=NAN), "scale"), (prompt, dict(), "workspace"),
    (prompt, dict(S=1 << 18, S_max=1 << 20, B=1), "2^23"), (prompt, dict(B=-2), "bad B/S"),
    (scored, dict(q=NONE), "null pointer"), (scored, dict(scores=NONE), "null pointer"),
    (scored, dict(D=256), "head_dim"), (scored, dict(Hq=68), "Hq / Hkv"), (scored, dict(max_ctx=0), "max_ctx"),
    (scored, dict(max_ctx=65), "max_ctx"), (scored, dict(scale=-0.1), "scale"), (scored, dict(n=64), "workspace"),
    (scored, dict(ws=NONE, n=1 << 30), "workspace"), (scored, dict(B=-1), "bad B"), (scored, dict(S_max=0), "bad B"),
    (append, dict(raw=NONE), "null pointer"), (append, dict(k=NONE), "null pointer"), (append, dict(D=64), "head_dim"),
    (append, dict(Hq=6), "head counts"), (append, dict(max_pos=0), "max_pos"), (append, dict(B=-1), "bad B"),
    (append, dict(S_max=0), "S_max"),
    (evict, dict(k=NONE), "null pointer"), (evict, dict(ctx=NONE), "null pointer"), (evict, dict(D=64), "head_dim"),
    (evict, dict(B=-1), "B * Hkv"), (evict, dict(B=20000), "B * Hkv"), (evict, dict(S_max=0), "bad S_max"),
    (evict, dict(budget=0), "budget"), (evict, dict(recent=-1), "recent"), (evict, dict(sink=-1), "recent"),
    (evict, dict(recent=30, sink=3), "recent + sink"), (evict, dict(S_out=31, k2=7, v2=8, sc2=9, sp2=10), "31 slots"),
    (evict, dict(S_out=63), "exactly this one"), (evict, dict(v2=8), "exactly this one"),
    (evict, dict(sp2=8), "exactly this one"), (evict, dict(n=1000), "workspace"), (evict, dict(ws=NONE), "workspace"),
]
# addresses that no load of 16 bytes may take, everything else in order
A = 1 << 20
for _fn, _names, _rest in (
        (shared, ("q", "kp", "vp", "k", "v", "out", "ws"), dict(n=A)),
        (prompt, ("q", "k", "v", "out", "ws"), dict(n=A)),
        (scored, ("q", "k", "v", "out", "ws"), dict(n=A)),
        (evict, ("k", "v", "k2", "v2"), dict(sc2=9, sp2=10))):
    _good = {name: (i + 1) * A for i, name in enumerate(_names)}
    REFUSED += [(_fn, {**_good, **_rest, name: _good[name] + 8}, "16-byte aligned") for name in _names]


@pytest.mark.parametrize("fn,change,msg", REFUSED, ids=lambda x: getattr(x, "__name__", None) or str(x)[:40])
def test_c_entries_refuse(fn, change, msg):
    assert fn(_lib.lib(), **change) == ERR
    assert msg in _lib.last_error(), _lib.last_error()


def test_empty_batches_launch_nothing():
    l = _lib.lib()
    assert shared(l, q=NONE, k=NONE, v=NONE, ctx=NONE, out=NONE, B=0, ws=NONE) == 0
    assert shared(l, q=NONE, out=NONE, S=0, ws=NONE) == 0
    assert prompt(l, q=NONE, out=NONE, B=0, ws=NONE) == 0
    assert prompt(l, q=NONE, out=NONE, S=0, ws=NONE) == 0
    assert scored(l, q=NONE, k=NONE, v=NONE, ctx=NONE, scores=NONE, out=NONE, B=0, ws=NONE) == 0
    assert append(l, raw=NONE, pos=NONE, slots=NONE, q=NONE, k=NONE, v=NONE, B=0) == 0
    assert evict(l, k=NONE, v=NONE, sc=NONE, sp=NONE, ctx=NONE, k2=NONE, v2=NONE, sc2=NONE, sp2=NONE, B=0, ws=NONE) == 0


def test_workspace_queries():
    l = _lib.lib()
    assert l.qmoe_attn_shared_workspace(0, 1, 32, 4, 128, 100, 10) == 0
    assert l.qmoe_attn_shared_workspace(2, 1, 32, 4, 128, 1000, 100) > 0
    for bad in [(-1, 1, 32, 4, 128, 1, 1), (1, 1, 33, 4, 128, 1, 1), (1, 1, 32, 4, 64, 1, 1), (1, 1, 32, 4, 128, -1, 1),
                (1, 1, 32, 4, 128, 1, -1), (1, 1, 32, 4, 128, 1 << 23, 1), (1, 1, 32, 4, 128, 1, 1 << 23)]:
        assert l.qmoe_attn_shared_workspace(*bad) == -1, bad
    assert l.qmoe_attn_prefill_scored_workspace(0, 5, 32, 4, 128, 0) == 0
    assert l.qmoe_attn_prefill_scored_workspace(1, 5, 32, 4, 128, 0) >= 5 * 32 * 4
    for bad in [(1, 5, 32, 4, 128, -1), (1, -5, 32, 4, 128, 0), (1, 5, 32, 4, 128, 1 << 22), (1, 5, 32, 3, 128, 0)]:
        assert l.qmoe_attn_prefill_scored_workspace(*bad) == -1, bad
    # 128 outputs, a maximum, a sum and the logits of each split: five of 64 keys, or 17 of 256
    assert l.qmoe_attn_decode_scored_workspace(3, 32, 128, 257) == 3 * 32 * 5 * (130 + 64) * 4
    assert l.qmoe_attn_decode_scored_workspace(3, 32, 128, 4200) == 3 * 32 * 17 * (130 + 256) * 4
    assert l.qmoe_attn_decode_scored_workspace(3, 32, 64, 257) == -1
    assert l.qmoe_attn_decode_scored_workspace(3, 32, 128, -1) == -1
    assert l.qmoe_kv_evict_workspace(2, 4, 100, 50) == 2 * 2 * 4 * 50 * 4
    assert l.qmoe_kv_evict_workspace(2, 4, 100, 500) == 2 * 2 * 4 * 100 * 4
    assert l.qmoe_kv_evict_workspace(2, -4, 100, 50) == -1


def _bf(*shape):
    return torch.zeros(*shape, dtype=torch.bfloat16)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_wrappers_refuse():
    """Without a GPU the wrappers get as far as the operand that says where the
    call runs (the rest of their checks: tests/test_gpu_cache_ops.py)."""
    q, k, kp = _bf(2, 32, 128), _bf(2, 4, 8, 128), _bf(4, 9, 128)
    sc, sp, n = torch.zeros(2, 4, 8), _i(2, 4, 8), _i(2)
    calls = [
        (lambda: ops.attn_shared(q, kp, kp, k, k, n, 2, 1), "q: must be on a GPU"),
        (lambda: ops.attn_shared(q[0], kp, kp, k, k, n, 2, 1), "q must be"),
        (lambda: ops.attn_shared(None, kp, kp, k, k, n, 2, 1), "q: expected a tensor, got NoneType"),
        (lambda: ops.attn_prefill_scored(q, k, k, sc, 1, 2), "q: must be on a GPU"),
        (lambda: ops.attn_decode_scored(q[0], k, k, n, sc), "q must be"),
        (lambda: ops.attn_decode_scored(q, k, k, n, sc), "q: must be on a GPU"),
        (lambda: ops.kv_append(torch.zeros(2, 5120), _bf(128), _bf(128), torch.zeros(4, 64), torch.zeros(4, 64), n, n,
                               32, 4, k, k, 1e-6), "qkv: must be on a GPU"),
        (lambda: ops.kv_append(_bf(2), _bf(128), _bf(128), n, n, n, n, 32, 4, k, k, 1e-6), "qkv must be"),
        (lambda: ops.kv_evict(k, k, sc, sp, n, 4), "k_cache: must be on a GPU"),
        (lambda: ops.kv_evict(k[0], k[0], sc, sp, n, 4), "k_cache must be"),
        (lambda: ops.kv_evict("k", k, sc, sp, n, 4), "k_cache: expected a tensor, got str"),
        (lambda: ops.attn_shared_workspace(1, 1, 32, 4, 128, 1, 1, "cpu"), "on a GPU"),
    ]
    for call, msg in calls:
        with pytest.raises(ValueError, match=msg):
            call()


def test_cache_budget_bookkeeping(monkeypatch):
    """Where the rows stand, on the host and on the device, through a prompt, steps
    and evictions (the eviction itself replaced by a note that it ran)."""
    from types import SimpleNamespace

    from qmoe.attention import CacheBudget

    b = CacheBudget(2, 10, 3, 2, 4, "cpu")
    assert b.capacity == 14
    calls = []
    monkeypatch.setattr(ops, "kv_evict", lambda k, v, sc, sp, ctx, *a: calls.append((k, ctx.tolist(), a)))
    caches = [SimpleNamespace(k=i, v=i, scores=i, slot_pos=i) for i in range(3)]
    b.begin([20, 5])
    assert b.used == [10, 5] and b.slots.tolist() == [10, 5] and b.ctx.tolist() == [11, 6]
    assert b.lengths.tolist() == [20, 5]
    for step in range(5):
        b.make_room(caches)
        assert max(b.used) < b.capacity and b.slots.tolist() == b.used
        b.slots.add_(1)
        b.ctx.add_(1)
        b.advance()
    assert [c[0] for c in calls] == [0, 1, 2] and calls[0][1] == [14, 9] and calls[0][2] == (10, 3, 2)
    assert b.used == [11, 10]
    cache, scores, pos = b.prompt_cache(4, 6, 128)
    scores.fill_(3.0)
    again = b.prompt_cache(4, 5, 128)
    assert again[0] is cache and not bool(again[1].any()) and pos[1, 3].tolist() == list(range(6))
    assert b.prompt_cache(4, 7, 128)[0] is not cache
    for bad in [(2, 0, 0, 0, 4), (2, 10, 8, 3, 4), (2, 10, -1, 0, 4), (2, 10, 0, 0, 0)]:
        with pytest.raises(ValueError, match="at least one slot"):
            CacheBudget(*bad, "cpu")


def test_config_of_the_budget():
    from qmoe.model import MoENeuronConfig

    c = MoENeuronConfig(kv_cache_budget=100)
    assert (c.kv_cache_recent, c.kv_cache_sink, c.kv_cache_slack) == (25, 4, 64)
    c = MoENeuronConfig()
    assert (c.kv_cache_budget, c.kv_cache_recent, c.kv_cache_sink) == (0, 0, 0)
    with pytest.raises(ValueError, match="kv_cache_budget"):
        MoENeuronConfig(kv_cache_budget=-1)


def test_default_split_of_small_budgets():
    from qmoe.attention import check_budget
    from qmoe.model import MoENeuronConfig

    for budget in range(1, 40):
        c = MoENeuronConfig(kv_cache_budget=budget)
        check_budget(budget, c.kv_cache_recent, c.kv_cache_sink)


@pytest.mark.parametrize("bad", ["2", 2.0, None, 2 ** 70, [2]], ids=str)
def test_wrappers_refuse_what_is_no_integer(bad):
    """As every wrapper does: a ValueError that names the argument."""
    q, k, kp = _bf(2, 32, 128), _bf(2, 4, 8, 128), _bf(4, 9, 128)
    sc, sp, n, t, w = torch.zeros(2, 4, 8), _i(2, 4, 8), _i(2), torch.zeros(4, 64), _bf(128)
    raw = torch.zeros(2, 40 * 128)
    calls = {
        "B": [lambda: ops.attn_shared(q, kp, kp, k, k, n, bad, 1), lambda: ops.attn_prefill_scored(q, k, k, sc, bad, 1)],
        "S": [lambda: ops.attn_shared(q, kp, kp, k, k, n, 2, bad), lambda: ops.attn_prefill_scored(q, k, k, sc, 2, bad)],
        "start": [lambda: ops.attn_prefill_scored(q, k, k, sc, 2, 1, bad)],
        "Hq": [lambda: ops.kv_append(raw, w, w, t, t, n, n, bad, 4, k, k, 1e-6)],
        "Hkv": [lambda: ops.kv_append(raw, w, w, t, t, n, n, 32, bad, k, k, 1e-6)],
        "budget": [lambda: ops.kv_evict(k, k, sc, sp, n, bad)],
        "recent": [lambda: ops.kv_evict(k, k, sc, sp, n, 4, bad)],
        "sink": [lambda: ops.kv_evict(k, k, sc, sp, n, 4, 1, bad)],
    }
    for name, fs in calls.items():
        for f in fs:
            with pytest.raises(ValueError, match=f"^{name} must be an integer"):
                f()
    if not isinstance(bad, (int, float)):
        with pytest.raises(ValueError, match="^eps must be a number"):
            ops.kv_append(raw, w, w, t, t, n, n, 32, 4, k, k, bad)


def test_wrappers_refuse_negative_counts():
    q, k, kp, sc, n = _bf(2, 32, 128), _bf(2, 4, 8, 128), _bf(4, 9, 128), torch.zeros(2, 4, 8), _i(2)
    for f in (lambda: ops.attn_shared(q, kp, kp, k, k, n, -2, -1), lambda: ops.attn_shared(q, kp, kp, k, k, n, 2, -1),
              lambda: ops.attn_shared(q, kp, kp, k, k, n, 2 ** 33, 1), lambda: ops.attn_prefill_scored(q, k, k, sc, -1, -2)):
        with pytest.raises(ValueError, match="must be in"):
            f()


BIG = 2 ** 63 - 1


@pytest.mark.parametrize("fn,change,msg", [
    (prompt, dict(start=BIG, ws=NONE), "start + S"), (prompt, dict(start=BIG - 3, ws=NONE), "start + S"),
    (append, dict(Hq=2 ** 62, Hkv=2 ** 62, raw=A, qn=A, kn=A), "head counts"),
    (evict, dict(B=2 ** 33, Hkv=2 ** 31, ws=NONE), "B * Hkv"),
    (scored, dict(B=65535, Hq=32767, Hkv=32767, S_max=2 ** 30 - 1, max_ctx=2 ** 30 - 1, ws=NONE), "too large"),
], ids=["start", "start3", "heads", "rows", "entries"])
def test_c_entries_refuse_sizes_whose_sum_or_product_wraps(fn, change, msg):
    """(With the workspace missing, so that nothing could run if they were not.)"""
    assert fn(_lib.lib(), **change) == ERR
    assert msg in _lib.last_error(), _lib.last_error()


def test_workspace_queries_of_sizes_that_wrap():
    l = _lib.lib()
    for start in (BIG, BIG - 3, (1 << 22) - 4):
        assert l.qmoe_attn_prefill_scored_workspace(1, 5, 32, 4, 128, start) == -1
    assert l.qmoe_attn_prefill_scored_workspace(1, BIG, 32, 4, 128, 0) == -1
    assert l.qmoe_attn_decode_scored_workspace(65535, 32767, 128, 2 ** 30 - 1) == -1
    assert l.qmoe_attn_decode_scored_workspace(2 ** 40, 2 ** 40, 128, 64) == -1
    assert l.qmoe_kv_evict_workspace(2 ** 33, 2 ** 31, 64, 32) == -1
    assert l.qmoe_kv_evict_workspace(1, 1, 2 ** 62, 2 ** 62) == -1
    # as large as the calls take
    assert l.qmoe_attn_prefill_scored_workspace(1, 5, 32, 4, 128, (1 << 22) - 5) > 0
    assert l.qmoe_attn_decode_scored_workspace(64, 32, 128, 1 << 22) == 64 * 32 * (1 << 14) * (130 + 256) * 4
    assert l.qmoe_kv_evict_workspace(8191, 8, 2 ** 30 - 1, 1000) == 2 * 8191 * 8 * 1000 * 4


def test_plain_prefill_attention_refuses_a_start_that_wraps():
    l = _lib.lib()
    for start in (BIG, BIG - 3):
        for call in (lambda: l.qmoe_attn_prefill(1, 1, 1, 1, 4, 32, 4, 128, 64, start, 0.1, 1, NONE),
                     lambda: l.qmoe_attn_prefill_ws(1, 1, 1, 1, 4, 32, 4, 128, 64, start, 0.1, NONE, 0, 1, NONE)):
            assert call() == ERR and "start + S" in _lib.last_error()


def test_scored_prompt_refuses_an_output_on_its_queries():
    """The attention would write over the queries that the scores still need (2 * 4 * 32 rows of 256 bytes)."""
    l, rows = _lib.lib(), 2 * 4 * 32 * 256
    for out in (A, A + rows - 16, A - rows + 16):
        assert prompt(l, q=A, k=4 * A, v=5 * A, ws=6 * A, n=A, out=out) == ERR
        assert "out overlaps q" in _lib.last_error(), _lib.last_error()
    for out in (A + rows, A - rows):
        assert prompt(l, q=A, k=4 * A, v=5 * A, ws=6 * A, out=out) == ERR
        assert "workspace of 0 bytes" in _lib.last_error()
