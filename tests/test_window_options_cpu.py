"""The attention window's options: what a checkpoint's config means, when a window
hides nothing, and what is refused when.  The layers are replaced by a recorder, so
no GPU is touched."""

import json

import pytest
import torch

from qmoe import model as qm
from qmoe import ops
from qmoe.attention import Attention, BoundedKVCache, CacheBudget, KV4Cache, KVCache, SharedPrefix
from test_cache_model_cpu import _Causal, _tokens


def _config(extra=None, **kw):
    def load(cfg):
        for k, v in (extra or {}).items():
            setattr(cfg, k, v)
    return qm.Qwen3MoeInferenceConfig(qm.MoENeuronConfig(**kw), load_config=load)


# ------------------------------------------------------------------ the checkpoint's config
def test_a_window_in_use_without_a_length_has_the_published_default(tmp_path):
    """The published config class has 4096 for a key that is absent, and no window for
    one that is null."""
    assert _config({"use_sliding_window": True}).window() == 4096
    assert _config({"use_sliding_window": True, "sliding_window": None}).window() == 0
    assert _config({"use_sliding_window": False}).window() == 0
    assert _config({"use_sliding_window": True}, attention_window=0).window() == 0
    assert _config({"use_sliding_window": True}, attention_window=100).window() == 100
    for written, want in (({"use_sliding_window": True}, 4096), ({"use_sliding_window": True, "sliding_window": None}, 0),
                          ({"use_sliding_window": True, "sliding_window": 77}, 77), ({}, 0)):
        (tmp_path / "config.json").write_text(json.dumps(written))
        config = qm.Qwen3MoeInferenceConfig(qm.MoENeuronConfig(), qm.load_pretrained_config(str(tmp_path)))
        assert config.window() == want, written


@pytest.mark.parametrize("kw", [{}, {"use_sliding_window": True}, {"use_sliding_window": True, "sliding_window": None},
                                {"use_sliding_window": True, "sliding_window": 77}, {"sliding_window": 77}], ids=str)
def test_the_window_of_the_published_config_class(kw):
    published = pytest.importorskip("transformers").Qwen3MoeConfig(**kw)
    assert _config(kw).window() == (published.sliding_window or 0)


# ------------------------------------------------------------------ a window that hides nothing
@pytest.mark.parametrize("window", [21, 4096])
def test_a_window_of_all_positions_leaves_plain_caches_as_they_are(window):
    """Their steps past the last position are zero rows, not refused."""
    m = _Causal(attention_window=window, attention_sink=2)
    assert m.model.plain_attention() and not m.config.hides()
    m.prefill(_tokens(2, 21))
    m.decode_step(_tokens(2))
    assert m.calls[-1][3] is None  # no bucket, as without a window
    m.decode_step(_tokens(2), torch.tensor([3, 30]))
    assert m.position == 31
    shorter = _Causal(attention_window=20)
    assert shorter.config.hides() and not shorter.model.plain_attention()
    few = _Causal(attention_window=10, max_position_embeddings=10)  # positions that the cache has room past
    few.prefill(_tokens(2, 10))
    few.decode_step(_tokens(2))
    assert few.model.plain_attention() and few.model.layers[0].cache.capacity == 21


@pytest.mark.parametrize("window", [21, 4096])
def test_a_window_of_all_positions_goes_with_prefixes_and_budgets(window):
    m = _Causal(attention_window=window)
    m.share_prefix(_tokens(6))
    prefix = m.model.caches()[0].prefix
    assert m.model.base == 6 and prefix.length == 6 and prefix.tokens == 6
    m.prefill(_tokens(2, 10))
    m.decode_step(_tokens(2))
    b = _Causal(attention_window=window, kv_cache_budget=8, kv_cache_slack=3)
    b.prefill(_tokens(2, 10))
    b.decode_step(_tokens(2))
    assert isinstance(b.model.caches()[0], BoundedKVCache)


@pytest.mark.parametrize("kind", ["prefix", "prefix cut down", "bounded"])
@pytest.mark.parametrize("hides", [True, False])
def test_the_layer_takes_special_caches_unless_its_window_hides_something(monkeypatch, kind, hides):
    """Positions are those of the prefix (all its tokens, also those that were dropped)
    and of the tables behind it."""
    d, hq, hkv, h, rows = 128, 4, 2, 512, 10
    w = torch.ones(d, dtype=torch.bfloat16)
    before = {"prefix": 4, "prefix cut down": 9, "bounded": 0}[kind]
    a = Attention(torch.zeros((hq + 2 * hkv) * d, h, dtype=torch.bfloat16), w, w,
                  torch.zeros(h, hq * d, dtype=torch.bfloat16), hq, hkv, d, 1e-6, before + rows - hides, 1)
    called = []
    monkeypatch.setattr(Attention, "_special", lambda self, *args: called.append(args) or torch.zeros(2, hq * d))
    monkeypatch.setattr(ops, "gemm", lambda *args, **kw: None)
    monkeypatch.setattr(ops, "gemm_workspace", lambda *args: None)
    if kind == "bounded":
        cache = BoundedKVCache(CacheBudget(1, 8, 2, 1, 3, "cpu"), hkv, d)
    else:
        cache = KVCache(1, hkv, 8, d, "cpu")
        cache.prefix = SharedPrefix(cache.k[0], cache.v[0], 4, *([9] if kind == "prefix cut down" else []))
    rope = torch.zeros(rows, d // 2)
    call = lambda: a.forward(torch.zeros(2, h, dtype=torch.bfloat16), torch.zeros(2, h),
                             torch.arange(2, dtype=torch.int32), 1, 2, cache, rope, rope)
    if hides:
        with pytest.raises(ValueError, match="no window"):
            call()
    else:
        call()
    assert len(called) == (not hides)


@pytest.mark.parametrize("window,S,plain", [(0, 8, True), (8, 8, True), (7, 8, False), (9, 8, True), (20, 21, False)])
def test_a_prompt_no_longer_than_the_window_is_attended_without_it(monkeypatch, window, S, plain):
    """Also on its way to a cache in 4 bits."""
    d, h = 128, 512
    w = torch.ones(d, dtype=torch.bfloat16)
    a = Attention(torch.zeros(3 * d, h, dtype=torch.bfloat16), w, w, torch.zeros(h, d, dtype=torch.bfloat16), 1, 1, d,
                  1e-6, window, 2)
    called = []
    for name in ("attn_window", "attn_prefill"):
        monkeypatch.setattr(ops, name, lambda *args, name=name, **kw: called.append(name) or torch.zeros(S, d))
    for name in ("qkv_norm_rope", "gemm", "gemm_workspace", "kv4_store", "attn_prefill_workspace"):
        monkeypatch.setattr(ops, name, lambda *args, **kw: None)
    monkeypatch.setattr(ops, "qkv_norm_rope_workspace", lambda *args: 0)
    rope = torch.zeros(30, d // 2)
    for cache in (KV4Cache(1, 1, 30, d, "cpu"), KVCache(1, 1, 30, d, "cpu")):
        a.forward(torch.zeros(S, h, dtype=torch.bfloat16), torch.zeros(S, h), torch.arange(S, dtype=torch.int32), 1, S,
                  cache, rope, rope)
    assert called == ["attn_prefill" if plain else "attn_window"] * 2


# ------------------------------------------------------------------ refusals
def test_a_budget_with_a_window_that_hides_something_is_refused_by_the_config():
    """Before any weight is read; a checkpoint's own window too."""
    for extra, kw in ((None, dict(attention_window=32)), ({"use_sliding_window": True}, dict(max_length=5000)),
                      ({"use_sliding_window": True, "sliding_window": 77}, {})):
        with pytest.raises(ValueError, match="window"):
            _config(extra, kv_cache_budget=64, **kw)
    for extra, kw in ((None, dict(attention_window=641)), ({"use_sliding_window": True}, {}),
                      ({"use_sliding_window": True, "sliding_window": 77}, dict(attention_window=0))):
        assert not _config(extra, kv_cache_budget=64, **kw).hides()
    with pytest.raises(ValueError, match="negative"):
        _config({"sliding_window": -5, "use_sliding_window": True})


@pytest.mark.parametrize("kw", [dict(kv_cache_bits=4), dict(attention_window=5)], ids=str)
def test_speculation_past_the_last_position_is_refused_before_it_begins(kw):
    """As the plain steps are: a verified token there would come from a zero query."""
    m = _Causal(batch=1, max_position_embeddings=14, **kw)
    assert m._positions() == 14 and m.model.caches()[0].capacity == 21
    greedy = lambda ids, n: (m.reset(), m.prefill(ids), m.greedy_decode(ids[:, -1], n - 1, use_graph=False))
    for new in (6, 9):
        with pytest.raises(ValueError, match="steps at positions"):
            greedy(_tokens(1, 10), new)
        n = len(m.calls)
        with pytest.raises(ValueError, match="steps at positions"):
            m.spec_generate(_tokens(1, 10), new)
        assert len(m.calls) == n
    m._top(torch.tensor([10]), 4)  # four steps give five tokens with the prompt's
    m.greedy_decode = lambda tok, k: torch.ones(1, 1, dtype=torch.long)
    m._verify_graph = lambda S: pytest.fail("no candidates here")
    out, _ = m.spec_generate(torch.arange(10).view(1, 10) + 20, 5, ngram=9, ngram_min=9)
    assert out.shape == (1, 15)


def test_speculation_past_the_last_position_of_plain_caches():
    """Not refused, as the plain steps are not."""
    m = _Causal(batch=1, max_position_embeddings=14, attention_window=14)
    m.greedy_decode = lambda tok, k: torch.ones(1, 1, dtype=torch.long)
    m._verify_graph = lambda S: pytest.fail("no candidates here")
    out, _ = m.spec_generate(torch.arange(10).view(1, 10) + 20, 9, ngram=9, ngram_min=9)
    assert out.shape == (1, 19)


# ------------------------------------------------------------------ large chunks
@pytest.mark.parametrize("B,S,calls", [(2, 5, 1), (1, 65535, 1), (64, 1024, 2), (3, 30000, 2), (7, 40000, 7),
                                       (2, 70000, 4), (1, 131070, 2), (60000, 2, 2)])
def test_chunks_of_any_size_go_to_a_cache_of_four_bits(monkeypatch, B, S, calls):
    """A call of the append takes fewer than 65536 tokens: every token of a larger chunk
    goes once, with its own position, row of the batch and query."""
    d, h = 128, 512
    w = torch.ones(d, dtype=torch.bfloat16)
    a = Attention(torch.zeros(3 * d, h, dtype=torch.bfloat16), w, w, torch.zeros(h, d, dtype=torch.bfloat16), 1, 1, d,
                  1e-6)
    token = torch.arange(B * S, dtype=torch.float32).view(-1, 1)
    seen, made, count = [], [], [0]

    def append(qkv, qn, kn, cos, sin, positions, slots, hq, hkv, cache, eps, S=1, q_out=None):
        n = qkv.shape[0]
        count[0] += 1
        assert n < 65536 and n == cache[0].shape[0] * S and torch.equal(positions, slots)
        first = cache[0].flatten()[0] if cache[0].numel() else 0
        row = first + torch.arange(cache[0].shape[0]).repeat_interleave(S)
        seen.append(torch.stack([qkv[:, 0].long(), positions.long(), row]))
        q_out = torch.empty(n, hq) if q_out is None else q_out
        q_out.view(n, -1)[:] = (qkv[:, :1] % 251).to(q_out.dtype)  # exact in bf16
        return q_out

    def attend(q, cache, ctx, B, S, *args, **kw):
        made.append(q)
        return torch.zeros(B * S, d, dtype=torch.bfloat16)

    monkeypatch.setattr(ops, "kv4_append", append)
    monkeypatch.setattr(ops, "attn_kv4", attend)
    monkeypatch.setattr(ops, "gemm", lambda *args, **kw: None)
    monkeypatch.setattr(ops, "gemm_workspace", lambda *args: None)
    monkeypatch.setattr(Attention, "_raw", lambda self, *args: token)
    cache = KV4Cache(1, 1, 1, d, "cpu")
    cache.tensors = tuple(torch.arange(B).view(B, 1, 1, 1) for _ in range(4))
    cache.k = torch.empty(B, 1, 1 << 20, 0)
    positions = (9 + torch.arange(S, dtype=torch.int32)).repeat(B)
    rope = torch.zeros(1, d // 2)
    a.forward(torch.zeros(B * S, h, dtype=torch.bfloat16)[:0], torch.zeros(0, h), positions, B, S, cache, rope, rope, 9)
    assert count[0] == calls
    seen = torch.cat(seen, 1)
    assert torch.equal(seen[0], torch.arange(B * S)) and torch.equal(seen[1], positions.long())
    assert torch.equal(seen[2], torch.arange(B).repeat_interleave(S))
    assert torch.equal(made[0].view(B * S, -1)[:, 0].float(), token[:, 0] % 251)
