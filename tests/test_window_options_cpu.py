"""The attention window's options: what a checkpoint's config means, when a window
hides nothing, and what is refused when.  The layers are replaced by a recorder, so
no GPU is touched."""

import json

import pytest
import torch

from qmoe import model as qm
from qmoe import ops
from qmoe.attention import Attention, BoundedKVCache, CacheBudget, KVCache, SharedPrefix
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
