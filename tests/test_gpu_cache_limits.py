"""The model and its layers on shared prefixes and bounded caches at their limits:
prompts and steps past the last position."""

import pytest
import torch

from gpu_util import announce
from qmoe import model as qm

import qwen_with_nki as qn

pytestmark = pytest.mark.gpu


def _model(batch, max_length, **kw):
    """Two layers whose routers send every token to the same experts."""
    nc = qn.MoENeuronConfig(batch_size=batch, max_batch_size=batch, seq_len=max_length, max_length=max_length, seed=5,
                            **kw)
    cfg = qn.Qwen3MoeInferenceConfig(nc)
    cfg.num_hidden_layers, cfg.vocab_size = 2, 4096
    m = qn.NeuronQwen3MoeForCausalLM(None, cfg)
    params = qm.random_params(cfg, m.device, seed=5)
    for layer in params["layers"]:
        layer["router"].zero_()
    m.load(params=params)
    return m


def _tokens(n, *shape):
    return torch.randint(0, 4096, shape, generator=torch.Generator().manual_seed(n))


def _cache_bits(m):
    return [t.clone() for c in m.model.caches() for t in (c.k, c.v, c.scores, c.slot_pos)]


def test_prompt_past_the_last_position(dev):
    announce("prompts past the last position")
    m, P = _model(2, 30), 12
    m.share_prefix(_tokens(1, P))
    want = m.prefill(_tokens(2, 2, 31 - P))  # every position there is
    assert bool(torch.isfinite(want).all())
    with pytest.raises(ValueError, match="positions"):
        m.prefill(_tokens(2, 2, 32 - P))
    assert torch.equal(m.prefill(_tokens(2, 2, 31 - P)), want)
    b = _model(2, 30, kv_cache_budget=16, kv_cache_slack=3)
    want = b.prefill(_tokens(2, 2, 31))
    assert bool(torch.isfinite(want).all())
    bits, used = _cache_bits(b), list(b.model.budget.used)
    with pytest.raises(ValueError, match="positions"):
        b.prefill(_tokens(2, 2, 32))
    assert b.model.budget.used == used and all(torch.equal(x, y) for x, y in zip(_cache_bits(b), bits))


@pytest.mark.parametrize("graphs", [True, False])
def test_steps_past_the_last_position(dev, graphs):
    """One step past the end: refused, with every slot, score and position as it was."""
    announce(f"steps past the last position, graphs {graphs}")
    b = _model(2, 30, kv_cache_budget=12, kv_cache_slack=3, use_hip_graphs=graphs)
    first = b.prefill(_tokens(1, 2, 20)).argmax(-1)
    b.greedy_decode(first, 10)  # positions 20 to 29 of 31
    bits, budget = _cache_bits(b), b.model.budget
    state = [list(budget.used), budget.slots.tolist(), budget.ctx.tolist()]
    for call in (lambda: b.greedy_decode(first, 2), lambda: b.decode_step(first, torch.tensor([3, 31])),
                 lambda: b.decode_step(first, torch.tensor([-1, 3]))):
        with pytest.raises(ValueError, match="positions"):
            call()
    assert [list(budget.used), budget.slots.tolist(), budget.ctx.tolist()] == state and b.position == 30
    assert all(torch.equal(x, y) for x, y in zip(_cache_bits(b), bits))
    assert b.greedy_decode(first, 1).shape == (2, 1) and b.position == 31
    for c in b.model.caches():  # every live slot holds a position
        assert all(bool((c.slot_pos[r, :, :n] >= 0).all()) for r, n in enumerate(budget.used))
    m = _model(2, 30, use_hip_graphs=graphs)
    m.share_prefix(_tokens(1, 12))
    first = m.prefill(_tokens(2, 2, 10)).argmax(-1)
    m.greedy_decode(first, 9)  # the last of 19 positions
    bits = [t.clone() for c in m.model.caches() for t in (c.k, c.v)]
    for call in (lambda: m.greedy_decode(first, 1), lambda: m.decode_step(first)):
        with pytest.raises(ValueError, match="after a prefix of 12"):
            call()
    assert m.position == 19
    assert all(torch.equal(x, y) for x, y in zip([t for c in m.model.caches() for t in (c.k, c.v)], bits))


def test_captured_steps_on_new_caches(dev):
    """Steps captured before the caches were replaced are not replayed on them."""
    announce("captured steps on new caches")
    m, prompt = _model(2, 40), _tokens(1, 2, 9)
    ad = qn.HuggingFaceGenerationAdapter(m)
    want = ad.generate(prompt, max_new_tokens=12)
    old = [c.k for c in m.model.caches()]  # kept, so that a replay into them would show
    m.model.allocate_cache(2, 41)
    before = [t.clone() for t in old]
    assert torch.equal(ad.generate(prompt, max_new_tokens=12), want)
    assert all(torch.equal(x, y) for x, y in zip(old, before))
    assert all(bool(c.k[:, :, 20 - 1].any()) for c in m.model.caches())


def test_a_failed_capture_leaves_the_rows_where_they_stand(dev, monkeypatch):
    announce("a capture that fails in its warm-up")
    outs = []
    for fails in (False, True):
        m = _model(2, 60, kv_cache_budget=16, kv_cache_slack=3)
        first = m.prefill(_tokens(1, 2, 20)).argmax(-1)
        if fails:
            bits, stand = _cache_bits(m), [m.model.budget.slots.tolist(), m.model.budget.ctx.tolist()]
            with monkeypatch.context() as mp:
                mp.setattr(m.model, "logits", lambda h, out=None: (_ for _ in ()).throw(RuntimeError("no memory")))
                with pytest.raises(RuntimeError, match="no memory"):
                    m.greedy_decode(first, 12)
            assert [m.model.budget.slots.tolist(), m.model.budget.ctx.tolist()] == stand
            assert all(torch.equal(x, y) for x, y in zip(_cache_bits(m), bits))
        outs.append(m.greedy_decode(first, 12))
    assert torch.equal(*outs)
