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
