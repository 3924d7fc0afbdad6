"""The model's options of an attention window and of caches in 4 bits, on the GPU."""

import pytest
import torch

from gpu_util import announce
from test_gpu_cache_model import _model, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["plain", "prefix", "prefix cut down", "budget"])
def test_a_window_of_all_positions_changes_no_bit(dev, kind):
    """Prompts, captured and eager steps and, on plain caches, steps past the last
    position are those of a model without a window."""
    announce(f"a window of all positions, {kind}")
    B = 2
    kw = dict(kv_cache_budget=24, kv_cache_slack=4) if kind == "budget" else {}
    models = [_model(B, 60, **kw), _model(B, 60, attention_window=61, attention_sink=3, **kw)]
    prompts, lengths = _tokens(2, B, 33), torch.tensor([33, 20])
    steps = [_tokens(3 + i, B) for i in range(4)]
    out = []
    for m in models:
        if kind.startswith("prefix"):
            m.share_prefix(_tokens(1, 17), *([9] if kind == "prefix cut down" else []))
        got = [m.prefill(prompts, lengths)]
        got += [m.decode_step(t, lengths + i) for i, t in enumerate(steps)]
        got.append(m.greedy_decode(steps[0], 5, positions=(lengths + 4).int()))
        if kind == "plain":
            got += [m.decode_step(steps[0], torch.tensor([60, 61])), m.decode_step(steps[1], torch.tensor([61, 70]))]
        out.append(got)
    assert all(torch.equal(a, b) for a, b in zip(*out))
