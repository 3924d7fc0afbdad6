"""The model's options of an attention window and of caches in 4 bits, on the GPU."""

import pytest
import torch

from gpu_util import announce, bf16_randn
from qmoe import _lib, ops
from qmoe.attention import Attention, KV4Cache, rope_tables
from test_gpu_cache_model import _model, _tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["plain", "prefix", "prefix cut down", "budget", "4 bits"])
def test_a_window_of_all_positions_changes_no_bit(dev, kind):
    """Prompts, captured and eager steps and, on plain caches, steps past the last
    position are those of a model without a window."""
    announce(f"a window of all positions, {kind}")
    B = 2
    kw = {"budget": dict(kv_cache_budget=24, kv_cache_slack=4), "4 bits": dict(kv_cache_bits=4)}.get(kind, {})
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


@pytest.mark.parametrize("B,S", [(3, 22001), (1, 65600)])
def test_a_chunk_of_more_tokens_than_an_append_takes(dev, B, S):
    """Against a call of the append for every 1000 tokens of a row: entries, and
    outputs of the layer, bit for bit."""
    announce(f"chunk of {B} x {S} tokens into a 4-bit cache")
    hq, hkv, d, h, first = 2, 1, 128, 512, 5
    g = torch.Generator(device=dev).manual_seed(B)
    w = torch.ones(d, dtype=torch.bfloat16, device=dev)
    at = Attention(bf16_randn(((hq + 2 * hkv) * d, h), g, dev, 0.05), w, w, bf16_randn((h, hq * d), g, dev, 0.05), hq,
                   hkv, d, 1e-6, 64, 2)
    n = first + S + 3
    cos, sin = rope_tables(d, n, 1e6, dev)
    cache, want = KV4Cache(B, hkv, n, d, dev), ops.kv4_cache(B, hkv, n, d, dev)
    x, res = bf16_randn((B * S, h), g, dev), torch.zeros(B * S, h, device=dev)
    pos = (first + torch.arange(S, dtype=torch.int32, device=dev)).repeat(B)
    at.forward(x, res, pos, B, S, cache, cos, sin, first)
    raw, q = at._raw_of_any(x), []
    for b in range(B):
        for s in range(b * S, (b + 1) * S, 1000):
            e = min(s + 1000, (b + 1) * S)
            q.append(ops.kv4_append(raw[s:e], w, w, cos, sin, pos[s:e], pos[s:e], hq, hkv, tuple(t[b:b + 1] for t in want),
                                    1e-6, S=e - s))
    assert all(torch.equal(a, b) for a, b in zip(cache.tensors, want))
    ctx = torch.full((B,), first + 1, dtype=torch.int32, device=dev)
    o = ops.attn_kv4(torch.cat(q), want, ctx, B, S, 64, 2, max_ctx=first + S)
    ref = torch.zeros_like(res)
    ops.gemm(o, at.wo, _lib.GEMM_ADD_F32, out=ref, workspace=ops.gemm_workspace(B * S, h, hq * d, dev))
    assert torch.equal(res, ref) and bool(torch.isfinite(res).all()) and bool(res.any())
