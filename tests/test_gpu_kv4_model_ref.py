"""A model on caches in 4 bits against the 32-bit oracle on the same entries, and the
entries against the oracle's keys and values."""

import math

import pytest
import torch
import torch.nn.functional as F

import kv4_ref as ref
import model_ref
import oracle
from gpu_util import announce
from qmoe import model as qm
from test_gpu_cache_model import _close, _model, _tokens

pytestmark = pytest.mark.gpu

EXPERTS = 8  # routers give every expert the same logit, and ties go to the first


class Oracle:
    """The model of ``_model`` in 32 bits.  A prompt attends its own keys and values;
    a step attends the entries that the model's caches hold."""

    def __init__(self, m, dev):
        self.m, self.config = m, m.config
        self.params = qm.random_params(m.config, dev, seed=5)
        self.cfg = model_ref.cfg_dict(m.config)
        self.layers = [model_ref.layer_weights_f32(lw, experts=False) for lw in self.params["layers"]]

    def logits(self, ids, pos, window, sink):
        """``ids, pos[B, S]``, after the model's own pass over them; the logits ``[B, S, V]``."""
        B, S = ids.shape
        c = self.cfg
        h = F.embedding(ids, self.params["embed_tokens"]).float()
        for i, w in enumerate(self.layers):
            x = oracle.rmsnorm(h, w["input_layernorm"], c["eps"])
            q, k, v = oracle.qkv_norm_rope(x, w["q_proj"], w["k_proj"], w["v_proj"], w["q_norm"], w["k_norm"], pos,
                                           c["n_q"], c["n_kv"], c["head_dim"], c["eps"], c["theta"])
            held = self.entries(i, k, v, pos)
            if S == 1:
                k, v = held
            entry = torch.arange(k.shape[2], device=ids.device)
            at = pos.view(B, S, 1)
            sees = (entry <= at) & ((entry > at - (window or 1 << 30)) | (entry < sink))
            group = c["n_q"] // c["n_kv"]
            k, v = (t.repeat_interleave(group, 1) for t in (k, v))
            score = q @ k.transpose(2, 3) / math.sqrt(c["head_dim"])
            p = torch.softmax(score.masked_fill(~sees.unsqueeze(1), -math.inf), -1)
            h = h + (p @ v).transpose(1, 2).reshape(B, S, -1) @ w["o_proj"].t()
            y = oracle.rmsnorm(h, w["post_attention_layernorm"], c["eps"]).view(B * S, -1)
            out = sum(oracle.expert_swiglu(y, *model_ref.expert_f32(self.params["layers"][i], e)) for e in range(EXPERTS))
            h = h + (out / EXPERTS).view(B, S, -1)
        last = oracle.rmsnorm(h, self.params["norm"].float(), c["eps"])
        return last @ self.params["lm_head"].float().t()

    def entries(self, i, k, v, pos):
        """Layer i's cache in 32 bits up to the largest position.  The entries at ``pos``
        are the oracle's keys and values, each within half a step of a block's numbers (a
        power at most) and what the model's roundings leave of the oracle's value: a few
        of 2^-9 of the row, a quarter of a power at the least (a block's largest of 32 is
        below 7 powers)."""
        cache = self.m.model.caches()[i].tensors
        held = []
        for x, codes, powers in ((k, *cache[:2]), (v, *cache[2:])):
            values = ref.values(codes, powers)
            scale = ref.two_to(powers).repeat_interleave(ref.BLOCK, -1)
            for b in range(pos.shape[0]):
                at = pos[b].long()
                off = ((values[b, :, at] - x[b].double()).abs() / scale[b, :, at])
                assert float(off.max()) <= 1.25, (i, b, float(off.max()))
            held.append(values[:, :, :int(pos.max()) + 1].float())
        return held


@pytest.mark.parametrize("window,sink", [(0, 0), (24, 3)])
def test_logits_of_a_model_on_four_bits(dev, window, sink):
    """A padded batch's prompt and steps, past the window's length."""
    announce(f"model on 4 bits against the oracle, window {window}")
    B, S = 3, 40
    m = _model(B, 100, kv_cache_bits=4, attention_window=window, attention_sink=sink)
    o = Oracle(m, dev)
    ids, lengths = _tokens(2, B, S), torch.tensor([40, 7, 29])
    got = m.prefill(ids, lengths)
    pos = torch.arange(S, device=dev).expand(B, S)
    want = o.logits(ids.to(dev), pos, window, sink)
    _close(got, want[torch.arange(B, device=dev), lengths.to(dev) - 1], "prompt")
    for i in range(4):
        t = _tokens(10 + i, B)
        got = m.decode_step(t, lengths + i)
        want = o.logits(t.to(dev).view(B, 1), (lengths.to(dev) + i).view(B, 1), window, sink)
        _close(got, want[:, 0], f"step {i}")
