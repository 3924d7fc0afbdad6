"""Host logic of the model on a shared prefix and on bounded caches: what prefill and
the decode steps refuse, what a refusal leaves as it was, and what the caches'
state says.  The layers are replaced by a recorder, so no GPU is touched."""

import pytest
import torch

from qmoe import model as qm
from qmoe import ops
from qmoe.attention import Attention, BoundedKVCache, CacheBudget, KVCache, SharedPrefix

H, E, D, V, HKV = 64, 4, 16, 50, 1


class _Causal(qm.NeuronQwen3MoeForCausalLM):
    """The real host class over a real model object on the CPU whose layers do nothing but note the call."""

    def __init__(self, batch=2, max_length=20, max_position_embeddings=40960, **kw):
        nc = qm.MoENeuronConfig(batch_size=batch, max_batch_size=batch, seq_len=max_length, max_length=max_length,
                                **kw)
        config = qm.Qwen3MoeInferenceConfig(
            nc, num_hidden_layers=2, hidden_size=H, num_experts=E, moe_intermediate_size=32, num_attention_heads=2,
            num_key_value_heads=HKV, head_dim=D, vocab_size=V, num_experts_per_tok=2, tie_word_embeddings=False,
            max_position_embeddings=max_position_embeddings)
        super().__init__(None, config)
        self.device = torch.device("cpu")
        params = qm.random_params(config, "cpu", seed=1)
        self.model = qm.NeuronQwen3MoeModel(config, params)
        self.calls = []
        self.model.hidden = self._hidden
        self.model.logits = lambda h, out=None: torch.zeros(h.shape[0], V)
        self.model.allocate_cache(batch, max_length + 1)
        self.reset()

    def _hidden(self, ids, positions, B, S, start, h_buf=None, max_ctx=None):
        self.calls.append((positions.tolist(), B, S, max_ctx))
        return torch.zeros(B * S, H)


def _tokens(*shape):
    return torch.zeros(*shape, dtype=torch.long)


def _stand(m):
    b = m.model.budget
    return None if b is None else (list(b.used), b.slots.tolist(), b.ctx.tolist(), b.lengths.tolist())


# ------------------------------------------------------------------ prompts past the last position
@pytest.mark.parametrize("kind", ["plain", "prefix", "bounded"])
def test_prefill_refuses_a_prompt_past_the_last_position(kind):
    m = _Causal(**(dict(kv_cache_budget=8, kv_cache_slack=3) if kind == "bounded" else {}))
    P = 6 if kind == "prefix" else 0
    if P:
        m.share_prefix(_tokens(P))
    m.prefill(_tokens(2, 21 - P))  # as many as there are positions
    assert m.calls[-1][2] == 21 - P
    m.reset()
    if kind == "bounded":
        m.decode_step(_tokens(2))
    before, n, position = _stand(m), len(m.calls), m.position
    calls = [lambda: m.prefill(_tokens(2, 22 - P)), lambda: m.forward(_tokens(2, 22 - P))]
    if kind != "plain":  # (there the operators refuse it)
        calls.append(lambda: m.prefill(_tokens(2, 40), torch.tensor([3, 4])))
    for call in calls:
        with pytest.raises(ValueError, match="positions"):
            call()
    assert (_stand(m), len(m.calls), m.position) == (before, n, position)


def test_padding_past_the_tables_of_a_plain_cache():
    """Positions that the model has no embedding for, in rows that end before them."""
    m = _Causal(max_position_embeddings=10)
    assert m._positions() == 10 and m.model.caches()[0].capacity == 21
    m.prefill(_tokens(2, 15), torch.tensor([9, 10]))
    assert m.calls[-1][2] == 15
    for lengths in (torch.tensor([9, 11]), None):
        with pytest.raises(ValueError, match="positions"):
            m.prefill(_tokens(2, 15), lengths)


@pytest.mark.parametrize("bounded", [False, True])
def test_attention_refuses_chunks_past_the_tables_or_the_cache(monkeypatch, bounded):
    """The layer itself: the projection would write neither queries nor entries there."""
    d, hq, hkv, h = 128, 4, 2, 512
    w = torch.ones(d, dtype=torch.bfloat16)
    a = Attention(torch.zeros((hq + 2 * hkv) * d, h, dtype=torch.bfloat16), w, w,
                  torch.zeros(h, hq * d, dtype=torch.bfloat16), hq, hkv, d, 1e-6)
    for name in ("gemm", "qkv_norm_rope", "attn_shared", "attn_prefill_scored", "kv_evict"):
        monkeypatch.setattr(ops, name, lambda *args, **kw: pytest.fail("launched"))
    if bounded:
        cache, chunks = BoundedKVCache(CacheBudget(1, 8, 2, 1, 3, "cpu"), hkv, d), [(0, 11), (0, 400)]
    else:
        cache, chunks = KVCache(1, hkv, 8, d, "cpu"), [(0, 9), (5, 4), (9, 2), (-1, 4)]
        cache.prefix = SharedPrefix(cache.k[0], cache.v[0], 4)
    rope = torch.zeros(10, d // 2)
    for start, S in chunks:
        x, pos = torch.zeros(S, h, dtype=torch.bfloat16), torch.arange(S, dtype=torch.int32) + start
        with pytest.raises(ValueError, match="start \\+ S <= "):
            a.forward(x, torch.zeros(S, h), pos, 1, S, cache, rope, rope, start)


# ------------------------------------------------------------------ steps past the last position
@pytest.mark.parametrize("kind", ["prefix", "bounded"])
def test_steps_past_the_last_position_are_refused(kind):
    m = _Causal(**(dict(kv_cache_budget=8, kv_cache_slack=30) if kind == "bounded" else {}))
    P = 6 if kind == "prefix" else 0
    if P:
        m.share_prefix(_tokens(P))
    end = 21 - P  # positions 0 to end - 1
    m.prefill(_tokens(2, end - 2))
    m.decode_step(_tokens(2), torch.tensor([0, end - 2]))
    m.decode_step(_tokens(2))
    assert m.calls[-1][0] == [end - 1] * 2 and m.position == end
    before, n = _stand(m), len(m.calls)
    for call in (lambda: m.decode_step(_tokens(2)), lambda: m.forward(_tokens(2, 1)),
                 lambda: m.decode_step(_tokens(2), torch.tensor([0, end])),
                 lambda: m.decode_step(_tokens(2), torch.tensor([-1, 0])),
                 lambda: m.greedy_decode(_tokens(2), 1, use_graph=False),
                 lambda: m.greedy_decode(_tokens(2), 1, use_graph=True),
                 lambda: m.greedy_decode(_tokens(2), 4, False, torch.tensor([0, end - 3])),
                 lambda: m.greedy_decode(_tokens(2), 4, True, torch.tensor([0, end - 3])),
                 lambda: m.greedy_decode(_tokens(2), 1, True, torch.tensor([-1, 3]))):
        with pytest.raises(ValueError, match="positions"):
            call()
        assert (_stand(m), len(m.calls), m.position) == (before, n, end)


def test_steps_past_the_last_position_of_plain_caches():
    """They write nothing and get zeros, as the fused decode says: not refused."""
    m = _Causal()
    m.prefill(_tokens(2, 21))
    m.decode_step(_tokens(2))
    m.decode_step(_tokens(2), torch.tensor([3, 30]))
    assert m.position == 31


# ------------------------------------------------------------------ new caches
def test_new_caches_have_no_prefix():
    m = _Causal()
    m.share_prefix(_tokens(6))
    assert m.model.base == 6 and m._positions() == 15 and not m._contiguous()
    m.model.allocate_cache(3, 21)
    assert m.model.base == 0 and m._positions() == 21 and m._contiguous()
    assert all(c.prefix is None and c.k.shape[0] == 3 for c in m.model.caches())
    m.prefill(_tokens(3, 21))
    m.model.config.neuron_config.kv_cache_budget = 8
    m.model.allocate_cache(3, 21)
    assert m._budget_of(3) is m.model.budget and m.model.caches()[0].state is m.model.budget
    m.model.config.neuron_config.kv_cache_budget = 0  # and no state of bounded caches on plain ones
    m.model.allocate_cache(2, 21)
    assert m.model.budget is None and m._contiguous()


def test_captured_steps_go_with_the_caches(monkeypatch):
    """A step that was captured with caches that are gone would write into memory
    that something else has by now (the capture itself needs a GPU: its place in
    the table is what is looked at)."""
    monkeypatch.setattr(ops, "argmax_workspace", lambda *args: None)
    m = _Causal()
    state = m._decode_state(2)
    m._graphs[("decode", 2, 21)] = captured = object()
    m._graphs[("verify", 4)] = captured
    assert m._decode_graph(2, 21) is captured and m._verify_graph(4) is captured and m._decode_state(2) is state
    m.model.allocate_cache(2, 21)
    again = m._decode_state(2)
    assert again is not state and list(m._graphs) == [("state", 2)]
    assert m._decode_state(2) is again
    m._graphs[("decode", 2, 21)] = captured
    m.load(params=qm.random_params(m.config, "cpu", seed=2))
    assert not m._graphs


def test_a_failed_capture_leaves_the_rows_where_they_stand(monkeypatch):
    def fail(*args, **kw):
        raise RuntimeError("no memory")

    monkeypatch.setattr(ops, "argmax_workspace", lambda *args: None)
    m = _Causal(kv_cache_budget=8, kv_cache_slack=3)
    m.prefill(_tokens(2, 7), torch.tensor([7, 4]))
    before = _stand(m)
    assert before[1:3] == ([7, 4], [8, 5])
    monkeypatch.setattr(torch.cuda, "Stream", fail)
    with pytest.raises(RuntimeError, match="no memory"):
        m._decode_graph(2, 11)
    assert _stand(m) == before and ("decode", 2, 11) not in m._graphs


# ------------------------------------------------------------------ a step's projection, by its operands
def _off(offset, *shape):
    """bf16 zeros, ``offset`` bytes past a 16-byte boundary."""
    n = 1
    for k in shape:
        n *= k
    t = torch.zeros(n + 16, dtype=torch.bfloat16)
    first = (-t.data_ptr() % 16 + offset) // 2
    return t[first:first + n].view(shape)


def _step(monkeypatch, kind, B, h, w_off=0, x_off=0, hq=4, hkv=2):
    """The names of a step's calls up to its attention, and the operands of its GEMMs."""
    d, names, gemms = 128, [], []

    def record(name, result):
        def fn(*args, **kw):
            names.append(name)
            if name == "gemm":
                gemms.append(args[:2])
            return result(*args)
        monkeypatch.setattr(ops, name, fn)

    rows = torch.zeros(B, hq * d, dtype=torch.bfloat16)
    record("gemm", lambda a, b, *_: torch.empty(a.shape[0], b.shape[0]))
    record("qkv_norm_rope", lambda *_: rows.view(B, hq, d))
    record("kv_append", lambda raw, *_: rows.view(B, hq, d) if raw.shape == (B, (hq + 2 * hkv) * d)
           and raw.is_contiguous() else pytest.fail(str(raw.shape)))
    record("attn_shared", lambda *_: rows)
    record("attn_decode_scored", lambda *_: rows)
    monkeypatch.setattr(ops, "gemm_workspace", lambda *_: None)
    w = torch.ones(d, dtype=torch.bfloat16)
    a = Attention(_off(w_off, (hq + 2 * hkv) * d, h), w, w, torch.zeros(h, hq * d, dtype=torch.bfloat16), hq, hkv, d,
                  1e-6)
    if kind == "bounded":
        cache = BoundedKVCache(CacheBudget(B, 8, 2, 1, 3, "cpu"), hkv, d)
    else:
        cache = KVCache(B, hkv, 8, d, "cpu")
        cache.prefix = SharedPrefix(cache.k[0], cache.v[0], 4)
    rope = torch.zeros(10, d // 2)
    a.forward(_off(x_off, B, h), torch.zeros(B, h), torch.zeros(B, dtype=torch.int32), B, 1, cache, rope, rope)
    return names[:-1], gemms[:-1]  # (the last one is the output projection)


ATTN = {"prefix": "attn_shared", "bounded": "attn_decode_scored"}


@pytest.mark.parametrize("kind", ["prefix", "bounded"])
@pytest.mark.parametrize("B,h", [(1, 2048), (16, 2048), (17, 2048), (20, 512), (64, 1024), (9, 4096)])
def test_steps_on_the_alignment_take_the_raw_projection(monkeypatch, kind, B, h):
    names, gemms = _step(monkeypatch, kind, B, h)
    assert names == ["gemm", "kv_append", ATTN[kind]] and len(gemms) == 1


@pytest.mark.parametrize("kind", ["prefix", "bounded"])
@pytest.mark.parametrize("B,h", [(17, 2048), (20, 512), (64, 1024), (9, 4096), (33, 4096), (70, 2048)])
@pytest.mark.parametrize("w_off,x_off", [(4, 0), (0, 8), (12, 2)])
def test_steps_off_the_alignment(monkeypatch, kind, B, h, w_off, x_off):
    """As on plain caches: no GEMM gets operands that its LDS-DMA kernels do not take."""
    names, gemms = _step(monkeypatch, kind, B, h, w_off, x_off)
    if kind == "prefix":
        assert names == ["qkv_norm_rope", "attn_shared"]
    else:
        assert names == ["gemm", "kv_append", "attn_decode_scored"]
    assert all(t.data_ptr() % 16 == 0 for operands in gemms for t in operands)


@pytest.mark.parametrize("kind", ["prefix", "bounded"])
def test_steps_whose_weights_the_gemm_refuses(monkeypatch, kind):
    # 2 GiB of weights (never touched), and a hidden size that the GEMV does not take
    names, gemms = _step(monkeypatch, kind, 9, 4096, hq=1792, hkv=128)
    assert names[0] == ("qkv_norm_rope" if kind == "prefix" else "gemm")
    assert all(b.numel() * 2 < 2**31 for _, b in gemms)
    assert kind == "prefix" or sum(b.shape[0] for _, b in gemms) == 2048 * 128
    names, gemms = _step(monkeypatch, kind, 3, 576)
    assert names[0] == ("qkv_norm_rope" if kind == "prefix" else "gemm")
    assert all(a.shape[0] > 16 for a, _ in gemms)


# ------------------------------------------------------------------ the layer's own cache
class _OnGpu(torch.Tensor):
    is_cuda = True  # as far as the layer's first check goes


def test_a_refused_cache_is_not_the_layers(monkeypatch):
    m = _Causal()
    layer, own = m.model.layers[0], m.model.caches()[0]
    monkeypatch.setattr(layer, "run", lambda *args, **kw: pytest.fail("ran"))
    x = torch.zeros(2, 3, H).as_subclass(_OnGpu)
    prefixed, small = KVCache(2, HKV, 30, D, "cpu"), KVCache(2, HKV, 2, D, "cpu")
    prefixed.prefix = SharedPrefix(prefixed.k[0], prefixed.v[0], 4)
    bounded = BoundedKVCache(CacheBudget(2, 8, 2, 1, 3, "cpu"), HKV, D)
    for cache, why in ((prefixed, "driven by the model"), (bounded, "driven by the model"),
                       (KVCache(3, HKV, 30, D, "cpu"), "no KV cache"), (small, "beyond the KV cache")):
        with pytest.raises(ValueError, match=why):
            layer.forward(x, past_key_value=cache)
        assert layer.cache is own


# ------------------------------------------------------------------ eager steps run in the captured step's bucket
def test_eager_steps_take_the_bucket(monkeypatch):
    m = _Causal(max_length=700)
    m.prefill(_tokens(2, 250))
    m.decode_step(_tokens(2))
    assert m.calls[-1][3] is None  # plain caches split by their capacity
    m.share_prefix(_tokens(90))
    m.prefill(_tokens(2, 250))
    for pos, bucket in ((250, 256), (255, 256), (256, 512), (512, 701)):
        m.decode_step(_tokens(2), torch.tensor([3, pos]))
        assert m.calls[-1][3] == bucket
    monkeypatch.setattr(ops, "kv_evict", lambda *args: None)
    m = _Causal(max_length=900, kv_cache_budget=400, kv_cache_slack=112)
    m.prefill(_tokens(2, 255))
    for used, bucket in ((256, 256), (257, 512)):
        m.decode_step(_tokens(2))
        assert m.calls[-1][3] == bucket and m.model.budget.used == [used, used]
    m.prefill(_tokens(2, 600))
    for _ in range(113):  # the last one evicts first
        m.decode_step(_tokens(2))
    assert m.calls[-1][3] == 512 and m.model.budget.used == [401, 401]


# ------------------------------------------------------------------ lengths of padded prompts
@pytest.mark.parametrize("kind", ["plain", "prefix", "bounded"])
def test_prefill_refuses_lengths_outside_the_prompt(kind):
    """A row's last token is looked up behind them, and a bounded row stands at them."""
    m = _Causal(**(dict(kv_cache_budget=8, kv_cache_slack=3) if kind == "bounded" else {}))
    if kind == "prefix":
        m.share_prefix(_tokens(6))
    m.prefill(_tokens(2, 5), torch.tensor([5, 1]))
    before, n = _stand(m), len(m.calls)
    for bad in ([6, 1], [5, 0], [-1, 5], [5], [5, 5, 5]):
        with pytest.raises(ValueError, match="lengths"):
            m.prefill(_tokens(2, 5), torch.tensor(bad))
    with pytest.raises(ValueError, match="lengths"):
        m.prefill(_tokens(2, 1), torch.tensor([1, 2]))
    assert (_stand(m), len(m.calls), m.position) == (before, n, 5)


def test_a_prefix_set_on_the_model_itself(monkeypatch):
    """As through share_prefix: captured steps go with the prefix that they saw, and
    bounded caches, whose attention would not see it, take none."""
    monkeypatch.setattr(ops, "argmax_workspace", lambda *args: None)
    m = _Causal()
    for P in (4, 6, 0):
        state = m._decode_state(2)
        m._graphs[("decode", 2, 21)] = object()
        m.model.set_prefix(_tokens(1, P))
        assert m._decode_state(2) is not state and list(m._graphs) == [("state", 2)]
    state = m._decode_state(2)
    with pytest.raises(ValueError, match="no position"):  # refused: nothing changes
        m.model.set_prefix(_tokens(1, 21))
    assert m._decode_state(2) is state
    m = _Causal(kv_cache_budget=8)
    for call in (lambda: m.model.set_prefix(_tokens(1, 4)), lambda: m.share_prefix(_tokens(4))):
        with pytest.raises(ValueError, match="kv_cache_budget"):
            call()
    assert m.model.base == 0
