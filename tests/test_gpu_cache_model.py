"""The cache operators as the package uses them: a decode batch's steps together
(append, scored attention, eviction; a prompt cut down and then shared), captured
into graphs, and the model's generation on a shared prefix and on bounded
caches."""

import math

import pytest
import torch

import cache_ref as ref
from gpu_util import announce, bf16_randn, mean_rel
from qmoe import model as qm
from qmoe import ops
from qmoe.attention import (FUSED_DECODE_MAX_ROWS, Attention, BoundedKVCache, CacheBudget, KVCache, SharedPrefix,
                            rope_tables)

import qwen_with_nki as qn

pytestmark = pytest.mark.gpu

HQ, HKV, D, H = 32, 4, 128, 2048
SCALE = 1.0 / math.sqrt(D)


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _check(got, want, bound, what):
    worst = float(((got.double() - want).abs() / bound).max())
    print(f"  {what}: worst error {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, what


# ------------------------------------------------------------------ operators together
def test_prompt_evict_and_steps_together(dev):
    """A padded batch's prompt with scores, its eviction into bounded caches, and
    decode steps with evictions between them; every result against 64 bits from
    the caches as the kernels left them."""
    B, S, lengths, budget, recent, sink, cap = 3, 90, [90, 41, 77], 40, 8, 2, 45
    announce("prompt, eviction, steps")
    g = _gen(dev, 3)
    q = bf16_randn((B * S, HQ, D), g, dev, 2.0)
    k, v = bf16_randn((B, HKV, S, D), g, dev), bf16_randn((B, HKV, S, D), g, dev)
    sc = torch.zeros(B, HKV, S, device=dev)
    pos = torch.arange(S, dtype=torch.int32, device=dev).repeat(B, HKV, 1)
    n = _i32(lengths, dev)
    out = ops.attn_prefill_scored(q, k, v, sc, B, S, lengths=n)
    want, bound, add, off = ref.scored(q, k, v, [1] * B, B, S, lengths, SCALE)
    _check(out, want, bound, "prompt")
    _check(sc, add, off + 1e-12, "prompt scores")
    cache = [torch.zeros(B, HKV, cap, D, dtype=torch.bfloat16, device=dev),
             torch.zeros(B, HKV, cap, D, dtype=torch.bfloat16, device=dev),
             torch.zeros(B, HKV, cap, device=dev), torch.zeros(B, HKV, cap, dtype=torch.int32, device=dev)]
    expect = ref.evict(k.cpu(), v.cpu(), sc.cpu(), pos.cpu(), lengths, budget, recent, sink, [t.cpu() for t in cache])
    ops.kv_evict(k, v, sc, pos, n, budget, recent, sink, out=tuple(cache))
    for x, y in zip(cache, expect):
        assert torch.equal(x.cpu(), y)
    kc, vc, scc, spc = cache
    cos, sin = rope_tables(D, 400, 1e6, dev)
    ones = torch.ones(D, dtype=torch.bfloat16, device=dev)
    used, at = [min(x, budget) for x in lengths], list(lengths)
    for step in range(14):
        if max(used) == cap:
            expect = ref.evict(*[t.cpu() for t in cache], used, budget, recent, sink)
            ops.kv_evict(*cache, _i32(used, dev), budget, recent, sink)
            for x, y in zip(cache, expect):
                assert torch.equal(x.cpu(), y)
            used = [min(x, budget) for x in used]
        raw = torch.randn(B, (HQ + 2 * HKV) * D, generator=g, device=dev) * 2
        qs = ops.kv_append(raw, ones, ones, cos, sin, _i32(at, dev), _i32(used, dev), HQ, HKV, kc, vc, 1e-6,
                           scores=scc, slot_pos=spc)
        used = [x + 1 for x in used]
        before = scc.double()
        out = ops.attn_decode_scored(qs, kc, vc, _i32(used, dev), scc)
        want, bound, add, off = ref.scored(qs, kc, vc, used, B, 1, None, SCALE)
        _check(out, want, bound, f"step {step}")
        _check(scc, before + add, off + 2 * ref.F32 * (before + add) + 1e-12, f"scores {step}")
        for b in range(B):
            live = spc[b, :, :used[b]]
            assert bool((live >= 0).all()) and bool((live[:, used[b] - 1] == at[b]).all())
            for h in range(HKV):  # a position is held once, the last ones and the first always
                held = set(live[h].tolist())
                assert len(held) == used[b]
                assert set(range(sink)) <= held and set(range(at[b] - recent + 1, at[b] + 1)) <= held
        at = [x + 1 for x in at]


def test_prompt_cut_down_then_shared(dev):
    """A long prompt's cache is cut down to a budget, then shared by a batch."""
    S, B, budget = 300, 5, 96
    announce("cut down, then shared")
    g = _gen(dev, 4)
    q0 = bf16_randn((S, HQ, D), g, dev, 2.0)
    k0, v0 = bf16_randn((1, HKV, S, D), g, dev), bf16_randn((1, HKV, S, D), g, dev)
    sc = torch.zeros(1, HKV, S, device=dev)
    pos = torch.arange(S, dtype=torch.int32, device=dev).repeat(1, HKV, 1)
    ops.attn_prefill_scored(q0, k0, v0, sc, 1, S)
    ops.kv_evict(k0, v0, sc, pos, _i32([S], dev), budget, recent=16, sink=4)
    ctx = [1, 7, 30, 0, 33]
    q = bf16_randn((B, HQ, D), g, dev, 2.0)
    k, v = bf16_randn((B, HKV, 33, D), g, dev), bf16_randn((B, HKV, 33, D), g, dev)
    out = ops.attn_shared(q, k0[0], v0[0], k, v, _i32(ctx, dev), B, 1, prefix_len=budget)
    want, bound = ref.shared(q, k0[0], v0[0], k, v, ctx, B, 1, budget, 33, SCALE)
    _check(out, want, bound, "out")


def test_graph_replays_with_changing_lengths(dev):
    """One graph of a shared-prefix step and one of a bounded cache's append,
    scored attention and eviction, replayed with other lengths and eager work in
    between; two graphs that share a workspace; every replay as the eager call."""
    B, P, S_max = 6, 500, 70
    announce("graph replays")
    g = _gen(dev, 5)
    q = bf16_randn((B, HQ, D), g, dev, 2.0)
    kp, vp = bf16_randn((HKV, P, D), g, dev), bf16_randn((HKV, P, D), g, dev)
    k, v = bf16_randn((B, HKV, S_max, D), g, dev), bf16_randn((B, HKV, S_max, D), g, dev)
    ctx = _i32([1] * B, dev)
    out = torch.zeros(B, HQ * D, dtype=torch.bfloat16, device=dev)
    ws = ops.attn_shared_workspace(B, 1, HQ, HKV, D, P, S_max, dev)
    raw = torch.randn(B, (HQ + 2 * HKV) * D, generator=g, device=dev)
    ones = torch.ones(D, dtype=torch.bfloat16, device=dev)
    cos, sin = rope_tables(D, 400, 1e6, dev)
    pos, slots, ctx2 = _i32([50] * B, dev), _i32([60] * B, dev), _i32([61] * B, dev)
    sc, sp = torch.rand(B, HKV, S_max, generator=g, device=dev), torch.zeros(B, HKV, S_max, dtype=torch.int32, device=dev)
    sp.copy_(torch.arange(S_max, device=dev))
    out2 = torch.zeros_like(out)

    def first():
        ops.attn_shared(q, kp, vp, k, v, ctx, B, 1, workspace=ws, out=out)

    def other():  # the same workspace, another split of the work
        ops.attn_shared(q, kp, vp, k, v, ctx, B, 1, prefix_len=300, workspace=ws, out=out2)

    def second(k, v, sc, sp, o):
        qs = ops.kv_append(raw, ones, ones, cos, sin, pos, slots, HQ, HKV, k, v, 1e-6, scores=sc, slot_pos=sp)
        ops.attn_decode_scored(qs, k, v, ctx2, sc, out=o)
        ops.kv_evict(k, v, sc, sp, ctx2, 48, recent=4, sink=2)

    state, o3 = [k.clone(), v.clone(), sc.clone(), sp.clone()], torch.zeros_like(out)
    start = [t.clone() for t in state]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        first(), other(), second(*state, o3)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for f in (first, other, lambda: second(*state, o3)):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f()
        graphs.append(gr)
    for rep, (n, m) in enumerate([(1, 61), (70, 49), (13, 70), (0, 12), (64, 64)]):
        ctx.copy_(_i32([max(0, n - 3 * i) for i in range(B)], dev))
        ctx2.copy_(_i32([max(1, m - 2 * i) for i in range(B)], dev))
        slots.copy_(ctx2 - 1)
        pos.fill_(100 + rep)
        q.normal_(0.0, 2.0, generator=g)
        for t, x in zip(state, start):
            t.copy_(x)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        want = ops.attn_shared(q, kp, vp, k, v, ctx, B, 1)
        want2 = ops.attn_shared(q, kp, vp, k, v, ctx, B, 1, prefix_len=300)
        eager, o4 = [t.clone() for t in start], torch.zeros_like(out)
        second(*eager, o4)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(out2, want2) and torch.equal(o3, o4)
        for x, y in zip(state, eager):
            assert torch.equal(x, y)


def test_calls_on_another_stream(dev):
    """Calls take the current stream, whichever it is."""
    announce("another stream")
    g = _gen(dev, 6)
    q = bf16_randn((4, HQ, D), g, dev, 2.0)
    k, v = bf16_randn((4, HKV, 100, D), g, dev), bf16_randn((4, HKV, 100, D), g, dev)
    ctx = _i32([100, 3, 50, 64], dev)
    sc = torch.zeros(4, HKV, 100, device=dev)
    want = ops.attn_decode_scored(q, k, v, ctx, sc)
    torch.cuda.synchronize()
    s, late, sc2 = torch.cuda.Stream(), torch.empty_like(q), torch.zeros_like(sc)
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        late.copy_(q)  # ready only on this stream, after the wait
        got = ops.attn_decode_scored(late, k, v, ctx, sc2)
        shared = ops.attn_shared(late, k[0], v[0], k, v, ctx, 4, 1)
    s.synchronize()
    assert torch.equal(got, want) and torch.equal(sc, sc2)
    assert torch.equal(shared, ops.attn_shared(q, k[0], v[0], k, v, ctx, 4, 1))


# ------------------------------------------------------------------ the attention layer
def _attention(dev, seed):
    g = _gen(dev, seed)
    std = 0.03
    return Attention(bf16_randn(((HQ + 2 * HKV) * D, H), g, dev, std),
                     (1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16),
                     (1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16),
                     bf16_randn((H, HQ * D), g, dev, std), HQ, HKV, D, 1e-6), g


@pytest.mark.parametrize("B,P,S,steps", [(1, 40, 1, 2), (3, 100, 7, 3), (20, 65, 3, 2), (70, 33, 2, 2), (2, 130, 150, 2)])
def test_attention_layer_on_a_shared_prefix(dev, B, P, S, steps):
    """The layer with the prefix held once against the layer whose rows each hold
    it, on the same tokens.  Each side's outputs are sums over bf16 weights of
    probabilities and of attention outputs that were rounded to bf16: four
    roundings between the two, of 2^-9 on average."""
    announce(f"attention layer, prefix {P}, B={B} S={S}")
    at, g = _attention(dev, B + P)
    cos, sin = rope_tables(D, P + S + steps, 1e6, dev)
    x = bf16_randn((P, H), g, dev)
    pos = torch.arange(P, dtype=torch.int32, device=dev)
    pre = KVCache(1, HKV, P, D, dev)
    at.forward(x, torch.zeros(P, H, device=dev), pos, 1, P, pre, cos, sin)
    full, own = KVCache(B, HKV, P + S + steps, D, dev), KVCache(B, HKV, S + steps, D, dev)
    full.k[:, :, :P], full.v[:, :, :P] = pre.k, pre.v
    own.prefix = SharedPrefix(pre.k[0], pre.v[0], P)
    at0 = 0
    for n in [S] + [1] * steps:
        y = bf16_randn((B * n, H), g, dev)
        p = (at0 + torch.arange(n, dtype=torch.int32, device=dev)).repeat(B)
        a, b = torch.zeros(B * n, H, device=dev), torch.zeros(B * n, H, device=dev)
        at.forward(y, a, p + P, B, n, full, cos, sin, P + at0)
        at.forward(y, b, p, B, n, own, cos[P:], sin[P:], at0)
        torch.cuda.synchronize()
        rel = mean_rel(b, a)
        print(f"  {n} queries at {at0}: mean rel {rel:.2e}", flush=True)
        assert rel <= 4 * 2.0 ** -9
        at0 += n
    for a, b in ((full.k, own.k), (full.v, own.v)):
        a, b = a[:, :, P:P + at0].double(), b[:, :, :at0].double()
        if B <= FUSED_DECODE_MAX_ROWS:  # both sides project with the same kernels
            assert torch.equal(a, b)
        # else two orders of a 32-bit sum of 2048 products, each side rounded to bf16: off by two
        # half steps (2^-8 of the value each), and by 2048 * 2^-24 of the sum of the products'
        # magnitudes (2048 * E|x| E|w| = 2048 * 0.8 * 0.024 = 39)
        assert bool(((a - b).abs() <= 2 * ref.HALF_BF16 * a.abs() + 2048 * ref.F32 * 39).all())


def test_layer_contract_refuses_special_caches(dev):
    nc = qn.MoENeuronConfig(max_length=32)
    cfg = qn.Qwen3MoeInferenceConfig(nc)
    cfg.num_experts = 8
    layer = qm.NeuronQwen3MoeDecoderLayer(cfg, 0)
    x = torch.zeros(1, 2, cfg.hidden_size, device=dev)
    cache = KVCache(1, HKV, 40, D, dev)
    cache.prefix = SharedPrefix(cache.k[0], cache.v[0], 4)
    with pytest.raises(ValueError, match="driven by the model"):
        layer.forward(x, past_key_value=cache)
    layer.cache = BoundedKVCache(CacheBudget(1, 8, 2, 1, 4, dev), HKV, D)
    with pytest.raises(ValueError, match="driven by the model"):
        layer.forward(x)
    at, _ = _attention(dev, 1)
    cos, sin = rope_tables(D, 40, 1e6, dev)
    rows, res = torch.zeros(2, H, dtype=torch.bfloat16, device=dev), torch.zeros(2, H, device=dev)
    with pytest.raises(ValueError, match="first token"):
        at.forward(rows, res, _i32([3, 4], dev), 1, 2, layer.cache, cos, sin, 3)
    with pytest.raises(ValueError, match="device-held"):
        at.forward(rows, res, _i32([3, 4], dev), 1, 2, cache, cos, sin, _i32([3], dev))


# ------------------------------------------------------------------ the model
def _model(batch, max_length, **kw):
    """Two layers whose routers give every expert the same logit, so all tokens go
    to experts 0-7: a router's near tie would make one rounding a whole expert's
    difference."""
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


def _close(a, b, what):
    """Logits of two orders of the same sums: a few dozen roundings to bf16 (2^-9
    each on average) of the values on the way, whose errors add up as squares."""
    rel = float((a.double() - b.double()).norm() / b.double().norm())
    print(f"  {what}: relative difference {rel:.2e}", flush=True)
    assert rel <= 6 * 2.0 ** -8, what


def test_model_on_a_shared_prefix(dev):
    announce("model on a shared prefix")
    B, P = 3, 50
    m = _model(B, 100)
    prefix, prompts, lengths = _tokens(1, P), _tokens(2, B, 9), torch.tensor([9, 4, 1])
    whole = torch.cat([prefix.expand(B, P), prompts], 1)
    want = [m.prefill(whole, lengths + P)]
    steps = [_tokens(3 + i, B) for i in range(3)]
    want += [m.decode_step(t, lengths + P + i) for i, t in enumerate(steps)]
    m.share_prefix(prefix)
    got = [m.prefill(prompts, lengths)] + [m.decode_step(t, lengths + i) for i, t in enumerate(steps)]
    for i, (a, b) in enumerate(zip(got, want)):
        _close(a, b, f"step {i}")
    assert m.model.caches()[0].prefix.k.shape[1] == P
    ad = qn.HuggingFaceGenerationAdapter(m)
    mask = (torch.arange(9) < lengths[:, None]).long()
    graph = ad.generate(prompts, attention_mask=mask, max_new_tokens=20)
    m.neuron_config.use_hip_graphs = False
    eager = ad.generate(prompts, attention_mask=mask, max_new_tokens=20)
    assert graph.shape == (B, 29) and torch.equal(graph, eager)
    with pytest.raises(ValueError, match="exceed max_length"):
        ad.generate(prompts, max_new_tokens=43)
    with pytest.raises(ValueError, match="contiguous caches"):
        m.spec_generate(prompts[:1], 4)
    # another prefix, then none: the captured steps follow
    m.neuron_config.use_hip_graphs = True
    m.share_prefix(_tokens(9, 1, 20))
    other = ad.generate(prompts, max_new_tokens=8)
    m.drop_prefix()
    plain = ad.generate(torch.cat([_tokens(9, 20).expand(B, 20), prompts], 1), max_new_tokens=1)
    assert m.model.base == 0 and plain.shape == (B, 30)
    assert torch.equal(other[:, 9], plain[:, 29])
    with pytest.raises(ValueError, match="no position"):
        m.share_prefix(_tokens(1, 101))
    with pytest.raises(ValueError, match="prefix_ids"):
        m.share_prefix(_tokens(1, 2, 5))


def test_model_prefix_cut_down(dev):
    announce("model, prefix cut down")
    m = _model(2, 200)
    prefix, prompts = _tokens(1, 120), _tokens(2, 2, 6)
    m.share_prefix(prefix)
    want = m.prefill(prompts)
    full = m.model.caches()[1].prefix
    m.share_prefix(prefix, budget=120)
    assert torch.equal(m.prefill(prompts), want)
    m.share_prefix(prefix, budget=60, recent=10, sink=2)
    cut = m.model.caches()[1].prefix
    assert cut.length == 60 and m.model.base == 120
    for h in range(HKV):  # rows of the whole prefix, the first and last among them
        rows = (full.k[h, None, :] == cut.k[h, :60, None]).all(-1)
        assert bool(rows.any(1).all())
        kept = rows.any(0).nonzero()[:, 0].tolist()
        assert kept[:2] == [0, 1] and kept[-10:] == list(range(110, 120))
    out = qn.HuggingFaceGenerationAdapter(m).generate(prompts, max_new_tokens=5)
    assert out.shape == (2, 11)


@pytest.mark.parametrize("lengths", [[30, 30], [30, 11]])
def test_model_bounded_cache_that_holds_everything(dev, lengths):
    """A budget that nothing exceeds is the contiguous cache's generation."""
    announce(f"bounded caches without eviction, {lengths}")
    n = torch.tensor(lengths)
    prompts, steps = _tokens(1, 2, 30), [_tokens(2 + i, 2) for i in range(3)]
    a, b = _model(2, 64), _model(2, 64, kv_cache_budget=40, kv_cache_slack=24)
    want, got = [a.prefill(prompts, n)], [b.prefill(prompts, n)]
    for i, t in enumerate(steps):
        want.append(a.decode_step(t, n + i))
        got.append(b.decode_step(t, n + i))
    for i, (x, y) in enumerate(zip(got, want)):
        _close(x, y, f"step {i}")
    assert b.model.budget.used == [x + 3 for x in lengths]


def test_model_bounded_cache_evicts(dev):
    announce("bounded caches with eviction")
    prompts = _tokens(1, 2, 50)
    mask = (torch.arange(50) < torch.tensor([[50], [13]])).long()
    outs = []
    for graphs in (True, False):
        m = _model(2, 120, kv_cache_budget=24, kv_cache_recent=6, kv_cache_sink=2, kv_cache_slack=5,
                   use_hip_graphs=graphs)
        ad = qn.HuggingFaceGenerationAdapter(m)
        outs.append(ad.generate(prompts, attention_mask=mask, max_new_tokens=40))
        st, used = m.model.budget, m.model.budget.used
        assert st.slots.tolist() == used and st.ctx.tolist() == [x + 1 for x in used]
        assert max(used) <= 29 and m.model.caches()[0].capacity == 29
        last = [50 + 39 - 1, 13 + 39 - 1]
        for c in m.model.caches():
            for b in range(2):
                live = c.slot_pos[b, :, :used[b]]
                assert bool((live.max(1).values == last[b]).all())
                for h in range(HKV):
                    held = set(live[h].tolist())
                    assert len(held) == used[b] and {0, 1} <= held and set(range(last[b] - 5, last[b] + 1)) <= held
                # every step's attention has weight 1 a head, so the scores cannot exceed what was given
                assert float(c.scores[b].sum()) <= (last[b] + 1) * HQ * (1 + 1e-5)
                assert not bool(c.scores[b, :, used[b]:].any())
        outs.append(ad.generate(prompts, attention_mask=mask, max_new_tokens=40))  # the caches start over
        with pytest.raises(ValueError, match="kv_cache_budget"):
            m.share_prefix(_tokens(3, 5))
        with pytest.raises(ValueError, match="contiguous caches"):
            m.spec_generate(prompts[:1], 4)
    for o in outs[1:]:
        assert torch.equal(outs[0], o)


def test_model_bounded_cache_one_token_prompt(dev):
    announce("bounded caches, one token")
    a, b = _model(2, 40), _model(2, 40, kv_cache_budget=16, kv_cache_slack=3)
    one = _tokens(1, 2, 1)
    _close(b.prefill(one), a.prefill(one), "prompt")
    t = _tokens(2, 2)
    _close(b.decode_step(t), a.decode_step(t), "step")
    assert b.model.budget.used == [2, 2] and b.model.caches()[0].slot_pos[:, :, :2].tolist() == [[[0, 1]] * HKV] * 2
    with pytest.raises(ValueError, match="hold 2 rows"):
        b.prefill(_tokens(1, 3, 4))


def test_model_prefix_refused_changes_nothing(dev):
    """Sizes that do not fit leave the old prefix as it was; tokens outside the
    vocabulary leave none; the smallest budgets work with the default split."""
    announce("refused prefixes")
    m = _model(2, 60)
    prefix, prompts = _tokens(1, 20), _tokens(2, 2, 6)
    m.share_prefix(prefix)
    want = m.prefill(prompts)
    for bad in (dict(budget=-3), dict(budget=10, recent=-1), dict(budget=10, recent=8, sink=3),
                dict(budget=30, recent=28, sink=3)):
        with pytest.raises(ValueError, match="recent \\+ sink"):
            m.share_prefix(_tokens(3, 20), **bad)
    with pytest.raises(ValueError, match="no position"):
        m.share_prefix(_tokens(3, 61))
    assert m.model.base == 20 and torch.equal(m.prefill(prompts), want)
    for budget in (1, 4, 5):
        m.share_prefix(prefix, budget=budget)
        assert m.model.caches()[0].prefix.length == budget
    m.drop_prefix()
    plain = m.prefill(prompts)
    m.share_prefix(prefix)
    with pytest.raises(ValueError, match="token id"):
        m.share_prefix(torch.full((8,), 5000))
    assert m.model.base == 0 and torch.equal(m.prefill(prompts), plain)


def test_model_bounded_cache_starts_over(dev):
    """Steps after reset() see nothing of the sequence before, and another number
    of rows is refused before anything changes, for eager and captured steps."""
    announce("bounded caches start over")
    m = _model(2, 40, kv_cache_budget=16, kv_cache_slack=3)
    a, b = _tokens(1, 2), _tokens(2, 2)
    first = [m.decode_step(a), m.decode_step(b)]
    m.prefill(_tokens(3, 2, 12))
    m.decode_step(a)
    m.reset()
    assert m.model.budget.used == [0, 0]
    assert torch.equal(m.decode_step(a), first[0]) and torch.equal(m.decode_step(b), first[1])
    for call in (lambda: m.decode_step(_tokens(4, 3)), lambda: m.greedy_decode(_tokens(4, 3), 2),
                 lambda: m.greedy_decode(_tokens(4, 1), 2, use_graph=False)):
        with pytest.raises(ValueError, match="hold 2 rows"):
            call()
    st = m.model.budget
    assert st.used == [2, 2] and st.slots.tolist() == [2, 2] and st.ctx.tolist() == [3, 3] and m.position == 2


@pytest.mark.parametrize("P", [1, 2, 17])
def test_model_on_a_short_prefix(dev, P):
    """A prefix of one token runs as a decode step, of two as a chunk, and prompts of
    one token continue it as steps."""
    announce(f"model on a prefix of {P}")
    m = _model(2, 40)
    prefix, steps = _tokens(1, P), [_tokens(3 + i, 2) for i in range(3)]
    want = [m.prefill(torch.cat([prefix.expand(2, P), steps[0][:, None]], 1))]
    want += [m.decode_step(t) for t in steps[1:]]
    m.share_prefix(prefix)
    got = [m.prefill(steps[0][:, None])] + [m.decode_step(t) for t in steps[1:]]
    for i, (a, b) in enumerate(zip(got, want)):
        _close(a, b, f"step {i}")
    assert m.position == 3
