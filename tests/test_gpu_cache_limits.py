"""The model and its layers on shared prefixes and bounded caches at their limits:
prompts and steps past the last position, captured steps, operands off the
alignment; and the operators' arguments that need none."""

import pytest
import torch

from gpu_util import announce, bf16_randn, mean_rel
from qmoe import model as qm
from qmoe import ops
from qmoe.attention import Attention, BoundedKVCache, CacheBudget, KVCache, SharedPrefix, rope_tables

import qwen_with_nki as qn

pytestmark = pytest.mark.gpu

HQ, HKV, D, H = 32, 4, 128, 2048


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


def _off(t, offset):
    """A copy of ``t`` that starts ``offset`` bytes past a 16-byte boundary."""
    buf = torch.empty(t.numel() + 8, dtype=t.dtype, device=t.device)
    first = offset // t.element_size()
    out = buf[first:first + t.numel()].view(t.shape)
    assert out.data_ptr() % 16 == offset
    return out.copy_(t)


@pytest.mark.parametrize("w_off,x_off", [(8, 0), (0, 4), (12, 2)])
@pytest.mark.parametrize("B", [17, 70])
def test_steps_off_the_alignment(dev, B, w_off, x_off):
    """A step whose operands are off the alignment: on bounded caches the bits of
    the aligned step (the same products on copies); on a shared prefix close to
    the layer whose rows hold the prefix themselves and off the alignment
    too, whose entries come from the same kernel."""
    announce(f"steps off the alignment, B={B} {w_off} {x_off}")
    g = torch.Generator(device=dev).manual_seed(B)
    w, wo = bf16_randn(((HQ + 2 * HKV) * D, H), g, dev, 0.03), bf16_randn((H, HQ * D), g, dev, 0.03)
    nw = torch.ones(D, dtype=torch.bfloat16, device=dev)
    x, P = bf16_randn((B, H), g, dev), 40
    cos, sin = rope_tables(D, P + 4, 1e6, dev)
    at, off = [Attention(t, nw, nw, wo, HQ, HKV, D, 1e-6) for t in (w, _off(w, w_off))]
    pos = torch.arange(B, dtype=torch.int32, device=dev) % 4
    outs = []
    for a, y in ((at, x), (off, _off(x, x_off))):
        state = CacheBudget(B, 8, 2, 1, 3, dev)
        state.slots.copy_(pos)
        state.ctx.copy_(pos + 1)
        cache, res = BoundedKVCache(state, HKV, D), torch.zeros(B, H, device=dev)
        a.forward(y, res, pos, B, 1, cache, cos, sin)
        outs.append((res, cache.k, cache.v, cache.scores, cache.slot_pos))
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    pre = bf16_randn((2, HKV, P, D), g, dev)
    full, own = KVCache(B, HKV, P + 4, D, dev), KVCache(B, HKV, 4, D, dev)
    for t, e in ((full.k, pre[0]), (full.v, pre[1])):
        t.normal_(generator=g)
        t[:, :, :P] = e
    own.k.copy_(full.k[:, :, P:])
    own.v.copy_(full.v[:, :, P:])
    own.prefix = SharedPrefix(pre[0], pre[1], P)
    a, b = torch.zeros(B, H, device=dev), torch.zeros(B, H, device=dev)
    off.forward(_off(x, x_off), a, pos + P, B, 1, full, cos, sin)
    off.forward(_off(x, x_off), b, pos, B, 1, own, cos[P:], sin[P:])
    rel = mean_rel(b, a)
    print(f"  mean rel {rel:.2e}", flush=True)
    # two roundings to bf16 on either side of the attention (its weights, its output)
    assert rel <= 4 * 2.0 ** -9
    assert torch.equal(own.k, full.k[:, :, P:]) and torch.equal(own.v, full.v[:, :, P:])


@pytest.mark.parametrize("B,h,heads", [(3, 576, 40), (16, 64, 8), (9, 4096, 2049)])
def test_raw_projection_of_any_operands(dev, B, h, heads):
    """Hidden sizes that the GEMV does not take, and 2 GiB of weights, in the raw
    projection of a bounded cache's step.  Bound: a sum of h products in 32 bits."""
    announce(f"raw projection, B={B} h={h} heads={heads}")
    g = torch.Generator(device=dev).manual_seed(h)
    w, x = bf16_randn((heads * D, h), g, dev, 0.1), bf16_randn((B, h), g, dev)
    a = Attention(w, None, None, None, heads - 2, 1, D, 1e-6)
    got = a._raw_of_any(x)
    assert got.shape == (B, heads * D) and got.is_contiguous()
    for c in {0, heads * D // 2 - 256, heads * D // 2, heads * D - 512}:  # (the middle: where the pieces meet)
        c = max(0, c)
        part = w[c:c + 512].double()
        want, size = x.double() @ part.t(), x.double().abs() @ part.abs().t()
        assert bool(((got[:, c:c + 512].double() - want).abs() <= h * 2.0 ** -24 * size).all())


def test_captured_and_eager_steps_give_the_same_bits(dev):
    """Caches of more slots than the first context bucket, which the rows do not
    leave at first: entries, scores and positions after eager steps are those
    after captured ones, and so is what an eviction keeps."""
    announce("captured and eager steps, caches past a bucket")
    prompts, runs = _tokens(1, 16, 200), []
    for graphs in (True, False):
        m = _model(16, 700, kv_cache_budget=560, kv_cache_slack=40, use_hip_graphs=graphs)
        first, stages = m.prefill(prompts).argmax(-1), []
        for n in (30, 60, 320):  # in the buckets of 256 and 512, then past an eviction
            first = m.greedy_decode(first, n)[:, -1]
            stages += [first.clone(), *_cache_bits(m)]
        runs.append(stages)
    assert m.model.caches()[0].capacity == 600
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a, b), i
    runs = []
    for graphs in (True, False):
        m = _model(5, 700, use_hip_graphs=graphs)
        m.share_prefix(_tokens(2, 100))
        first = m.prefill(_tokens(3, 5, 230)).argmax(-1)
        toks = m.greedy_decode(first, 60)
        runs.append([toks] + [t[:, :, :290].clone() for c in m.model.caches() for t in (c.k, c.v)])
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a, b), i


def test_arguments_that_need_no_alignment(dev):
    """Lengths, positions, slots, scores and tables are read in single words, and
    kv_append's rows too: a slice of a batch's lengths is as good as its start."""
    announce("arguments off 16 bytes")
    g = torch.Generator(device=dev).manual_seed(8)
    B, S_max, cap = 3, 70, 5

    def i32(*values):
        return torch.tensor(values, dtype=torch.int32, device=dev)

    def off(t):  # one element behind a boundary
        return _off(t, t.element_size())

    q, k, v = [bf16_randn(s, g, dev) for s in ((B, HQ, D), (B, HKV, S_max, D), (B, HKV, S_max, D))]
    lens, many = i32(70, 3, 66), i32(9, 70, 3, 66)
    assert many[1:].data_ptr() % 16
    want = ops.attn_shared(q, k[0], v[0], k, v, lens, B, 1)
    assert torch.equal(want, ops.attn_shared(q, k[0], v[0], k, v, many[1:], B, 1))
    scores = torch.rand(B, HKV, S_max, generator=g, device=dev)
    runs = []
    for n, sc in ((lens, scores.clone()), (many[1:], off(scores))):
        out = ops.attn_decode_scored(q, k, v, n, sc)
        runs.append([out, ops.attn_prefill_scored(q, k, v, sc, B, 1, 5, lengths=off(i32(1, 0, 1))), sc])
    raw = torch.randn(B, (HQ + 2 * HKV) * D, generator=g, device=dev)
    w, (cos, sin) = bf16_randn((2, D), g, dev), rope_tables(D, 50, 1e6, dev)
    k2, v2 = bf16_randn((B, HKV, cap, D), g, dev), bf16_randn((B, HKV, cap, D), g, dev)
    pos, slots, at = i32(7, 49, 0), i32(4, 0, 2), torch.arange(S_max, dtype=torch.int32, device=dev).repeat(B, HKV, 1)
    for same in (torch.clone, off):
        cache = [same(t) for t in (k2, v2, scores[:, :, :cap].contiguous(), at[:, :, :cap].contiguous())]
        got = ops.kv_append(same(raw), same(w[0]), same(w[1]), same(cos), same(sin), same(pos), same(slots), HQ, HKV,
                            cache[0], cache[1], 1e-6, scores=cache[2], slot_pos=cache[3], q_out=same(q))
        full = [k.clone(), v.clone(), same(scores), same(at)]
        ops.kv_evict(*full, same(lens), 40, 5, 2,
                     workspace=same(torch.zeros(2 * B * HKV * 40, dtype=torch.int32, device=dev)))
        runs[same is off] += [got, *cache, *full]
    for i, (a, b) in enumerate(zip(*runs)):
        assert torch.equal(a, b), i
    for bad in (dict(k=off(k)), dict(out=off(want)), dict(q=off(q))):  # and what does need it is still refused
        args = dict(q=q, k=k, v=v, out=None)
        args.update(bad)
        with pytest.raises(ValueError, match="16-byte aligned"):
            ops.attn_decode_scored(args["q"], args["k"], args["v"], lens, scores, out=args["out"])


def test_scored_prompt_refuses_its_queries_as_output(dev):
    announce("scored prompt onto its queries")
    g = torch.Generator(device=dev).manual_seed(9)
    q, k, v = [bf16_randn(s, g, dev) for s in ((30, HQ, D), (1, HKV, 30, D), (1, HKV, 30, D))]
    scores, q0 = torch.zeros(1, HKV, 30, device=dev), q.clone()
    with pytest.raises(ValueError, match="out overlaps q"):
        ops.attn_prefill_scored(q, k, v, scores, 1, 30, out=q.view(30, HQ * D))
    assert torch.equal(q, q0) and not bool(scores.any())
    # the other two read their queries first: out may be q
    want = ops.attn_shared(q, k[0], v[0], k, v, torch.ones(1, dtype=torch.int32, device=dev), 1, 30)
    mine = q.clone()
    ops.attn_shared(mine, k[0], v[0], k, v, torch.ones(1, dtype=torch.int32, device=dev), 1, 30,
                    out=mine.view(30, HQ * D))
    assert torch.equal(mine.view(30, HQ * D), want)


@pytest.mark.parametrize("n,budget,recent,sink", [(9, 3, 1, 2), (313, 6, 0, 6), (881, 84, 37, 4), (20_000, 90, 40, 9)])
def test_eviction_with_more_protected_entries_than_the_budget(dev, n, budget, recent, sink):
    """Positions that repeat: more entries are protected than stay.  They rank alike
    whatever their scores, NaN among them, so the lowest slots stay."""
    announce(f"eviction, {n} entries to {budget}, positions that repeat")
    g = torch.Generator(device=dev).manual_seed(n)
    k, v = [bf16_randn((1, 2, n, D), g, dev) for _ in range(2)]
    sc = torch.randn(1, 2, n, generator=g, device=dev)
    sc[torch.rand(1, 2, n, generator=g, device=dev) < 0.2] = float("nan")
    pos = (torch.rand(1, 2, n, generator=g, device=dev).argsort(-1) // 3).int().contiguous()
    k0, pos0 = k.clone(), pos.clone()
    ops.kv_evict(k, v, sc, pos, torch.tensor([n], dtype=torch.int32, device=dev), budget, recent, sink)
    for h in range(2):
        held = ((pos0[0, h] < sink) | (pos0[0, h] > pos0[0, h].max() - recent)).nonzero()[:, 0]
        assert len(held) > budget
        keep = held[:budget]
        stay, order = keep[keep < budget], torch.arange(budget, device=dev)
        hole = torch.ones(budget, dtype=torch.bool, device=dev)
        hole[stay] = False
        order[hole] = keep[keep >= budget]
        assert torch.equal(pos[0, h, :budget], pos0[0, h, order]) and torch.equal(k[0, h, :budget], k0[0, h, order])
        assert bool((pos[0, h, budget:] == -1).all())
