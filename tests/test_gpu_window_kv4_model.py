"""Windowed attention and caches in 4 bits as the package uses them: a batch's prompt,
steps and chunks together, captured into graphs, on other streams, in the attention
layer and in the model's generation."""

import math

import pytest
import torch

import kv4_ref as ref
from gpu_util import announce, bf16_randn, mean_rel
from qmoe import model as qm
from qmoe import ops
from qmoe.attention import Attention, KV4Cache, KVCache, rope_tables
from test_gpu_cache_model import _close, _model, _tokens

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


def _held(cache):
    return ref.values(*cache[:2]), ref.values(*cache[2:])


# ------------------------------------------------------------------ operators together
@pytest.mark.parametrize("window,sink", [(0, 0), (24, 3)])
def test_prompt_steps_and_chunks_together(dev, window, sink):
    """A padded batch's prompt attended in bf16 and stored in 4 bits, steps, then a
    chunk; every result against 64 bits from the cache as the kernels left it."""
    B, S, lengths, cap = 3, 70, [70, 33, 51], 100
    announce(f"prompt, steps, chunk; window {window}")
    g = _gen(dev, 3)
    q = bf16_randn((B * S, HQ, D), g, dev, 2.0)
    k, v = bf16_randn((B, HKV, S, D), g, dev), bf16_randn((B, HKV, S, D), g, dev)
    ones = _i32([1] * B, dev)
    if window:
        out = ops.attn_window(q, k, v, ones, B, S, window, sink)
        _check(out, *ref.window(q, k, v, [1] * B, B, S, window, sink, S, SCALE), "prompt")
    cache = ops.kv4_cache(B, HKV, cap, D, dev)
    ops.kv4_store(k, v, cache, lengths=_i32(lengths, dev))
    for b, n in enumerate(lengths):
        for i, x in ((0, k), (2, v)):
            codes, powers = ref.quantise(x[b, :, :n])
            assert torch.equal(cache[i][b, :, :n], codes) and not bool(cache[i][b, :, n:].any())
            assert torch.equal(cache[i + 1][b, :, :n], powers) and not bool(cache[i + 1][b, :, n:].any())
    cos, sin = rope_tables(D, 400, 1e6, dev)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    at = list(lengths)
    for n in [1] * 9 + [11]:
        raw = torch.randn(B * n, (HQ + 2 * HKV) * D, generator=g, device=dev) * 2
        pos = _i32([p + i for p in at for i in range(n)], dev)
        before = [t.clone() for t in cache]
        qs = ops.kv4_append(raw, w, w, cos, sin, pos, pos, HQ, HKV, cache, 1e-6, S=n)
        kn, vn = ref.append(raw, w, w, cos, sin, pos, HQ, HKV, 1e-6)
        for i, x in ((0, kn), (2, vn)):
            codes, powers = ref.quantise(x.view(B, n, HKV, D).transpose(1, 2))
            for b, p in enumerate(at):
                before[i][b, :, p:p + n], before[i + 1][b, :, p:p + n] = codes[b], powers[b]
        assert all(torch.equal(a, b) for a, b in zip(cache, before))
        ctx = [p + 1 for p in at]
        out = ops.attn_kv4(qs, cache, _i32(ctx, dev), B, n, window, sink)
        _check(out, *ref.window(qs, *_held(cache), ctx, B, n, window, sink, cap, SCALE), f"{n} queries at {at}")
        at = [p + n for p in at]
    kb, vb = ops.kv4_load(cache)
    want = _held(cache)
    assert torch.equal(kb.double(), want[0]) and torch.equal(vb.double(), want[1])


def test_graph_replays_with_changing_lengths(dev):
    """A graph of a windowed step, two of 4-bit steps that share a workspace and one of
    an append with its attention, replayed with other lengths and eager work in
    between; every replay as the eager call."""
    B, S_max = 6, 2000
    announce("graph replays")
    g = _gen(dev, 5)
    q = bf16_randn((B, HQ, D), g, dev, 2.0)
    k, v = bf16_randn((B, HKV, S_max, D), g, dev), bf16_randn((B, HKV, S_max, D), g, dev)
    cache = ops.kv4_cache(B, HKV, S_max, D, dev)
    ops.kv4_store(k, v, cache)
    ctx = _i32([1] * B, dev)
    outs = [torch.zeros(B, HQ * D, dtype=torch.bfloat16, device=dev) for _ in range(4)]
    raw = torch.randn(B, (HQ + 2 * HKV) * D, generator=g, device=dev)
    ones = torch.ones(D, dtype=torch.bfloat16, device=dev)
    cos, sin = rope_tables(D, S_max, 1e6, dev)
    slots = _i32([7] * B, dev)
    ws = ops.attn_kv4_workspace(B, 1, HQ, HKV, D, 0, 0, S_max, dev)
    wws = ops.attn_window_workspace(B, 1, HQ, HKV, D, 700, 4, S_max, dev)

    def calls(cache, outs, ws, wws):
        def window():
            ops.attn_window(q, k, v, ctx, B, 1, 700, 4, workspace=wws, out=outs[0])

        def four():
            ops.attn_kv4(q, cache, ctx, B, 1, workspace=ws, out=outs[1])

        def four_windowed():  # the same workspace, another split of the work
            ops.attn_kv4(q, cache, ctx, B, 1, 400, 4, workspace=ws, out=outs[2])

        def append():
            qs = ops.kv4_append(raw, ones, ones, cos, sin, slots, slots, HQ, HKV, cache, 1e-6)
            ops.attn_kv4(qs, cache, ctx, B, 1, out=outs[3])
        return window, four, four_windowed, append

    mine = calls(cache, outs, ws, wws)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for f in mine:
            f()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graphs = []
    for f in mine:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            f()
        graphs.append(gr)
    start = [t.clone() for t in cache]
    eager_outs = [torch.zeros_like(o) for o in outs]
    for rep, n in enumerate([1, 2000, 513, 0, 64, 1999]):
        ctx.copy_(_i32([max(0, n - 131 * i) for i in range(B)], dev))
        slots.copy_((ctx - 1).clamp_min(0))
        q.normal_(0.0, 2.0, generator=g)
        for t, x in zip(cache, start):
            t.copy_(x)
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        eager = tuple(t.clone() for t in start)
        for f in calls(eager, eager_outs, None, None):
            f()
        torch.cuda.synchronize()
        for a, b in zip(outs, eager_outs):
            assert torch.equal(a, b), rep
        assert all(torch.equal(a, b) for a, b in zip(cache, eager))


def test_graph_replays_of_long_batches_and_chunks(dev):
    """A step of a long batch, whose keys go in even shares, and chunks on tiles with
    and without a window: captured once, replayed with other lengths and eager work
    between, every replay as the eager call."""
    B, S_max, S = 40, 12000, 40
    announce("graph replays, long batches and chunks")
    g = _gen(dev, 9)
    k, v = bf16_randn((B, HKV, S_max, D), g, dev), bf16_randn((B, HKV, S_max, D), g, dev)
    cache = ops.kv4_cache(B, HKV, S_max, D, dev)
    ops.kv4_store(k, v, cache)
    q = bf16_randn((B * S, HQ, D), g, dev, 2.0)
    ctx = _i32([1] * B, dev)
    outs = [torch.zeros(n, HQ * D, dtype=torch.bfloat16, device=dev) for n in (B, B * S, B * S)]

    def calls(outs):
        ops.attn_kv4(q[:B], cache, ctx, B, 1, out=outs[0])
        ops.attn_kv4(q, cache, ctx, B, S, 1500, 4, out=outs[1])
        ops.attn_window(q, k, v, ctx, B, S, 700, 4, out=outs[2])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        calls(outs)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(outs)
    eager = [torch.zeros_like(o) for o in outs]
    for rep, n in enumerate([12000, 1, 5000, 0, 11999]):
        ctx.copy_(_i32([max(-S, n - 290 * i) for i in range(B)], dev))
        q.normal_(0.0, 2.0, generator=g)
        graph.replay()
        torch.cuda.synchronize()
        calls(eager)
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), rep
            assert not bool(torch.isnan(a).any())


def test_calls_on_another_stream(dev):
    """Calls take the current stream, whichever it is."""
    announce("another stream")
    g = _gen(dev, 6)
    q = bf16_randn((4, HQ, D), g, dev, 2.0)
    k, v = bf16_randn((4, HKV, 900, D), g, dev), bf16_randn((4, HKV, 900, D), g, dev)
    ctx = _i32([900, 3, 500, 64], dev)
    cache, cache2 = ops.kv4_cache(4, HKV, 900, D, dev), ops.kv4_cache(4, HKV, 900, D, dev)
    ops.kv4_store(k, v, cache)
    want = [ops.attn_window(q, k, v, ctx, 4, 1, 100, 4), ops.attn_kv4(q, cache, ctx, 4, 1), *ops.kv4_load(cache)]
    torch.cuda.synchronize()
    s, late = torch.cuda.Stream(), torch.empty_like(k)
    with torch.cuda.stream(s):
        torch.cuda._sleep(2_000_000)
        late.copy_(k)  # ready only on this stream, after the wait
        ops.kv4_store(late, v, cache2)
        got = [ops.attn_window(q, late, v, ctx, 4, 1, 100, 4), ops.attn_kv4(q, cache2, ctx, 4, 1), *ops.kv4_load(cache2)]
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_two_calls_at_once(dev):
    """Calls on two streams, each with workspaces of its own."""
    announce("two streams at once")
    g = _gen(dev, 7)
    q = bf16_randn((8, HQ, D), g, dev, 2.0)
    k, v = bf16_randn((8, HKV, 3000, D), g, dev), bf16_randn((8, HKV, 3000, D), g, dev)
    cache = ops.kv4_cache(8, HKV, 3000, D, dev)
    ops.kv4_store(k, v, cache)
    ctx = _i32([3000 - 300 * i for i in range(8)], dev)
    want = ops.attn_window(q, k, v, ctx, 8, 1, 1500, 4), ops.attn_kv4(q, cache, ctx, 8, 1)
    torch.cuda.synchronize()
    a, b, got = torch.cuda.Stream(), torch.cuda.Stream(), []
    for _ in range(10):
        for st in (a, b):
            with torch.cuda.stream(st):
                got.append((ops.attn_window(q, k, v, ctx, 8, 1, 1500, 4), ops.attn_kv4(q, cache, ctx, 8, 1)))
    torch.cuda.synchronize()
    for x in got:
        assert torch.equal(x[0], want[0]) and torch.equal(x[1], want[1])


def test_offsets_past_32_bits(dev):
    """The last row of caches of 2^32 elements and more (bf16) and bytes (4 bits)."""
    announce("offsets past 32 bits")
    g = _gen(dev, 8)
    n = 1 << 22
    for B, S, window in ((9, 1, 300), (9, 40, 300)):
        k = torch.zeros(B, 1, n, D, dtype=torch.bfloat16, device=dev)
        v = torch.zeros_like(k)
        for t in (k, v):
            t[-1, 0, -700:] = bf16_randn((700, D), g, dev)
            t[-1, 0, :8] = bf16_randn((8, D), g, dev)
        q = bf16_randn((B * S, 8, D), g, dev, 2.0)
        ctx = _i32([1] * (B - 1) + [n - S + 1], dev)
        got = ops.attn_window(q, k, v, ctx, B, S, window, 8)[-S:]
        keep = torch.cat([torch.arange(8, device=dev), torch.arange(n - 700, n, device=dev)])
        small = k[-1:, :, keep], v[-1:, :, keep]
        del k, v
        want, bound = ref.window(q[-S:], *small, [708 - S + 1], 1, S, window, 8, 708, SCALE)
        _check(got, want, bound, f"bf16, {S} queries")
    B = 20
    cache = ops.kv4_cache(B, 1, n, D, dev)  # 5.4 GB of codes each
    rows = bf16_randn((1, 1, 700, D), g, dev), bf16_randn((1, 1, 700, D), g, dev)
    src = [torch.zeros(B, 1, 700, D, dtype=torch.bfloat16, device=dev) for _ in rows]
    for t, r in zip(src, rows):
        t[-1] = r[0]
    ops.kv4_store(*src, cache, starts=_i32([0] * (B - 1) + [n - 700], dev))
    for S in (1, 40):
        q = bf16_randn((B * S, 8, D), g, dev, 2.0)
        ctx = _i32([1] * (B - 1) + [n - S + 1], dev)
        got = ops.attn_kv4(q, cache, ctx, B, S, 300, 0)[-S:]
        held = [ref.values(*ref.quantise(r)) for r in rows]
        want, bound = ref.window(q[-S:], *held, [700 - S + 1], 1, S, 300, 0, 700, SCALE)
        _check(got, want, bound, f"4 bits, {S} queries")
    cos, sin = rope_tables(D, 10, 1e6, dev)
    raw = torch.randn(B, 10 * D, generator=g, device=dev)
    w = torch.ones(D, dtype=torch.bfloat16, device=dev)
    pos = _i32([9] * B, dev)
    ops.kv4_append(raw, w, w, cos, sin, pos, _i32([n - 1] * B, dev), 8, 1, cache, 1e-6)
    kn, vn = ref.append(raw, w, w, cos, sin, pos, 8, 1, 1e-6)
    for i, x in ((0, kn), (2, vn)):
        codes, powers = ref.quantise(x)
        assert torch.equal(cache[i][:, :, n - 1], codes) and torch.equal(cache[i + 1][:, :, n - 1], powers)
    last = tuple(t[-1:] for t in cache)
    kl, vl = ops.kv4_load(last)
    assert torch.equal(kl[0, 0, -700:-1].double(), ref.values(*ref.quantise(rows[0]))[0, 0, :-1])
    assert torch.equal(vl[0, 0, -1].double(), ref.values(*ref.quantise(vn))[-1, 0])


# ------------------------------------------------------------------ the attention layer
def _attention(dev, seed, window, sink):
    g = _gen(dev, seed)
    std = 0.03
    return Attention(bf16_randn(((HQ + 2 * HKV) * D, H), g, dev, std),
                     (1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16),
                     (1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16),
                     bf16_randn((H, HQ * D), g, dev, std), HQ, HKV, D, 1e-6, window, sink), g


@pytest.mark.parametrize("B,S,chunk,window,sink,four", [
    (1, 40, 1, 16, 2, False), (1, 40, 5, 16, 2, True), (3, 100, 3, 30, 4, False), (3, 100, 9, 0, 0, True),
    (20, 30, 2, 12, 1, True), (70, 21, 1, 9, 3, False), (70, 21, 1, 0, 0, True), (2, 150, 40, 64, 4, True)])
def test_attention_layer(dev, B, S, chunk, window, sink, four):
    """The layer's prompt, steps and chunks, at host- and device-held starts, against
    its own queries attended in 64 bits to the cache as it left it.  The outputs
    then pass three roundings to bf16 that the reference has not: weights, attention
    outputs, and in the o_proj none; 2^-9 each on average."""
    announce(f"attention layer B={B} S={S} window={window} four={four}")
    at, g = _attention(dev, B + S, window, sink)
    n = S + chunk + 3
    cos, sin = rope_tables(D, n, 1e6, dev)
    cache = KV4Cache(B, HKV, n, D, dev) if four else KVCache(B, HKV, n, D, dev)
    first = 0
    for count, device_start in ((S, False), (1, False), (1, False), (chunk, chunk > 1), (1, False)):
        x = bf16_randn((B * count, H), g, dev)
        pos = (first + torch.arange(count, dtype=torch.int32, device=dev)).repeat(B)
        res = torch.zeros(B * count, H, device=dev)
        start = _i32([first], dev) if device_start else first
        at.forward(x, res, pos, B, count, cache, cos, sin, start)
        own = KVCache(B, HKV, n, D, dev)
        q = ops.qkv_norm_rope(x, at.wqkv, at.q_norm, at.k_norm, cos, sin, pos, B, count, HQ, HKV, own.k, own.v, 1e-6)
        k, v = cache
        if four and first == 0:
            k, v = own.k, own.v  # a prompt attends what it has just computed
        want, _ = ref.window(q.view(B * count, HQ, D), k, v, [first + 1] * B, B, count, window, sink, n, SCALE)
        want = want @ at.wo.double().t()
        torch.cuda.synchronize()
        rel = mean_rel(res, want)
        print(f"  {count} queries at {first}: mean rel {rel:.2e}", flush=True)
        assert rel <= 4 * 2.0 ** -9
        first += count


def test_a_window_that_hides_nothing_takes_the_plain_path(dev):
    """Up to the window's length a layer's outputs are those without one, bit for bit;
    past it they differ."""
    plain, g = _attention(dev, 3, 0, 0)
    at = Attention(plain.wqkv, plain.q_norm, plain.k_norm, plain.wo, HQ, HKV, D, 1e-6, 40, 0)
    cos, sin = rope_tables(D, 100, 1e6, dev)
    a, b = KVCache(2, HKV, 100, D, dev), KVCache(2, HKV, 100, D, dev)
    first = 0
    for n, bucket, same in ((38, None, True), (1, 40, True), (1, 40, True), (1, 64, False), (20, None, False)):
        x = bf16_randn((2 * n, H), g, dev)
        pos = (first + torch.arange(n, dtype=torch.int32, device=dev)).repeat(2)
        out = [torch.zeros(2 * n, H, device=dev) for _ in range(2)]
        for layer, cache, res in ((plain, a, out[0]), (at, b, out[1])):
            layer.forward(x, res, pos, 2, n, cache, cos, sin, first, max_ctx=bucket)
        assert torch.equal(*out) == same
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
        first += n


def test_a_layer_with_a_window_refuses_special_caches(dev):
    from qmoe.attention import BoundedKVCache, CacheBudget, SharedPrefix

    at, _ = _attention(dev, 1, 16, 0)
    cos, sin = rope_tables(D, 40, 1e6, dev)
    rows, res = torch.zeros(2, H, dtype=torch.bfloat16, device=dev), torch.zeros(2, H, device=dev)
    cache = KVCache(1, HKV, 40, D, dev)
    cache.prefix = SharedPrefix(cache.k[0], cache.v[0], 4)
    for c in (cache, BoundedKVCache(CacheBudget(1, 8, 2, 1, 4, dev), HKV, D)):
        with pytest.raises(ValueError, match="no window"):
            at.forward(rows, res, _i32([0, 1], dev), 1, 2, c, cos, sin)


def test_layer_contract_with_a_window_and_four_bits(dev):
    """The reference's layer call: its own cache is made in the config's bits and
    unpacks as (K, V)."""
    nc = qn.MoENeuronConfig(max_length=64, kv_cache_bits=4, attention_window=20, attention_sink=2)
    cfg = qn.Qwen3MoeInferenceConfig(nc)
    layer = qm.NeuronQwen3MoeDecoderLayer(cfg, 0)
    g = _gen(dev, 2)
    x = bf16_randn((2, 30, cfg.hidden_size), g, dev)
    out, present, *_ = layer.forward(x)
    assert out.shape == x.shape and isinstance(present, KV4Cache) and present.capacity == 65
    k, v = present
    assert k.shape == (2, HKV, 65, D) and k.dtype == torch.bfloat16 and torch.equal(present[1], v)
    assert bool(k[:, :, :30].any()) and not bool(k[:, :, 30:].any())
    for n, at in ((1, 30), (4, 31)):
        y = bf16_randn((2, n, cfg.hidden_size), g, dev)
        pos = torch.arange(at, at + n).expand(2, n)
        out, again, *_ = layer.forward(y, position_ids=pos, past_key_value=present)
        assert again is present and bool(torch.isfinite(out).all())
        assert bool(present[0][:, :, at + n - 1].any())


# ------------------------------------------------------------------ the model
OPTIONS = [dict(attention_window=24, attention_sink=3), dict(attention_window=260), dict(kv_cache_bits=4),
           dict(kv_cache_bits=4, attention_window=24, attention_sink=3)]


@pytest.mark.parametrize("kw", OPTIONS, ids=str)
def test_model_generates(dev, kw):
    announce(f"model {kw}")
    B = 3
    m = _model(B, 400, **kw)
    prompts, lengths = _tokens(2, B, 40), torch.tensor([40, 4, 29])
    ad = qn.HuggingFaceGenerationAdapter(m)
    mask = (torch.arange(40) < lengths[:, None]).long()
    graph = ad.generate(prompts, attention_mask=mask, max_new_tokens=230)  # two buckets
    again = ad.generate(prompts, attention_mask=mask, max_new_tokens=230)
    m.neuron_config.use_hip_graphs = False
    eager = ad.generate(prompts, attention_mask=mask, max_new_tokens=230)
    assert graph.shape == (B, 270) and torch.equal(graph, eager) and torch.equal(graph, again)


def test_a_window_past_the_end_is_no_window(dev):
    announce("a window past the end")
    B = 2
    plain, windowed = _model(B, 100), _model(B, 100, attention_window=1000, attention_sink=4)
    prompts, lengths = _tokens(2, B, 33), torch.tensor([33, 20])
    steps = [_tokens(3 + i, B) for i in range(3)]
    for i in range(4):
        a, b = ((x.prefill(prompts, lengths) if i == 0 else x.decode_step(steps[i - 1], lengths + i - 1))
                for x in (windowed, plain))
        _close(a, b, f"step {i}")


def test_prompts_and_steps_see_the_same_window(dev):
    """A token's logits, as a prompt's last and as a step after the prompt without it."""
    announce("prompt and step")
    m = _model(2, 100, attention_window=16, attention_sink=2)
    ids = _tokens(4, 2, 60)
    m.prefill(ids[:, :59])
    step = m.decode_step(ids[:, 59])
    _close(step, m.prefill(ids), "step and prompt")
    other = _model(2, 100)
    far = float((other.prefill(ids).double() - step.double()).norm() / step.double().norm())
    assert far > 6 * 2.0 ** -8  # and the window does hide something


@pytest.mark.parametrize("kw", OPTIONS, ids=str)
def test_speculation_verifies_as_steps_do(dev, kw):
    announce(f"speculation {kw}")
    m = _model(1, 120, **kw)
    ids = _tokens(5, 1, 50)
    five = _tokens(6, 5)
    m.prefill(ids)
    want = torch.cat([m.decode_step(five[i:i + 1]) for i in range(5)])
    m.reset()
    m.prefill(ids)
    st = m._verify_graph(5)
    for _ in range(2):
        st["tok"].copy_(five)
        st["pos"].copy_(torch.arange(50, 55, dtype=torch.int32))
        st["start"].fill_(50)
        st["graph"].replay()
        torch.cuda.synchronize()
        _close(st["logits"], want, "five tokens")
    out, stats = m.spec_generate(ids.repeat(1, 1), 20)
    assert out.shape == (1, 70) and torch.equal(out[:, :50], ids)
