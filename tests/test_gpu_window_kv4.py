"""Windowed attention and the cache in 4 bits against plain 64-bit forms, alone and
together."""

import math

import pytest
import torch

import kv4_ref as ref
from gpu_util import announce, bf16_randn
from qmoe import ops

pytestmark = pytest.mark.gpu

D = 128
SCALE = 1.0 / math.sqrt(D)
NAN = float("nan")


def _gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _fenced(shape, dtype, dev, fill=7):
    """A tensor between two fences of a known value, and a check of them."""
    n = math.prod(shape)
    buf = torch.full((n + 128,), fill, dtype=dtype, device=dev)
    t = buf[64:64 + n].view(shape)

    def whole():
        return bool((buf[:64] == fill).all() and (buf[64 + n:] == fill).all())

    return t, whole


def _within(got, want, bound, what):
    assert not bool(torch.isnan(got).any()), f"{what}: NaN"
    over = (got.double() - want).abs() / bound
    worst = float(over.max()) if over.numel() else 0.0
    print(f"  {what}: worst error {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


def _cache(dev, seed, B, Hkv, S_max, std=1.0):
    """A 4-bit cache of normal entries, made by the reference, and its values."""
    g = _gen(dev, seed)
    k4, ks = ref.quantise(bf16_randn((B, Hkv, S_max, D), g, dev, std))
    v4, vs = ref.quantise(bf16_randn((B, Hkv, S_max, D), g, dev))
    return [k4, ks, v4, vs]


# ------------------------------------------------------------------ the format
def test_store_and_load_every_value(dev):
    """Every bf16 value next to a block maximum of every size, against the reference,
    byte for byte."""
    announce("kv4_store / kv4_load, every bf16 value")
    every = torch.arange(1 << 16, dtype=torch.int32, device=dev).to(torch.int16).view(torch.bfloat16)
    g = _gen(dev, 1)
    shuffled = every[torch.randperm(1 << 16, generator=g, device=dev)]
    # values in order share a binade, so every mantissa meets every rounding
    small = every.view(-1, 32)
    rows = torch.cat([every, shuffled, (small.flip(1)).reshape(-1)]).view(1, 1, -1, D).contiguous()
    n = rows.shape[2]
    cache = ops.kv4_cache(1, 1, n, D, dev)
    ops.kv4_store(rows, rows.flip(2).contiguous(), cache)
    k, v = ops.kv4_load(cache)
    torch.cuda.synchronize()
    for got, powers, back, x in ((cache[0], cache[1], k, rows), (cache[2], cache[3], v, rows.flip(2))):
        codes, p = ref.quantise(x.double())
        assert torch.equal(powers, p)
        at = (got != codes).nonzero()
        assert at.numel() == 0, (at.shape[0], [(i, x[tuple(i[:3])][2 * i[3]:2 * i[3] + 2].tolist(),
                                                int(got[tuple(i)]), int(codes[tuple(i)])) for i in at[:5].tolist()])
        want = ref.values(codes, p)
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(back), nan)
        assert torch.equal(back.double()[~nan], want[~nan])


def test_load_reads_any_bytes(dev):
    g = _gen(dev, 2)
    cache = [torch.randint(0, 256, (2, 3, 37, w), generator=g, device=dev, dtype=torch.uint8) for w in (64, 4, 64, 4)]
    cache[1].clamp_(1, 252)  # 4 * 2^(253 - 127) is past the largest bf16 value
    cache[3].clamp_(1, 252)
    cache[1][0, 0, :5] = 255
    ko, whole_k = _fenced((2, 3, 20, D), torch.bfloat16, dev)
    vo, whole_v = _fenced((2, 3, 20, D), torch.bfloat16, dev)
    k, v = ops.kv4_load(cache, n=20, out=(ko, vo))
    torch.cuda.synchronize()
    assert k is ko and v is vo and whole_k() and whole_v()
    for got, codes, powers in ((k, *cache[:2]), (v, *cache[2:])):
        want = ref.values(codes[:, :, :20], powers[:, :, :20])
        tiny = want.abs() < 2.0 ** -126  # subnormal numbers may be flushed
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got.double()[~nan & ~tiny], want[~nan & ~tiny])
    zeros = ops.kv4_load(ops.kv4_cache(1, 1, 3, D, dev))
    assert not bool(zeros[0].any() or zeros[1].any())


STORE = [
    # B, Hkv, S, S_max, starts, lengths, n
    (1, 4, 1, 1, None, None, None),
    (2, 4, 5, 9, None, None, None),
    (3, 2, 70, 70, [0, 3, -5], [70, 20, 70], None),
    (2, 8, 33, 64, [31, 40], None, 20),
    (4, 1, 10, 12, [-2_000_000_000, 2_000_000_000, 11, -9], [10, 10, 10, 2_000_000_000], None),
    (2, 3, 17, 40, [1, 2], [0, -3], None),
    (2, 3, 17, 40, None, [5, 17], 0),
]


@pytest.mark.parametrize("case", STORE, ids=lambda c: "B{}h{}S{}of{}".format(*c[:4]))
def test_kv4_store(dev, case):
    B, Hkv, S, S_max, starts, lengths, n = case
    announce(f"kv4_store {case}")
    g = _gen(dev, B * 7 + S)
    k, v = bf16_randn((B, Hkv, S, D), g, dev), bf16_randn((B, Hkv, S, D), g, dev)
    whole, cache = [], []
    for w in (64, 4, 64, 4):
        t, check = _fenced((B, Hkv, S_max, w), torch.uint8, dev)
        t.copy_(torch.randint(0, 250, t.shape, generator=g, device=dev, dtype=torch.uint8))
        cache.append(t)
        whole.append(check)
    want = [t.clone() for t in cache]
    for b in range(B):
        for s in range(min(S if n is None else n, S if lengths is None else lengths[b])):
            at = s + (starts[b] if starts else 0)
            if 0 <= at < S_max:
                for i, x in ((0, k), (2, v)):
                    want[i][b, :, at], want[i + 1][b, :, at] = ref.quantise(x[b, :, s])
    ops.kv4_store(k, v, tuple(cache), _i32(starts, dev) if starts else None, _i32(lengths, dev) if lengths else None, n)
    torch.cuda.synchronize()
    assert all(w() for w in whole)
    assert all(torch.equal(a, b) for a, b in zip(cache, want))


def _append_inputs(dev, seed, B, S, Hq, Hkv, S_max, max_pos):
    g = _gen(dev, seed)
    qkv = torch.randn(B * S, (Hq + 2 * Hkv) * D, generator=g, device=dev) * 1.5
    qn, kn = (1.0 + 0.1 * torch.randn(2, D, generator=g, device=dev)).to(torch.bfloat16)
    inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64, device=dev) / D)
    a = torch.arange(max_pos, dtype=torch.float64, device=dev)[:, None] * inv
    return qkv, qn, kn, a.cos().float(), a.sin().float()


@pytest.mark.parametrize("B,S,Hq,Hkv,S_max", [(1, 1, 32, 4, 9), (3, 1, 64, 4, 5), (2, 5, 8, 8, 33), (7, 3, 12, 4, 8),
                                              (64, 1, 32, 4, 70)])
def test_kv4_append(dev, B, S, Hq, Hkv, S_max):
    announce(f"kv4_append {B} {S} {Hq} {Hkv} {S_max}")
    max_pos = 300
    qkv, qn, kn, cos, sin = _append_inputs(dev, B + S, B, S, Hq, Hkv, S_max, max_pos)
    g = _gen(dev, 5)
    slots = torch.stack([torch.randperm(S_max, generator=g, device=dev)[:S] for _ in range(B)]).int().view(-1)
    positions = torch.randint(0, max_pos, (B * S,), generator=g, device=dev).int()
    if B * S > 3:  # rejected tokens
        positions[0], positions[1], slots[2], slots[3] = -1, max_pos, -1, S_max
    whole, cache = [], []
    for w in (64, 4, 64, 4):
        t, check = _fenced((B, Hkv, S_max, w), torch.uint8, dev)
        t.copy_(torch.randint(0, 250, t.shape, generator=g, device=dev, dtype=torch.uint8))
        cache.append(t)
        whole.append(check)
    want = [t.clone() for t in cache]
    k, v = ref.append(qkv, qn, kn, cos, sin, positions.clamp(0, max_pos - 1), Hq, Hkv, 1e-6)
    # the sixteen values 16 of a row are alike and next to a border of two numbers:
    # 64 bits put them on one side of it
    k4, v4 = ref.quantise(k), ref.quantise(v)
    for t in range(B * S):
        p, s = int(positions[t]), int(slots[t])
        if 0 <= p < max_pos and 0 <= s < S_max:
            for i in (0, 1):
                want[i][t // S, :, s], want[2 + i][t // S, :, s] = k4[i][t], v4[i][t]
    qo, whole_q = _fenced((B * S, Hq, D), torch.bfloat16, dev)
    q = ops.kv4_append(qkv, qn, kn, cos, sin, positions, slots, Hq, Hkv, tuple(cache), 1e-6, S=S, q_out=qo)
    kb = torch.zeros(B * S, Hkv, S_max, D, dtype=torch.bfloat16, device=dev)
    q2 = ops.kv_append(qkv, qn, kn, cos, sin, positions, slots, Hq, Hkv, kb, torch.zeros_like(kb), 1e-6)
    torch.cuda.synchronize()
    assert q is qo and whole_q() and all(w() for w in whole)
    assert torch.equal(q, q2)
    for got, need, name in zip(cache, want, ("k", "k_scales", "v", "v_scales")):
        assert torch.equal(got, need), f"{name}: {int((got != need).sum())} bytes differ"


def test_kv4_append_values_that_are_not_finite(dev):
    qkv, qn, kn, cos, sin = _append_inputs(dev, 9, 2, 1, 8, 2, 4, 8)
    x = qkv.view(2, 12, D)
    x[0, 10, 3], x[1, 11, 70], x[1, 8, 5] = math.inf, NAN, NAN  # a value of each row, a key of the second
    cache = ops.kv4_cache(2, 2, 4, D, dev)
    ops.kv4_append(qkv, qn, kn, cos, sin, _i32([3, 4], dev), _i32([0, 1], dev), 8, 2, cache, 1e-6)
    k, v = ops.kv4_load(cache)
    assert bool(torch.isnan(v[0, 0, 0, :32]).all()) and not bool(torch.isnan(v[0, 0, 0, 32:]).any())
    assert bool(torch.isnan(v[1, 1, 1, 64:96]).all()) and not bool(torch.isnan(v[1, 1, 1, :64]).any())
    assert bool(torch.isnan(k[1, 0, 1]).all()) and not bool(torch.isnan(k[0]).any() or torch.isnan(k[1, 1]).any())


# ------------------------------------------------------------------ attention
ATTEND = [
    # B, S, S_max, Hq, Hkv, ctx, window, sink, max_ctx
    (1, 1, 1, 32, 4, [1], 1, 0, None),
    (1, 1, 8, 32, 4, [5], 1, 0, None),
    (1, 1, 8, 32, 4, [5], 3, 1, None),
    (2, 1, 70, 32, 4, [65, 0], 1000, 4, None),            # a row that sees nothing
    (3, 1, 70, 32, 4, [70, 1, 64], 64, 0, None),
    (4, 1, 300, 32, 4, [300, 299, 65, 66], 64, 4, None),
    (5, 1, 400, 32, 4, [400, 131, 68, 5, 333], 63, 5, None),
    (3, 1, 50, 32, 4, [-3, 2_000_000_000, -2_000_000_000], 7, 2, None),
    (3, 1, 300, 32, 4, [300, 250, 100], 60, 3, 200),      # the bucket ends before some windows begin
    (3, 1, 300, 32, 4, [300, 230, 100], 60, 0, 200),
    (2, 1, 90, 32, 4, [90, 40], 5, 60, 30),               # and inside the first entries
    (9, 1, 1200, 64, 4, [1200 - 131 * i for i in range(9)], 500, 100, None),
    (33, 1, 700, 8, 8, [(97 * i) % 701 for i in range(33)], 129, 1, None),
    (7, 1, 2200, 12, 4, [2200, 2111, 1, 0, 1500, 64, 129], 1024, 4, None),
    (2, 1, 4500, 32, 4, [4500, 4097], 4096, 4, None),
    (1, 1, 8300, 32, 4, [8297], 1 << 40, 1 << 40, None),
    (1, 2, 8, 32, 4, [1], 1, 0, None),
    (2, 2, 100, 32, 4, [1, 90], 10, 2, None),
    (2, 5, 300, 32, 4, [1, 290], 64, 4, None),
    (3, 5, 310, 32, 4, [100, -2, 306], 33, 40, None),     # queries before the first entry
    (2, 7, 40, 12, 4, [38, 12], 9, 0, None),              # queries past the last
    (2, 3, 900, 64, 4, [800, 3], 256, 4, None),
    (2, 17, 600, 32, 4, [500, 1], 128, 4, None),          # rows past 128: tiles
    (1, 64, 64, 32, 4, [1], 16, 4, None),
    (1, 200, 200, 32, 4, [1], 1, 0, None),
    (1, 200, 200, 32, 4, [1], 1, 1, None),
    (2, 130, 700, 32, 4, [1, 500], 100, 4, None),
    (1, 333, 1000, 8, 8, [600], 250, 7, None),            # one head a group: tiles of 128 queries
    (2, 150, 400, 12, 4, [1, 251], 64, 65, None),
    (1, 301, 900, 64, 4, [555], 129, 0, None),
    (2, 300, 640, 32, 4, [1, 300], 90, 4, 350),           # the bucket cuts chunks
    (1, 640, 640, 16, 4, [1], 250, 4, None),
    (1, 700, 700, 4, 4, [-40], 33, 3, None),
    (1, 1100, 1100, 8, 1, [1], 1 << 30, 0, None),
    (3, 40, 3000, 16, 2, [2961, 1, 2000], 2500, 4, None),
    (1, 1500, 1700, 8, 8, [201], 700, 7, None),           # tiles: one head a group
    (1, 1400, 1400, 4, 4, [-40], 900, 3, None),
    (2, 700, 900, 12, 4, [1, 201], 300, 65, None),
    (2, 600, 700, 32, 4, [1, 90], 1, 0, None),
    (2, 600, 700, 32, 4, [1, 90], 1, 1, None),
    (2, 600, 700, 32, 4, [1, 101], 33, 40, 500),
    (1, 1000, 1000, 16, 1, [5], 64, 64, None),            # and queries past the cache
    (2, 600, 64, 32, 4, [1, 30], 100, 0, 0),              # nothing to see at all
    (3, 1, 64, 32, 4, [1, 30, 64], 100, 2, 0),
]


def _hide(see, *tensors):
    """Sets what no query of a row sees to ``fill``: (tensor, fill) pairs."""
    for t, fill in tensors:
        for b in range(t.shape[0]):
            t[b][:, ~see[b].any(0)] = fill


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "B{}S{}of{}h{}x{}w{}s{}".format(*c[:5], c[6], c[7]))
def test_attn_window(dev, case):
    B, S, S_max, Hq, Hkv, ctx, window, sink, max_ctx = case
    announce(f"attn_window {case}")
    top = S_max if max_ctx is None else max_ctx
    g = _gen(dev, B * 31 + S_max)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    k, v = bf16_randn((B, Hkv, S_max, D), g, dev), bf16_randn((B, Hkv, S_max, D), g, dev)
    see = [ref.sees(c, S, S_max, top, window, sink).to(dev) for c in ctx]
    _hide(see, (k, NAN), (v, NAN))
    out, whole = _fenced((B * S, Hq * D), torch.bfloat16, dev)
    got = ops.attn_window(q, k, v, _i32(ctx, dev), B, S, window, sink, out=out, max_ctx=max_ctx)
    again = ops.attn_window(q, k, v, _i32(ctx, dev), B, S, window, sink, max_ctx=max_ctx)
    torch.cuda.synchronize()
    assert got is out and whole()
    want, bound = ref.window(q, k, v, ctx, B, S, window, sink, top, SCALE)
    _within(got, want, bound, "out")
    assert torch.equal(got, again)
    blind = ~torch.stack(see).any(2).view(B * S)
    assert not bool(got[blind].any())


@pytest.mark.parametrize("case", ATTEND, ids=lambda c: "B{}S{}of{}h{}x{}w{}s{}".format(*c[:5], c[6], c[7]))
@pytest.mark.parametrize("windowed", [True, False], ids=["window", "all"])
def test_attn_kv4(dev, case, windowed):
    B, S, S_max, Hq, Hkv, ctx, window, sink, max_ctx = case
    window, sink = (window, sink) if windowed else (0, 0)
    announce(f"attn_kv4 {case} {windowed}")
    top = S_max if max_ctx is None else max_ctx
    g = _gen(dev, B * 31 + S_max)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    cache = _cache(dev, B + S_max, B, Hkv, S_max)
    see = [ref.sees(c, S, S_max, top, window, sink).to(dev) for c in ctx]
    _hide(see, (cache[1], 255), (cache[3], 255), (cache[0], 119), (cache[2], 119))
    out, whole = _fenced((B * S, Hq * D), torch.bfloat16, dev)
    got = ops.attn_kv4(q, cache, _i32(ctx, dev), B, S, window, sink, out=out, max_ctx=max_ctx)
    again = ops.attn_kv4(q, tuple(cache), _i32(ctx, dev), B, S, window, sink, max_ctx=max_ctx)
    torch.cuda.synchronize()
    assert got is out and whole()
    k, v = ref.values(*cache[:2]), ref.values(*cache[2:])
    want, bound = ref.window(q, k, v, ctx, B, S, window, sink, top, SCALE)
    _within(got, want, bound, "out")
    assert torch.equal(got, again)
    blind = ~torch.stack(see).any(2).view(B * S)
    assert not bool(got[blind].any())


@pytest.mark.parametrize("B,S,S_max,Hq,Hkv,window,ctx", [
    # every workgroup takes an even share of all keys (long batches)
    (33, 1, 18000, 8, 8, 0, [18000 - 541 * i for i in range(33)]),
    (64, 1, 9000, 32, 8, 0, [9000 - 300 * (i % 31) for i in range(64)]),
    (16, 1, 32768, 64, 4, 0, [0, 32768, 1, 5, 0, 20000, 32767, 31000] * 2),
    (17, 5, 17000, 32, 4, 0, [17000 - 1000 * i for i in range(17)]),        # three row tiles an item
    (300, 1, 9000, 2, 1, 8500, [30 * i for i in range(300)]),               # more sequences than threads
    (12, 3, 34000, 16, 4, 33000, [34000, 1, -1, 33990] * 3),
], ids=lambda x: str(x) if isinstance(x, int) else "")
def test_attn_kv4_of_long_batches(dev, B, S, S_max, Hq, Hkv, window, ctx):
    announce(f"attn_kv4 long {B} {S} {S_max} {Hq} {Hkv} {window}")
    g = _gen(dev, B)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    cache = ops.kv4_cache(B, Hkv, S_max, D, dev)
    for b in range(B):
        rows = [bf16_randn((1, Hkv, S_max, D), g, dev) for _ in range(2)]
        ops.kv4_store(*rows, tuple(t[b:b + 1] for t in cache))
    got = ops.attn_kv4(q, cache, _i32(ctx, dev), B, S, window, 4 if window else 0)
    again = ops.attn_kv4(q, cache, _i32(ctx, dev), B, S, window, 4 if window else 0)
    torch.cuda.synchronize()
    assert torch.equal(got, again) and not bool(torch.isnan(got).any())
    for b in sorted({0, 1, 2, B // 2, B - 2, B - 1}):
        one = slice(b * S, (b + 1) * S)
        k, v = (ref.values(c[b:b + 1], p[b:b + 1]) for c, p in (cache[:2], cache[2:]))
        _within(got[one], *ref.window(q[one], k, v, [ctx[b]], 1, S, window, 4 if window else 0, S_max, SCALE), f"row {b}")


@pytest.mark.parametrize("four", [False, True], ids=["bf16", "four"])
@pytest.mark.parametrize("B,S,n,Hq,Hkv", [
    # on both sides of where a workgroup has 1, 2, 4 and 8 waves, and a call one launch or two
    (1, 1, 60, 32, 4), (1, 1, 256, 32, 4), (1, 1, 257, 32, 4), (1, 1, 385, 32, 4), (1, 1, 513, 8, 8), (3, 1, 1000, 32, 4),
    (1, 1, 1030, 32, 4), (2, 1, 1280, 32, 4), (1, 1, 1290, 32, 4), (1, 1, 2045, 64, 4), (5, 1, 2050, 32, 4),
    (1, 1, 4100, 32, 4), (34, 1, 900, 32, 4), (33, 1, 1500, 32, 4), (70, 1, 400, 32, 4), (2, 5, 700, 32, 4),
    (1, 3, 1200, 64, 4), (1, 7, 3000, 32, 8)])
def test_few_rows_of_any_length(dev, B, S, n, Hq, Hkv, four):
    announce(f"few rows {B} {S} {n} {Hq} {Hkv} {'4 bits' if four else 'bf16'}")
    g = _gen(dev, n)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    ctx = [max(-S, n - S + 1 - 67 * i) for i in range(B)]
    k, v = (bf16_randn((B, Hkv, n, D), g, dev) for _ in range(2))
    for window, sink in (((0, 0),) if four else ()) + ((n, 0), (n - 10, 4), (n // 2, 5)):
        if four:
            cache = ops.kv4_cache(B, Hkv, n, D, dev)
            ops.kv4_store(k, v, cache)
            got = ops.attn_kv4(q, cache, _i32(ctx, dev), B, S, window, sink)
            held = [ref.values(*cache[i:i + 2]) for i in (0, 2)]
        else:
            got, held = ops.attn_window(q, k, v, _i32(ctx, dev), B, S, window, sink), [k, v]
        _within(got, *ref.window(q, *held, ctx, B, S, window, sink, n, SCALE), f"window {window}")


@pytest.mark.parametrize("scale", [1.0, 1e-3, 0.5])
def test_scales(dev, scale):
    g = _gen(dev, 3)
    q = bf16_randn((2, 32, D), g, dev)
    k, v = bf16_randn((2, 4, 200, D), g, dev), bf16_randn((2, 4, 200, D), g, dev)
    got = ops.attn_window(q, k, v, _i32([200, 90], dev), 2, 1, 70, 4, scale=scale)
    _within(got, *ref.window(q, k, v, [200, 90], 2, 1, 70, 4, 200, scale), "window")
    cache = _cache(dev, 4, 2, 4, 200)
    got = ops.attn_kv4(q, cache, _i32([200, 90], dev), 2, 1, scale=scale)
    k, v = ref.values(*cache[:2]), ref.values(*cache[2:])
    _within(got, *ref.window(q, k, v, [200, 90], 2, 1, 0, 0, 200, scale), "kv4")


def test_a_cache_of_all_powers(dev):
    """Keys and values of sizes from 2^-60 to 2^60, a power of its own in every block."""
    g = _gen(dev, 6)
    B, Hkv, n = 2, 2, 150
    cache = _cache(dev, 7, B, Hkv, n)
    cache[1].copy_(torch.randint(60, 128, cache[1].shape, generator=g, device=dev))
    cache[3].copy_(torch.randint(60, 190, cache[3].shape, generator=g, device=dev))
    q = bf16_randn((B, 16, D), g, dev)
    got = ops.attn_kv4(q, cache, _i32([n, 77], dev), B, 1)
    k, v = ref.values(*cache[:2]), ref.values(*cache[2:])
    _within(got, *ref.window(q, k, v, [n, 77], B, 1, 0, 0, n, SCALE), "out")


def test_workspaces_are_checked(dev):
    q = torch.zeros(64, 32, D, dtype=torch.bfloat16, device=dev)
    cache = ops.kv4_cache(64, 4, 20000, D, dev)
    ctx = torch.full((64,), 3, dtype=torch.int32, device=dev)
    ws = ops.attn_kv4_workspace(64, 1, 32, 4, D, 0, 0, 20000, dev)
    if ws is not None:
        a = ops.attn_kv4(q, cache, ctx, 64, 1, workspace=ws)
        assert torch.equal(a, torch.zeros_like(a))
        with pytest.raises(ValueError, match="needs"):
            ops.attn_kv4(q, cache, ctx, 64, 1, workspace=ws[:-1])
        with pytest.raises(ValueError, match="aligned"):
            ops.attn_kv4(q, cache, ctx, 64, 1, workspace=torch.empty(ws.numel() + 16, dtype=torch.uint8,
                                                                     device=dev)[8:])
    with pytest.raises(ValueError, match="overlaps"):
        ops.attn_kv4(q, cache, ctx, 64, 1, out=q.view(64, 32 * D))
    with pytest.raises(ValueError, match="uint8|Byte"):
        ops.attn_kv4(q, (cache[0].char(), *cache[1:]), ctx, 64, 1)
    with pytest.raises(ValueError, match="contiguous"):
        ops.attn_kv4(q, (cache[0][:, :, ::2], *(t[:, :, ::2] for t in cache[1:])), ctx, 64, 1)
    with pytest.raises(ValueError, match="hold B"):
        ops.attn_kv4(q[:32], cache, ctx[:32], 32, 1)
    with pytest.raises(ValueError, match="shape"):
        ops.attn_kv4(q, (cache[0], cache[1][..., :2].contiguous(), *cache[2:]), ctx, 64, 1)
