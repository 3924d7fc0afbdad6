"""The operators of a decode batch's cache against plain 64-bit forms: attention
over a shared prefix, attention that accumulates its weights, appending to and
evicting from a cache of bounded size, and a run of them together."""

import math

import pytest
import torch

import cache_ref as ref
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


def _fenced(shape, dtype, dev):
    """A tensor between two fences of a known value, and a check of them."""
    n = math.prod(shape)
    buf = torch.full((n + 128,), 7.0, dtype=dtype, device=dev)
    t = buf[64:64 + n].view(shape)

    def whole():
        return bool((buf[:64] == 7.0).all() and (buf[64 + n:] == 7.0).all())

    return t, whole


def _within(got, want, bound, what):
    over = ((got.double() - want).abs() / bound)
    assert not bool(torch.isnan(got).any()), f"{what}: NaN"
    worst = float(over.max()) if over.numel() else 0.0
    print(f"  {what}: worst error {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


# ------------------------------------------------------------------ shared prefix
def _shared_inputs(dev, seed, B, S, P, P_max, S_max, Hq, Hkv, ctx, max_ctx):
    g = _gen(dev, seed)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    kp, vp = bf16_randn((Hkv, P_max, D), g, dev), bf16_randn((Hkv, P_max, D), g, dev)
    k, v = bf16_randn((B, Hkv, S_max, D), g, dev), bf16_randn((B, Hkv, S_max, D), g, dev)
    for t in (kp, vp):  # nothing past the prefix is read
        t[:, P:] = NAN
    for b in range(B):
        end = min(max(ctx[b] + S - 1, 0), max_ctx, S_max)
        k[b, :, end:] = NAN
        v[b, :, end:] = NAN
    return q, kp, vp, k, v


SHARED = [
    # B, S, P, P_max, S_max, Hq, Hkv, own entries of each row, max_ctx
    (1, 1, 1, 1, 1, 32, 4, [0], None),
    (1, 1, 1, 1, 8, 32, 4, [1], None),
    (2, 1, 0, 5, 70, 32, 4, [65, 0], None),            # no prefix; a row that sees nothing
    (3, 1, 63, 80, 64, 32, 4, [64, 1, 63], None),
    (3, 1, 64, 64, 65, 32, 4, [65, 64, 0], None),
    (5, 1, 65, 100, 130, 32, 4, [130, 129, 128, 2, 1], None),
    (4, 1, 300, 300, 40, 32, 4, [24, 6, 18, 12], 24),
    (2, 1, 333, 400, 500, 32, 4, [500, 499], 200),     # the bucket cuts what a row sees
    (3, 1, 100, 100, 50, 32, 4, [-3, 2_000_000_000, -2_000_000_000], None),
    (16, 1, 1000, 1000, 100, 32, 4, list(range(0, 96, 6)), None),
    (17, 1, 2111, 2200, 300, 32, 4, [17 * i for i in range(17)], None),
    (33, 1, 700, 700, 90, 16, 4, [(7 * i) % 91 for i in range(33)], None),
    (20, 1, 515, 515, 77, 64, 4, [(5 * i) % 78 for i in range(20)], None),  # 16 heads a group
    (9, 1, 200, 200, 33, 8, 8, [(4 * i) % 34 for i in range(9)], None),     # one head a group
    (7, 1, 190, 190, 33, 12, 4, [(5 * i) % 34 for i in range(7)], None),    # three
    (2, 2, 100, 100, 64, 32, 4, [1, 1], None),
    (2, 5, 129, 129, 90, 32, 4, [1, 40], None),
    (1, 15, 64, 64, 15, 32, 4, [1], None),
    (3, 16, 97, 97, 80, 32, 4, [1, 0, 64], None),      # from 16 queries a tile holds one row's
    (2, 37, 500, 512, 120, 32, 4, [1, 84], None),
    (2, 101, 290, 290, 101, 32, 4, [1, 1], None),
    (1, 200, 0, 1, 200, 32, 4, [1], None),             # no prefix: a prompt
    (3, 70, 65, 65, 70, 32, 4, [1, -30, 1], 50),       # queries that see no own entry, and a bucket
    (2, 43, 130, 130, 60, 12, 4, [3, 17], None),
    (1, 130, 70, 70, 140, 8, 8, [5], None),
    (2, 9, 300, 300, 20, 64, 4, [1, 12], None),
    # a prefix that is attended in tiles (more than 65536 keys over the blocks of 32 rows)
    (70, 1, 2001, 2100, 40, 16, 1, [(3 * i) % 41 for i in range(70)], None),
    (20, 3, 4511, 4511, 50, 32, 4, [1 + 2 * i for i in range(20)], None),
    (9, 15, 2003, 2003, 30, 8, 1, [1 + (5 * i) % 16 for i in range(9)], None),   # and own keys in tiles
    (1, 60, 1111, 1111, 300, 2, 2, [200], None),                                # one head, 60 queries
]


@pytest.mark.parametrize("case", SHARED, ids=lambda c: "B{}S{}P{}h{}x{}".format(c[0], c[1], c[2], c[5], c[6]))
def test_attn_shared(dev, case):
    B, S, P, P_max, S_max, Hq, Hkv, ctx, max_ctx = case
    announce(f"attn_shared {case}")
    top = S_max if max_ctx is None else max_ctx
    q, kp, vp, k, v = _shared_inputs(dev, B * 31 + P, B, S, P, P_max, S_max, Hq, Hkv, ctx, top)
    out, whole = _fenced((B * S, Hq * D), torch.bfloat16, dev)
    args = (q, kp, vp, k, v, _i32(ctx, dev), B, S)
    got = ops.attn_shared(*args, prefix_len=P, out=out, max_ctx=max_ctx)
    again = ops.attn_shared(*args, prefix_len=P, max_ctx=max_ctx)
    torch.cuda.synchronize()
    assert got is out and whole()
    want, bound = ref.shared(q, kp, vp, k, v, ctx, B, S, P, top, SCALE)
    _within(got, want, bound, "out")
    assert torch.equal(got, again)
    if P == 0:  # rows that see nothing
        for b in range(B):
            if ctx[b] <= 0 and S == 1:
                assert not bool(got[b].any())


# ------------------------------------------------------------------ prompts
PROMPT = [
    # B, S, start, S_max, Hq, Hkv, lengths
    (1, 1, 0, 1, 32, 4, None),
    (1, 1, 77, 90, 32, 4, None),
    (2, 2, 0, 3, 32, 4, [2, 1]),
    (1, 15, 0, 15, 32, 4, None),
    (1, 16, 3, 30, 32, 4, None),
    (2, 33, 0, 33, 32, 4, [33, 0]),            # a row of padding alone
    (1, 64, 0, 64, 32, 4, None),
    (1, 65, 0, 70, 32, 4, None),
    (3, 100, 57, 160, 32, 4, [100, 1, 63]),
    (2, 257, 0, 300, 32, 4, [200, 257]),
    (1, 640, 0, 641, 32, 4, None),
    (1, 300, 511, 900, 32, 4, [299]),
    (2, 130, 20, 155, 8, 8, [130, 99]),
    (1, 90, 0, 90, 12, 4, None),
    (2, 50, 300, 350, 64, 4, [50, 17]),
    (1, 222, 0, 222, 16, 4, [5]),
    (2, 40, 0, 40, 32, 4, [50, -7]),           # lengths out of range are clamped
]


@pytest.mark.parametrize("case", PROMPT, ids=lambda c: "B{}S{}at{}h{}x{}".format(c[0], c[1], c[2], c[4], c[5]))
def test_attn_prefill_scored(dev, case):
    B, S, start, S_max, Hq, Hkv, lengths = case
    announce(f"attn_prefill_scored {case}")
    g = _gen(dev, S * 7 + start)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    k, v = bf16_randn((B, Hkv, S_max, D), g, dev), bf16_randn((B, Hkv, S_max, D), g, dev)
    k[:, :, start + S:] = NAN
    v[:, :, start + S:] = NAN
    base = torch.rand(B, Hkv, S_max, generator=g, device=dev)
    n = None if lengths is None else _i32(lengths, dev)
    for b, ln in enumerate(lengths or []):  # what padding holds does not reach the scores
        q.view(B, S, Hq, D)[b, max(0, min(ln, S)) + 1:] = NAN
    sc, whole_sc = _fenced((B, Hkv, S_max), torch.float32, dev)
    sc.copy_(base)
    out, whole = _fenced((B * S, Hq * D), torch.bfloat16, dev)
    got = ops.attn_prefill_scored(q, k, v, sc, B, S, start, lengths=n, out=out)
    sc2 = base.clone()
    again = ops.attn_prefill_scored(q, k, v, sc2, B, S, start, lengths=n)
    torch.cuda.synchronize()
    assert got is out and whole() and whole_sc()
    assert torch.equal(sc, sc2)
    real = torch.ones(B, S, dtype=torch.bool, device=dev)
    clamped = [max(0, min(ln, S)) for ln in lengths] if lengths is not None else [S] * B
    for b in range(B):
        real[b, clamped[b] + 1:] = False
    real = real.view(-1)
    want, bound, add, off = ref.scored(q.nan_to_num(0.0), k, v, [start + 1] * B, B, S, clamped, SCALE)
    _within(got[real], want[real], bound[real], "out")
    assert torch.equal(got[real], again[real])
    total = base.double() + add
    _within(sc, total, off + 2 * ref.F32 * total.abs() + 1e-12, "scores")
    assert torch.equal(sc[:, :, start + S:], base[:, :, start + S:])
    # the whole weight of a query is 1
    assert torch.allclose(add.sum((1, 2)), torch.tensor([float(c * Hq) for c in clamped], device=dev).double())


# ------------------------------------------------------------------ scored decode
SCORED = [
    # B, S_max, Hq, Hkv, ctx, max_ctx
    (1, 1, 32, 4, [1], None),
    (1, 300, 32, 4, [1], None),
    (2, 70, 32, 4, [0, 65], None),             # a row that sees nothing
    (3, 256, 32, 4, [64, 63, 256], None),
    (2, 257, 32, 4, [257, 256], None),
    (4, 1100, 32, 4, [1100, 1000, 3, 511], None),
    (3, 1100, 32, 4, [1100, -5, 2_000_000_000], 600),
    (1, 20000, 32, 4, [19777], None),          # more than 64 splits
    (9, 333, 64, 4, [37 * i for i in range(9)], None),
    (5, 200, 8, 8, [200, 1, 0, 64, 65], None),
    (5, 200, 12, 4, [200, 1, 0, 64, 65], None),
    (40, 130, 16, 4, [(9 * i) % 131 for i in range(40)], None),
    # four waves a workgroup (more than 512 waves' keys in all)
    (33, 300, 32, 4, [(29 * i) % 301 for i in range(33)], None),
    (9, 1000, 64, 4, [0, 1000, 257, 256, 64, 1, 999, 512, 300], None),
    (20, 500, 8, 8, [(53 * i) % 501 for i in range(20)], 480),
    (15, 800, 12, 4, [(97 * i) % 801 for i in range(15)], None),
]


@pytest.mark.parametrize("case", SCORED, ids=lambda c: "B{}L{}h{}x{}".format(c[0], c[1], c[2], c[3]))
def test_attn_decode_scored(dev, case):
    B, S_max, Hq, Hkv, ctx, max_ctx = case
    announce(f"attn_decode_scored {case}")
    g = _gen(dev, S_max + B)
    top = S_max if max_ctx is None else max_ctx
    seen = [max(0, min(c, top)) for c in ctx]
    q = bf16_randn((B, Hq, D), g, dev, 2.0)
    k, v = bf16_randn((B, Hkv, S_max, D), g, dev), bf16_randn((B, Hkv, S_max, D), g, dev)
    for b in range(B):
        k[b, :, seen[b]:] = NAN
        v[b, :, seen[b]:] = NAN
    base = torch.rand(B, Hkv, S_max, generator=g, device=dev)
    sc, whole_sc = _fenced((B, Hkv, S_max), torch.float32, dev)
    sc.copy_(base)
    out, whole = _fenced((B, Hq * D), torch.bfloat16, dev)
    got = ops.attn_decode_scored(q, k, v, _i32(ctx, dev), sc, out=out, max_ctx=max_ctx)
    sc2 = base.clone()
    again = ops.attn_decode_scored(q, k, v, _i32(ctx, dev), sc2, max_ctx=max_ctx)
    torch.cuda.synchronize()
    assert got is out and whole() and whole_sc()
    assert torch.equal(got, again) and torch.equal(sc, sc2)
    want, bound, add, off = ref.scored(q, k, v, seen, B, 1, None, SCALE)
    _within(got, want, bound, "out")
    total = base.double() + add
    _within(sc, total, off + 2 * ref.F32 * total.abs() + 1e-12, "scores")
    for b in range(B):
        assert torch.equal(sc[b, :, seen[b]:], base[b, :, seen[b]:])


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("B,Hq,Hkv,S_max", [(1, 32, 4, 1), (3, 32, 4, 70), (17, 8, 8, 9), (64, 32, 4, 40),
                                            (5, 12, 4, 33), (130, 64, 4, 12)])
def test_kv_append(dev, B, Hq, Hkv, S_max):
    announce(f"kv_append B={B} Hq={Hq} Hkv={Hkv}")
    g = _gen(dev, B + S_max)
    max_pos, eps = 300, 1e-6
    raw = torch.randn(B, (Hq + 2 * Hkv) * D, generator=g, device=dev) * 3
    qn, kn = [(1 + 0.1 * torch.randn(D, generator=g, device=dev)).to(torch.bfloat16) for _ in range(2)]
    ang = torch.randn(max_pos, D // 2, generator=g, device=dev) * 100
    cos, sin = ang.cos(), ang.sin()
    pos = torch.randint(0, max_pos, (B,), generator=g, device=dev).int()
    slot = torch.randint(0, S_max, (B,), generator=g, device=dev).int()
    bad = {}
    if B >= 17:  # rejected rows: no entry, a zero query
        for i, (p, s) in enumerate([(-1, 0), (max_pos, 0), (5, -1), (5, S_max), (2 ** 31 - 1, 0)]):
            pos[i], slot[i], bad[i] = p, s, True
    k, v = bf16_randn((B, Hkv, S_max, D), g, dev), bf16_randn((B, Hkv, S_max, D), g, dev)
    sc = torch.rand(B, Hkv, S_max, generator=g, device=dev) + 1
    sp = torch.full((B, Hkv, S_max), 99, dtype=torch.int32, device=dev)
    old = [t.clone() for t in (k, v, sc, sp)]
    q, whole = _fenced((B, Hq, D), torch.bfloat16, dev)
    ops.kv_append(raw, qn, kn, cos, sin, pos, slot, Hq, Hkv, k, v, eps, scores=sc, slot_pos=sp, q_out=q)
    k3, v3 = old[0].clone(), old[1].clone()
    q3 = ops.kv_append(raw, qn, kn, cos, sin, pos, slot, Hq, Hkv, k3, v3, eps)  # no scores, no positions
    torch.cuda.synchronize()
    assert whole() and torch.equal(q, q3) and torch.equal(k, k3) and torch.equal(v, v3)
    x = raw.double().view(B, Hq + 2 * Hkv, D)
    for b in range(B):
        if bad.get(b):
            assert not bool(q[b].any())
            continue
        p, s = int(pos[b]), int(slot[b])
        c, sn = cos[p].double(), sin[p].double()
        for h in range(Hq + 2 * Hkv):
            y, size = x[b, h], x[b, h].abs()
            if h < Hq + Hkv:
                y = y / torch.sqrt((y * y).mean() + eps) * (qn if h < Hq else kn).double()
                lo, hi = y[:64], y[64:]
                y = torch.cat([lo * c - hi * sn, hi * c + lo * sn])
                size = torch.cat([(lo * c).abs() + (hi * sn).abs(), (hi * c).abs() + (lo * sn).abs()])
            got = q[b, h] if h < Hq else (k[b, h - Hq, s] if h < Hq + Hkv else v[b, h - Hq - Hkv, s])
            # one rounding to bf16 of a value whose two products are off by 200 steps of 32 bits at most
            # (128 squares, the root, three factors)
            tol = y.abs() * ref.HALF_BF16 + size * 200 * ref.F32 + 1e-30
            assert bool(((got.double() - y).abs() <= tol).all()), (b, h)
        assert not bool(sc[b, :, s].any()) and bool((sp[b, :, s] == p).all())
        for t, o in zip((k, v, sc, sp), old):  # put the entry back: nothing else changed
            t[b, :, s] = o[b, :, s]
    for t, o in zip((k, v, sc, sp), old):
        assert torch.equal(t, o)


# ------------------------------------------------------------------ eviction
EVICT = [
    # B, Hkv, S_max, ctx, budget, recent, sink, distribution of the scores
    (1, 4, 1, [1], 1, 0, 0, "spread"),
    (1, 4, 2, [2], 1, 1, 0, "spread"),
    (2, 4, 64, [64, 63], 64, 8, 4, "spread"),            # nothing to evict
    (2, 4, 65, [65, 10], 64, 8, 4, "spread"),            # one entry, and none
    (3, 4, 200, [200, 0, 129], 128, 16, 4, "spread"),
    (2, 4, 300, [300, 299], 100, 100, 0, "spread"),      # the recent ones alone
    (2, 4, 300, [300, 299], 100, 0, 100, "spread"),      # the first ones alone
    (2, 4, 300, [300, 280], 100, 0, 0, "equal"),         # all equal: the lowest slots
    (2, 4, 777, [777, 700], 333, 20, 3, "few"),          # many ties
    (1, 4, 2500, [2500], 7, 2, 1, "spread"),
    (1, 4, 2500, [2500], 2499, 2, 1, "spread"),
    (2, 4, 1088, [1088, 1088], 1024, 128, 4, "spread"),
    (1, 2, 5000, [4999], 3000, 64, 4, "special"),        # infinities, NaN, zeros of both signs, negatives
    (3, 4, 90, [-4, 2_000_000_000, 90], 40, 5, 2, "spread"),
    (1, 8, 128, [128], 1000, 10, 4, "spread"),           # a budget past the capacity
    (1, 2, 9000, [8765], 300, 64, 4, "special"),         # 16 slots a thread
    (1, 2, 2000, [1999], 1700, 0, 0, "equal"),           # in place: 299 rows move in a launch of their own
    (2, 2, 1500, [1500, 1300], 1250, 40, 4, "few"),      # in place: the selection moves them
]


def _evict_inputs(dev, case):
    B, Hkv, S_max, ctx, budget, recent, sink, dist = case
    g = _gen(dev, S_max * 3 + budget)
    k, v = bf16_randn((B, Hkv, S_max, D), g, dev), bf16_randn((B, Hkv, S_max, D), g, dev)
    if dist == "equal":
        sc = torch.full((B, Hkv, S_max), 0.5, device=dev)
    elif dist == "few":
        sc = torch.randint(0, 3, (B, Hkv, S_max), generator=g, device=dev).float()
    else:
        sc = (torch.randn(B, Hkv, S_max, generator=g, device=dev) * 1.5).exp()
    if dist == "special":
        pick = torch.randint(0, 12, (B, Hkv, S_max), generator=g, device=dev)
        for i, x in enumerate([math.inf, -math.inf, NAN, 0.0, -0.0, -1.5, 1e-42, 3e38]):
            sc[pick == i] = x
    order = torch.rand(B, Hkv, S_max, generator=g, device=dev).argsort(-1)
    pos = order.int() * 2 + 1
    if sink:
        pos[pos < 2 * sink] -= 1  # some of the first positions
    return k, v, sc, pos.contiguous(), _i32(ctx, dev)


@pytest.mark.parametrize("case", EVICT, ids=lambda c: "B{}L{}to{}r{}s{}{}".format(c[0], c[2], c[4], c[5], c[6], c[7]))
@pytest.mark.parametrize("place", ["same", "other"])
def test_kv_evict(dev, case, place):
    B, Hkv, S_max, ctx, budget, recent, sink, _ = case
    announce(f"kv_evict {place} {case}")
    k, v, sc, pos, n = _evict_inputs(dev, case)
    src = (k, v, sc, pos)
    old = [t.clone() for t in src]
    if place == "same":
        want = ref.evict(k.cpu(), v.cpu(), sc.cpu(), pos.cpu(), ctx, budget, recent, sink)
        ops.kv_evict(*src, n, budget, recent=recent, sink=sink)
        got = src
    else:
        S_out = min(budget, S_max) + 9
        got = (torch.full((B, Hkv, S_out, D), 3.0, dtype=torch.bfloat16, device=dev),
               torch.full((B, Hkv, S_out, D), 4.0, dtype=torch.bfloat16, device=dev),
               torch.full((B, Hkv, S_out), 5.0, device=dev),
               torch.full((B, Hkv, S_out), 6, dtype=torch.int32, device=dev))
        want = ref.evict(k.cpu(), v.cpu(), sc.cpu(), pos.cpu(), ctx, budget, recent, sink, [t.cpu() for t in got])
        ops.kv_evict(*src, n, budget, recent=recent, sink=sink, out=got)
    torch.cuda.synchronize()
    for name, x, y in zip(("k", "v", "scores", "slot_pos"), got, want):
        x = x.cpu()
        same = (x == y) | ((x != x) & (y != y))
        assert bool(same.all()), name
    if place == "other":
        for x, y in zip(src, old):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


@pytest.mark.parametrize("n,budget", [(16_384, 5000), (20_001, 19_000), (40_001, 20_000)])
def test_kv_evict_of_long_caches(dev, n, budget):
    """As many entries as threads hold in registers, more (ranks in LDS), and more
    than that holds: sorted by torch instead of by lists."""
    B, Hkv, recent, sink = 1, 2, 100, 4
    announce(f"kv_evict n={n}")
    g = _gen(dev, 5)
    k, v = bf16_randn((B, Hkv, n, D), g, dev), bf16_randn((B, Hkv, n, D), g, dev)
    sc = torch.rand(B, Hkv, n, generator=g, device=dev)
    sc[:, :, ::3] = 0.25
    pos = torch.arange(n, dtype=torch.int32, device=dev).repeat(B, Hkv, 1)
    k0, sc0 = k.clone(), sc.clone()
    ops.kv_evict(k, v, sc, pos, _i32([n], dev), budget, recent=recent, sink=sink)
    torch.cuda.synchronize()
    for h in range(Hkv):
        rank = sc0[0, h].double().clone()
        rank[:sink] = math.inf
        rank[n - recent:] = math.inf
        keep = torch.sort(rank, descending=True, stable=True).indices[:budget].sort().values
        stay = keep[keep < budget]
        hole = torch.ones(budget, dtype=torch.bool, device=dev)
        hole[stay] = False
        want = torch.arange(budget, device=dev)
        want[hole] = keep[keep >= budget]
        assert torch.equal(pos[0, h, :budget].long(), want)
        assert torch.equal(k[0, h, :budget], k0[0, h, want]) and torch.equal(sc[0, h, :budget], sc0[0, h, want])
        assert bool((pos[0, h, budget:] == -1).all()) and not bool(sc[0, h, budget:].any())


# ------------------------------------------------------------------ refusals on the GPU
def test_wrappers_refuse_before_any_launch(dev):
    """Every argument that does not fit is named; the outputs stay as they were."""
    announce("refusals")
    B, S_max, P = 2, 8, 9
    q = torch.ones(B, 32, D, dtype=torch.bfloat16, device=dev)
    k, v = torch.ones(2, B, 4, S_max, D, dtype=torch.bfloat16, device=dev)
    kp = torch.ones(4, P, D, dtype=torch.bfloat16, device=dev)
    sc, sp = torch.ones(B, 4, S_max, device=dev), torch.ones(B, 4, S_max, dtype=torch.int32, device=dev)
    n = torch.ones(B, dtype=torch.int32, device=dev)
    out = torch.full((B, 32 * D), 7.0, dtype=torch.bfloat16, device=dev)
    raw, w = torch.ones(B, 40 * D, device=dev), torch.ones(D, dtype=torch.bfloat16, device=dev)
    cos = torch.ones(4, D // 2, device=dev)
    odd = torch.ones(B * 4 * S_max * D + 8, dtype=torch.bfloat16, device=dev)[1:-7].view(B, 4, S_max, D)
    tiny = torch.zeros(16, dtype=torch.uint8, device=dev)

    def shared(q=q, kp=kp, vp=kp, k=k, v=v, n=n, B=B, S=1, **kw):
        return ops.attn_shared(q, kp, vp, k, v, n, B, S, out=kw.pop("out", out), **kw)

    def prompt(q=q, k=k, v=v, sc=sc, B=1, S=2, start=0, **kw):
        return ops.attn_prefill_scored(q, k, v, sc, B, S, start, out=out, **kw)

    def scored(q=q, k=k, v=v, n=n, sc=sc, **kw):
        return ops.attn_decode_scored(q, k, v, n, sc, out=out, **kw)

    def append(raw=raw, qn=w, kn=w, cos=cos, sin=cos, pos=n, slots=n, Hq=32, Hkv=4, k=k, v=v, **kw):
        return ops.kv_append(raw, qn, kn, cos, sin, pos, slots, Hq, Hkv, k, v, 1e-6, **kw)

    def evict(k=k, v=v, sc=sc, sp=sp, n=n, budget=4, **kw):
        return ops.kv_evict(k, v, sc, sp, n, budget, **kw)

    other = tuple(torch.empty_like(t) for t in (k, v, sc, sp))
    refused = [
        (shared, dict(B=3), "q must be"), (shared, dict(q=q.float()), "q: dtype"),
        (shared, dict(q=q.transpose(0, 1).contiguous().transpose(0, 1)), "q: must be contiguous"),
        (shared, dict(k=k[:1]), "k_cache must be"), (shared, dict(v=v[:, :, :7].contiguous()), "v_cache: shape"),
        (shared, dict(v=v.cpu()), "v_cache: must be on a GPU"), (shared, dict(k=odd, v=odd), "16-byte aligned"),
        (shared, dict(q=q[:, :30].contiguous()), "multiple of Hkv"), (shared, dict(kp=kp[:3]), "k_prefix must be"),
        (shared, dict(vp=kp[:, :8].contiguous()), "v_prefix: shape"), (shared, dict(n=n.long()), "ctx_len: dtype"),
        (shared, dict(n=n[:1]), "ctx_len: shape"), (shared, dict(prefix_len=10), "prefix_len"),
        (shared, dict(prefix_len=-1), "prefix_len"), (shared, dict(max_ctx=9), "max_ctx"),
        (shared, dict(max_ctx=-1), "max_ctx"), (shared, dict(scale=0.0), "scale"),
        (shared, dict(scale=NAN), "scale"), (shared, dict(workspace=tiny), "workspace: needs"),
        (shared, dict(workspace=tiny.cpu()), "workspace: must be"), (shared, dict(out=out[:1]), "out: shape"),
        (shared, dict(out=out.float()), "out: dtype"),
        (prompt, dict(B=2, S=2), "q must be"), (prompt, dict(B=1, S=2), "k_cache must be"),
        (prompt, dict(k=k[:1], v=v[:1]), "scores: shape"),
        (prompt, dict(k=k[:1], v=v[:1], sc=sc[:1], start=7), "start"),
        (prompt, dict(k=k[:1], v=v[:1], sc=sc[:1], start=-1), "start"),
        (prompt, dict(k=k[:1], v=v[:1], sc=sc[:1], lengths=n), "lengths: shape"),
        (prompt, dict(k=k[:1], v=v[:1], sc=sc[:1], workspace=tiny), "workspace: needs"),
        (scored, dict(sc=sc.double()), "scores: dtype"), (scored, dict(max_ctx=0), "max_ctx"),
        (scored, dict(scale=-1.0), "scale"), (scored, dict(workspace=tiny), "workspace: needs"),
        (append, dict(Hkv=2), "heads"), (append, dict(raw=raw[:1]), "k_cache must be"),
        (append, dict(sin=cos[:3]), "rope_sin: shape"), (append, dict(qn=w.float()), "q_norm_w: dtype"),
        (append, dict(scores=sc[:1]), "scores: shape"), (append, dict(slot_pos=sp.long()), "slot_pos: dtype"),
        (append, dict(q_out=q[:1]), "q_out: shape"), (append, dict(Hq=30), "qkv: shape"),
        (evict, dict(budget=0), "budget"), (evict, dict(recent=3, sink=2), "recent"),
        (evict, dict(sp=sp[:1]), "slot_pos: shape"), (evict, dict(out=other[:3]), "out must be"),
        (evict, dict(out=(k, v, other[2], other[3])), "overlaps"),
        (evict, dict(out=(other[0], other[1], sc, other[3])), "overlaps"),
        (evict, dict(out=tuple(t[:, :, :3].contiguous() for t in other)), "at least 4 slots"),
        (evict, dict(workspace=tiny), "workspace: needs"),
    ]
    before = [t.clone() for t in (k, v, sc, sp, out)]
    for call, change, msg in refused:
        with pytest.raises(ValueError, match=msg):
            call(**change)
    torch.cuda.synchronize()
    for t, x in zip((k, v, sc, sp, out), before):
        assert torch.equal(t, x)


def test_empty_batches_and_given_workspaces(dev):
    announce("empty batches")
    none = torch.empty(0, 32, D, dtype=torch.bfloat16, device=dev)
    k = torch.zeros(0, 4, 8, D, dtype=torch.bfloat16, device=dev)
    kp = torch.zeros(4, 9, D, dtype=torch.bfloat16, device=dev)
    n, sc = torch.zeros(0, dtype=torch.int32, device=dev), torch.zeros(0, 4, 8, device=dev)
    sp = torch.zeros(0, 4, 8, dtype=torch.int32, device=dev)
    assert ops.attn_shared(none, kp, kp, k, k, n, 0, 1).shape == (0, 32 * D)
    assert ops.attn_decode_scored(none, k, k, n, sc).shape == (0, 32 * D)
    one = torch.zeros(1, 4, 8, D, dtype=torch.bfloat16, device=dev)
    assert ops.attn_prefill_scored(none, one, one, torch.zeros(1, 4, 8, device=dev), 1, 0).shape == (0, 32 * D)
    ops.kv_evict(k, k, sc, sp, n, 4)
    g = _gen(dev, 9)
    q = bf16_randn((3, 32, D), g, dev)
    k, v = bf16_randn((3, 4, 300, D), g, dev), bf16_randn((3, 4, 300, D), g, dev)
    n, sc = _i32([300, 2, 150], dev), torch.zeros(3, 4, 300, device=dev)
    pos = torch.arange(300, dtype=torch.int32, device=dev).repeat(3, 4, 1)
    a = ops.attn_decode_scored(q, k, v, n, sc)
    sc2 = torch.zeros_like(sc)
    b = ops.attn_decode_scored(q, k, v, n, sc2, workspace=ops.attn_decode_scored_workspace(3, 32, D, 300, dev))
    assert torch.equal(a, b) and torch.equal(sc, sc2)
    a = ops.attn_shared(q, k[0], v[0], k, v, n, 3, 1)
    b = ops.attn_shared(q, k[0], v[0], k, v, n, 3, 1, workspace=ops.attn_shared_workspace(3, 1, 32, 4, D, 300, 300, dev))
    assert torch.equal(a, b)
    a = ops.attn_prefill_scored(q, k[:1], v[:1], sc[:1], 1, 3)
    b = ops.attn_prefill_scored(q, k[:1], v[:1], sc2[:1], 1, 3,
                                workspace=ops.attn_prefill_scored_workspace(1, 3, 32, 4, D, 0, dev))
    assert torch.equal(a, b) and torch.equal(sc, sc2)
    x, y = [t.clone() for t in (k, v, sc, pos)], [t.clone() for t in (k, v, sc, pos)]
    ops.kv_evict(*x, n, 100, 5, 2)
    ops.kv_evict(*y, n, 100, 5, 2, workspace=ops.kv_evict_workspace(3, 4, 300, 100, dev))
    assert all(torch.equal(s, t) for s, t in zip(x, y))


def test_offsets_past_32_bits(dev):
    """Caches of 2^32 elements (8.6 GB): the last row's last head sits behind
    2^31 elements, and the longest run of keys that a call takes is 2^30 bytes.
    The keys of the last group's heads are planted at the far end: a logit of 2
    |q|^2 / sqrt(D) >= 60 against 4 million others of standard deviation 2 (at
    most 14 in all likelihood, together below e^(14 + 16)), so the output is that entry's
    value but for e^-30 and the rounding of its weight and its own."""
    announce("caches past 32-bit offsets")
    B, Hq, Hkv, n = 2, 32, 4, 1 << 22
    if torch.cuda.get_device_properties(dev).total_memory < 64 << 30:
        pytest.skip("needs 40 GB")
    g = _gen(dev, 77)
    k, v = [torch.empty(B, Hkv, n, D, dtype=torch.bfloat16, device=dev).normal_(generator=g) for _ in range(2)]
    q = bf16_randn((1, Hq, D), g, dev, 2.0).expand(B, Hq, D).contiguous()
    assert float((q[0].double() ** 2).sum(1).min()) * 2 * SCALE >= 60
    heads, far = range(Hq - 8, Hq), [n - 40 - 3 * i for i in range(8)]
    for b in range(B):
        k[b, 3, far] = 2 * q[b, Hq - 8:]
    sc = torch.zeros(B, Hkv, n, device=dev)

    def at_far(got, b, what):  # got [8, D]
        want = v[b, 3, far].double()
        _within(got, want, want.abs() * 2 * ref.HALF_BF16 + 1e-9, what)

    out = ops.attn_decode_scored(q, k, v, _i32([n, n - 1], dev), sc).view(B, Hq, D)
    for b in range(B):
        at_far(out[b, heads[0]:], b, f"scored, row {b}")
        assert bool(((sc[b, 3, far].double() - 1).abs() <= 1e-5).all())
    sc.zero_()
    ctx = [300, 257]
    out = ops.attn_decode_scored(q, k, v, _i32(ctx, dev), sc, max_ctx=300).view(B, Hq, D)
    for b, c in enumerate(ctx):
        sees = torch.ones(1, c, dtype=torch.bool, device=dev)
        add, off = 0, 0
        for h in heads:
            o, e, w, rel = ref.attend(q[b, h:h + 1], k[b, 3, :c], v[b, 3, :c], sees, SCALE)
            _within(out[b, h:h + 1], o, e, f"scored {c}, head {h}")
            add, off = add + w[0], off + w[0] * (rel + 64 * ref.F32)
        _within(sc[b, 3, :c], add, off + 1e-30, "scores")
        assert not bool(sc[b, 3, c:].any())
    out = ops.attn_shared(q, k[1], v[1], k, v, _i32([100, 7], dev), B, 1, max_ctx=100).view(B, Hq, D)
    for b in range(B):
        at_far(out[b, heads[0]:], 1, f"prefix, row {b}")
    out = ops.attn_shared(q, k[0, :, :50].contiguous(), v[0, :, :50].contiguous(), k, v, _i32([n, n], dev), B,
                          1).view(B, Hq, D)
    for b in range(B):
        at_far(out[b, heads[0]:], b, f"own entries, row {b}")
    S = 20
    sc.zero_()
    qc = bf16_randn((B * S, Hq, D), g, dev, 2.0).view(B, S, Hq, D)
    qc[:, 7] = q
    out = ops.attn_prefill_scored(qc.view(B * S, Hq, D), k, v, sc, B, S, n - S).view(B, S, Hq, D)
    for b in range(B):
        at_far(out[b, 7, heads[0]:], b, f"chunk, row {b}")
        assert bool((sc[b, 3, far] >= 1 - 1e-5).all())  # and what the other queries gave them
    # append to the last slot, then cut down to the best 1000
    pos = torch.arange(n, dtype=torch.int32, device=dev).repeat(B, Hkv, 1)
    raw = torch.randn(B, (Hq + 2 * Hkv) * D, generator=g, device=dev)
    w, cos = torch.ones(D, dtype=torch.bfloat16, device=dev), torch.ones(8, D // 2, device=dev)
    guard = k[1, 3, n - 2].clone()
    ops.kv_append(raw, w, w, cos, torch.zeros_like(cos), _i32([3, 5], dev), _i32([n - 1, n - 1], dev), Hq, Hkv, k, v,
                  1e-6, scores=sc, slot_pos=pos)
    assert torch.equal(v[:, :, n - 1].reshape(B, -1), raw[:, (Hq + Hkv) * D:].bfloat16())
    assert torch.equal(k[1, 3, n - 2], guard) and pos[:, :, n - 1].tolist() == [[3] * 4, [5] * 4]
    assert not bool(sc[:, :, n - 1].any())
    sc.copy_(torch.rand(B, Hkv, n, generator=g, device=dev))
    keep = sc[1, 3].sort(descending=True, stable=True).indices[:1000].sort().values
    rows = k[1, 3, keep].clone()
    ops.kv_evict(k, v, sc, pos, _i32([n, n], dev), 1000)
    stay = keep < 1000
    order = torch.empty(1000, dtype=torch.long, device=dev)
    hole = torch.ones(1000, dtype=torch.bool, device=dev)
    hole[keep[stay]] = False
    order[keep[stay]] = stay.nonzero()[:, 0]
    order[hole] = (~stay).nonzero()[:, 0]
    assert torch.equal(k[1, 3, :1000], rows[order]) and torch.equal(pos[1, 3, :1000].long(), keep[order])
