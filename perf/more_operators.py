"""What the operators of long contexts are measured on: attention with a sliding
window and a few first tokens that stay visible, and a key/value cache held in 4
bits.

``window``  attention in which a query sees the last ``window`` entries up to its own
            and the first ``sink`` ones (one query a row for decode, a chunk of
            them for prompts);
``attend4`` attention over a cache held in 4 bits, with a window or without one;
``store4``  a prompt's keys and values into the 4-bit cache and the cache back as the
            values it stands for;
``append4`` a decode step's raw projection rows to normalised, rotated queries and
            4-bit entries, and the cache back as values.

An entry of the 4-bit cache is a row of 128 e2m1 numbers (0, 0.5, 1, 1.5, 2, 3, 4, 6
and their negatives; two a byte, the even element in the low half) with a power of
two for every 32 of them (a byte, biased by 127).  The power is the smallest whose
seventh multiple is above the block's largest magnitude (within 2^-120 .. 2^125);
elements round to the nearest number, ties to the even code, and what is past 6 to 6.

Head layouts are those of Qwen3-30B-A3B (32 query and 4 key/value heads of 128),
and in the drawn cases others of the same head size.
"""

import math
import os
import random
import sys

import torch

own = False

D = 128
BLOCK = 32  # elements that share a power of two
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # one sequence past its window: a decode step where latency counts
        {"name": "window_1x1100", "kind": "window", "batch": 1, "queries": 1, "context": 1100, "window": 512,
         "sink": 4, "hq": 32, "hkv": 4},
        # a decode batch of different lengths, most of them far past the window
        {"name": "window_32x16384", "kind": "window", "batch": 32, "queries": 1, "context": 16384, "window": 4096,
         "sink": 4, "hq": 32, "hkv": 4},
        # a prompt of the usual length, an odd window
        {"name": "window_prompt_1x640", "kind": "window", "batch": 1, "queries": 640, "context": 640, "window": 250,
         "sink": 4, "hq": 32, "hkv": 4},
        # long prompts
        {"name": "window_prompt_2x8192", "kind": "window", "batch": 2, "queries": 8192, "context": 8192,
         "window": 1024, "sink": 4, "hq": 32, "hkv": 4},
        # one sequence shortly after its prompt on a 4-bit cache: the smallest call
        {"name": "attend4_1x800", "kind": "attend4", "batch": 1, "queries": 1, "context": 800, "window": 0, "sink": 0,
         "hq": 32, "hkv": 4},
        # a batch of different lengths
        {"name": "attend4_32x8192", "kind": "attend4", "batch": 32, "queries": 1, "context": 8192, "window": 0,
         "sink": 0, "hq": 32, "hkv": 4},
        # what 4 bits are for: the largest batch on long contexts
        {"name": "attend4_64x32768", "kind": "attend4", "batch": 64, "queries": 1, "context": 32768, "window": 0,
         "sink": 0, "hq": 32, "hkv": 4},
        # the next turn of a few conversations, an odd number of tokens on 4-bit caches
        {"name": "attend4_4x301q_2900", "kind": "attend4", "batch": 4, "queries": 301, "context": 2900, "window": 0,
         "sink": 0, "hq": 32, "hkv": 4},
        # a prompt of the usual length, and two long ones, into the cache
        {"name": "store4_1x640", "kind": "store4", "batch": 1, "queries": 640, "slots": 700, "hkv": 4},
        {"name": "store4_2x8192", "kind": "store4", "batch": 2, "queries": 8192, "slots": 8256, "hkv": 4},
        # one row appended, and a batch's
        {"name": "append4_1", "kind": "append4", "batch": 1, "queries": 1, "slots": 64, "hq": 32, "hkv": 4},
        {"name": "append4_64", "kind": "append4", "batch": 64, "queries": 1, "slots": 40, "hq": 32, "hkv": 4},
    ]


HEADS = [(32, 4), (32, 4), (32, 4), (16, 4), (32, 8), (64, 4), (8, 8), (12, 4)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(["window", "window", "window", "attend4", "attend4", "attend4", "store4", "append4"])
    hq, hkv = rng.choice(HEADS)
    if kind == "store4":
        batch = _log(rng, 1, 16)
        queries = _log(rng, 1, 8192 // batch)
        return {"kind": kind, "batch": batch, "queries": queries, "slots": queries + rng.randint(0, 200), "hkv": hkv}
    if kind == "append4":
        return {"kind": kind, "batch": _log(rng, 1, 64), "queries": rng.choice([1, 1, 1, rng.randint(2, 5)]),
                "slots": rng.randint(8, 60), "hq": hq, "hkv": hkv}
    window, sink = _log(rng, 1, 4096), rng.choice([0, 1, 4, 4, rng.randint(5, 100)])
    if kind == "attend4" and rng.random() < 0.7:
        window = sink = 0
    if rng.random() < 0.4:  # a chunk of queries
        batch = _log(rng, 1, 8)
        queries = _log(rng, 2, (2048 if kind == "window" else 512) // batch)
        context = queries + rng.choice([0, rng.randint(0, 2000)])
    else:
        batch, queries = _log(rng, 1, 64), 1
        context = _log(rng, 1, min(32768, 262144 // batch))
    return {"kind": kind, "batch": batch, "queries": queries, "context": context, "window": window, "sink": sink,
            "hq": hq, "hkv": hkv}


# ---------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """``n`` lengths from ``lo`` to ``hi``, evenly: the case alone says their sum."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _contexts(case):
    """The cache entries up to each row's first query, its own included."""
    if case["queries"] > 1:
        return [case["context"] - case["queries"] + 1] * case["batch"]
    return _spread(case["batch"], max(1, case["context"] // 4), case["context"])


def _lengths(case):
    """The tokens of each row's prompt that are real (the rest is padding on the right)."""
    return _spread(case["batch"], max(1, case["queries"] * 5 // 6), case["queries"])


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _cache4(g, b, hkv, n):
    """(K, K's powers, V, V's powers) of normal entries, a row of the batch at a time."""
    cache = [torch.empty(b, hkv, n, w, dtype=torch.uint8, device="cuda") for w in (D // 2, D // BLOCK) * 2]
    for i in range(b):
        for j in (0, 2):
            cache[j][i], cache[j + 1][i] = _quantise(_normal(g, hkv, n, D).float())
    return tuple(cache)


def prepare(case, seed):
    g = _generator(seed)
    kind, b, hkv = case["kind"], case["batch"], case["hkv"]
    s = dict(case)
    if kind in ("window", "attend4"):
        cap = case["context"] + 17
        s["q"] = _normal(g, b * case["queries"], case["hq"], D, std=2.0)
        if kind == "window":
            s["k"], s["v"] = _normal(g, b, hkv, cap, D), _normal(g, b, hkv, cap, D)
        else:
            s["cache"] = _cache4(g, b, hkv, cap)
        s["ctx"] = _ints(_contexts(case))[torch.randperm(b, generator=g, device="cuda")]
        return s
    cap = case["slots"]
    s["cache"] = _cache4(g, b, hkv, cap)
    if kind == "store4":
        s["k"], s["v"] = _normal(g, b, hkv, case["queries"], D), _normal(g, b, hkv, case["queries"], D)
        s["lengths"] = _ints(_lengths(case))[torch.randperm(b, generator=g, device="cuda")]
        s["starts"] = torch.randint(0, cap - case["queries"] + 1, (b,), generator=g, device="cuda").int()
        return s
    n = case["queries"]
    s["qkv"] = _normal(g, b * n, (case["hq"] + 2 * hkv) * D, std=1.5, dtype=torch.float32)
    s["qn"], s["kn"] = (1.0 + 0.1 * torch.randn(2, D, generator=g, device="cuda")).to(torch.bfloat16)
    inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
    angle = torch.arange(64 * cap, dtype=torch.float64, device="cuda")[:, None] * inv
    s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
    first = torch.randint(0, cap - n + 1, (b, 1), generator=g, device="cuda")
    s["slots_of"] = (first + torch.arange(n, device="cuda")).int().view(-1)
    s["positions"] = s["slots_of"] + torch.randint(0, 63 * cap, (b, 1), generator=g,
                                                   device="cuda").expand(b, n).reshape(-1).int()
    return s


# ---------------------------------------------------------------------- 4 bits
_NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _quantise(x):
    """``x[..., D]`` in 32 or 64 bits -> codes and powers."""
    x = x.view(*x.shape[:-1], D // BLOCK, BLOCK)
    m, e = torch.frexp(x.abs().amax(-1))  # the largest is m * 2^e, 0.5 <= m < 1
    power = (e + (m >= 0.875) + (127 - 3)).masked_fill(m == 0, 0).clamp(7, 252)
    if x.dtype == torch.float64:
        inverse = ((1023 + 127 - power.long()) << 52).view(torch.float64)
    else:
        inverse = ((254 - power.int()) << 23).view(torch.float32)
    y = x.abs() * inverse.unsqueeze(-1)
    code = (y > 0.25).byte()
    for below, border in ((False, 0.75), (True, 1.25), (False, 1.75), (True, 2.5), (False, 3.5), (True, 5.0)):
        code += (y > border) if below else (y >= border)
    code = (code + 8 * torch.signbit(x).byte()).flatten(-2)
    return code[..., 0::2] + 16 * code[..., 1::2], power.byte()


def _values(codes, powers):
    """What codes and powers stand for, in 32 bits."""
    table = torch.tensor(_NUMBERS + [-x for x in _NUMBERS], device="cuda")
    x = torch.stack([table[(codes & 15).int()], table[(codes >> 4).int()]], -1).view(*codes.shape[:-1], D // BLOCK, BLOCK)
    return (x * (powers.int() << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)


# ---------------------------------------------------------------------- one pass
def run(state):
    return _RUN[state["kind"]](state)


def _ops():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "nki-moe-7013_amd")
    if at not in sys.path:
        sys.path.insert(0, at)
    from qmoe import ops

    return ops


def _softmax(x):
    """Weights over the last axis; a row of -inf alone has none."""
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return p / torch.where(total > 0, total, torch.ones_like(total))


def _sees(at, entry, window, sink):
    """Whether the query at index ``at`` sees ``entry``."""
    return (entry <= at) & ((entry > at - (window or 1 << 30)) | (entry < sink))


def _attend(q, k, v, at, entry, st):
    """Queries [b*s, hq, D] at indices ``at[b, s]`` over k, v [b, hkv, n, D] in 32 bits,
    which hold the cache's entries ``entry[b or 1, n]``."""
    b, s = at.shape
    hq, hkv = q.shape[1], k.shape[1]
    group = hq // hkv
    x = q.float().view(b, s, hkv, group, D).permute(0, 2, 1, 3, 4).reshape(b, hkv, s * group, D) / math.sqrt(D)
    sees = _sees(at.unsqueeze(2), entry.unsqueeze(1), st["window"], st["sink"]).repeat_interleave(group, 1)
    p = _softmax((x @ k.transpose(2, 3)).masked_fill_(~sees.unsqueeze(1), -math.inf))
    o = (p @ v).view(b, hkv, s, group, D).permute(0, 2, 1, 3, 4)
    return o.reshape(b * s, hq * D).to(torch.bfloat16)


def _window(st):
    b, s, n = st["batch"], st["queries"], st["context"]
    if own:
        return _ops().attn_window(st["q"], st["k"], st["v"], st["ctx"], b, s, st["window"], st["sink"], max_ctx=n)
    at = st["ctx"].view(b, 1) - 1 + torch.arange(s, device="cuda")
    seen = min(n, st["window"] + st["sink"])
    if s > 1 or seen == n:
        return _attend(st["q"], st["k"][:, :, :n].float(), st["v"][:, :, :n].float(), at,
                       torch.arange(n, device="cuda").view(1, n), st)
    # the entries that a row's one query sees: the first ones and the window's
    entry = torch.arange(seen, device="cuda").view(1, seen)
    entry = torch.where(entry < st["sink"], entry, entry + (at - (seen - 1)).clamp_min(0))
    index = entry.view(b, 1, seen, 1).expand(b, st["hkv"], seen, D)
    return _attend(st["q"], st["k"].gather(2, index).float(), st["v"].gather(2, index).float(), at, entry, st)


def _attend4(st):
    b, s, n = st["batch"], st["queries"], st["context"]
    if own:
        return _ops().attn_kv4(st["q"], st["cache"], st["ctx"], b, s, st["window"], st["sink"], max_ctx=n)
    at = st["ctx"].view(b, 1) - 1 + torch.arange(s, device="cuda")
    entry = torch.arange(n, device="cuda").view(1, n)
    step = max(1, (1 << 27) // (n * st["hkv"] * D))  # rows of the batch at a time: their values in 32 bits
    q = st["q"].view(b, s, -1, D)
    out = []
    for i in range(0, b, step):
        k4, ks, v4, vs = (t[i:i + step, :, :n] for t in st["cache"])
        out.append(_attend(q[i:i + step].flatten(0, 1), _values(k4, ks), _values(v4, vs), at[i:i + step], entry, st))
    return torch.cat(out)


def _store4(st):
    b, n, cap = st["batch"], st["queries"], st["slots"]
    if own:
        _ops().kv4_store(st["k"], st["v"], st["cache"], starts=st["starts"], lengths=st["lengths"])
        return _ops().kv4_load(st["cache"])
    to = torch.arange(cap, device="cuda").view(1, cap) - st["starts"].view(b, 1)  # the token of each entry
    new = ((to >= 0) & (to < st["lengths"].view(b, 1))).view(b, 1, cap, 1)
    index = to.clamp(0, n - 1).view(b, 1, cap, 1)
    out = []
    for x, codes, powers in zip((st["k"], st["v"]), st["cache"][0::2], st["cache"][1::2]):
        for t, made in zip((codes, powers), _quantise(x.float())):
            t.copy_(torch.where(new, made.gather(2, index.expand(*t.shape)), t))
        out.append(_values(codes, powers).to(torch.bfloat16))
    return tuple(out)


def _append4(st):
    b, s, hq, hkv = st["batch"], st["queries"], st["hq"], st["hkv"]
    if own:
        q = _ops().kv4_append(st["qkv"], st["qn"], st["kn"], st["cos"], st["sin"], st["positions"], st["slots_of"],
                              hq, hkv, st["cache"], EPS, S=s)
        return (q, *_ops().kv4_load(st["cache"]))
    # in 64 bits: a key next to a border of two numbers goes to the right one
    x = st["qkv"].view(b * s, hq + 2 * hkv, D).double()
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    qk = qk / torch.sqrt(qk.square().mean(-1, keepdim=True) + EPS)
    qk = torch.cat([qk[:, :hq] * st["qn"].double(), qk[:, hq:] * st["kn"].double()], 1)
    pos, slot = st["positions"].long(), st["slots_of"].long()
    row = torch.arange(b, device="cuda").repeat_interleave(s)
    c, sn = st["cos"][pos].double().unsqueeze(1), st["sin"][pos].double().unsqueeze(1)
    lo, hi = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1)
    out = [qk[:, :hq].to(torch.bfloat16)]
    for made, codes, powers in zip((qk[:, hq:], v), st["cache"][0::2], st["cache"][1::2]):
        codes[row, :, slot], powers[row, :, slot] = _quantise(made.contiguous())
        out.append(_values(codes, powers).to(torch.bfloat16))
    return tuple(out)


_RUN = {"window": _window, "attend4": _attend4, "store4": _store4, "append4": _append4}


# ---------------------------------------------------------------------- floors
def _counts(case):
    """Entries that are read, and (query, entry) pairs, of all rows together."""
    s, window, sink = case["queries"], case["window"] or 1 << 30, case["sink"]
    read = pairs = 0
    for c in _contexts(case):
        first = max(c - window, 0)  # of the first query's window
        read += c + s - 1 - first + min(sink, first)
        for i in range(s):
            n = c + i
            low = max(n - window, 0)
            pairs += n - low + min(sink, low)
    return read, pairs


def work(case):
    kind, b, hkv = case["kind"], case["batch"], case["hkv"]
    entry, entry4 = 2 * D * 2, 2 * (D // 2 + D // BLOCK)  # a key and a value of one head
    if kind in ("window", "attend4"):
        read, pairs = _counts(case)
        rows = b * case["queries"] * case["hq"]
        return {"bytes": read * hkv * (entry if kind == "window" else entry4) + 2 * rows * D * 2 + 4 * b,
                "flops": 4 * D * case["hq"] * pairs}
    held = b * hkv * case["slots"]
    if kind == "store4":
        new = hkv * sum(_lengths(case))
        return {"bytes": new * (entry + entry4) + (held - new) * entry4 + held * entry, "flops": 10 * new * 2 * D}
    rows = b * case["queries"]
    new = rows * hkv
    return {"bytes": rows * ((case["hq"] + 2 * hkv) * D * 4 + D * 4 + case["hq"] * D * 2) + new * entry4 +
            (held - new) * entry4 + held * entry, "flops": rows * (case["hq"] + 2 * hkv) * D * 8}


# ---------------------------------------------------------------------- in 64 bits
def _nearest64(x):
    """The numbers that ``x[..., D]`` in 64 bits is held as."""
    x = x.view(*x.shape[:-1], D // BLOCK, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    power = torch.full_like(top, 2.0 ** -120)
    while bool((grow := (top >= 7 * power) & (power < 2.0 ** 125)).any()):
        power = torch.where(grow, power * 2, power)
    y = x.abs() / power
    step = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    y = (torch.round(y / step) * step).clamp_max(6.0)  # ties to the even multiple
    return (torch.copysign(y, x) * power).flatten(-2)


def _held64(codes, powers):
    """What a cache's bytes stand for."""
    numbers = torch.tensor(_NUMBERS, dtype=torch.float64, device="cuda")
    four = torch.stack([codes.long() % 16, codes.long() // 16], -1).flatten(-2)
    x = numbers[four % 8] * torch.where(four >= 8, -1.0, 1.0)
    return x * torch.pow(2.0, powers.double() - 127.0).repeat_interleave(BLOCK, -1)


def exact(case, seed):
    st = prepare(case, seed)
    kind, b, hkv = case["kind"], case["batch"], case["hkv"]
    if kind in ("window", "attend4"):
        hq, s, n = case["hq"], case["queries"], case["context"]
        group, window = hq // hkv, case["window"] or 1 << 30
        q = st["q"].view(b, s, hkv, group, D)
        out = torch.empty(b, s, hkv, group, D, dtype=torch.float64, device="cuda")
        part = max(1, (1 << 26) // (group * n))  # queries at a time
        for i in range(b):
            for h in range(hkv):
                if kind == "window":
                    keys, values = st["k"][i, h, :n].double(), st["v"][i, h, :n].double()
                else:
                    k4, ks, v4, vs = (t[i, h, :n] for t in st["cache"])
                    keys, values = _held64(k4, ks), _held64(v4, vs)
                for s0 in range(0, s, part):
                    rows = q[i, s0:s0 + part, h].double()
                    at = int(st["ctx"][i]) - 1 + s0 + torch.arange(rows.shape[0], device="cuda").view(-1, 1, 1)
                    back = at - torch.arange(n, device="cuda")  # how far an entry lies behind the query
                    sees = (back >= 0) & ((back < window) | (at - back < case["sink"]))
                    x = (rows.reshape(-1, D) @ keys.t()).view(-1, group, n) / math.sqrt(D)
                    x = torch.where(sees, x, -math.inf)
                    e = torch.exp(x - x.amax(-1, keepdim=True))
                    e = e / e.sum(-1, keepdim=True)
                    out[i, s0:s0 + part, h] = (e.view(-1, n) @ values).view(-1, group, D)
        return out.view(b * s, hq * D)
    held = [_held64(*st["cache"][:2]), _held64(*st["cache"][2:])]
    if kind == "store4":
        for i in range(b):
            at, n = int(st["starts"][i]), int(st["lengths"][i])
            for x, to in zip((st["k"], st["v"]), held):
                to[i, :, at:at + n] = _nearest64(x[i, :, :n].double())
        return tuple(held)
    hq, s = case["hq"], case["queries"]
    rows = st["qkv"].double().view(b * s, hq + 2 * hkv, D)
    q = torch.empty(b * s, hq, D, dtype=torch.float64, device="cuda")
    for r in range(b * s):
        p, at = int(st["positions"][r]), int(st["slots_of"][r])
        turn = torch.complex(st["cos"][p].double(), st["sin"][p].double())
        weight = torch.cat([st["qn"].double().expand(hq, D), st["kn"].double().expand(hkv, D)])
        x = rows[r, :hq + hkv]
        x = x * ((x * x).sum(-1, keepdim=True) / D + EPS) ** -0.5 * weight
        z = torch.complex(x[:, :D // 2], x[:, D // 2:]) * turn
        x = torch.cat([z.real, z.imag], -1)
        q[r] = x[:hq]
        held[0][r // s, :, at] = _nearest64(x[hq:].contiguous())
        held[1][r // s, :, at] = _nearest64(rows[r, hq + hkv:].contiguous())
    return (q, *held)
