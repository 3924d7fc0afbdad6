"""What the operators of a decode batch's cache are measured on: attention over a
prefix that the batch shares, and a cache of bounded size that keeps the
entries with the most accumulated attention weight.

``shared``  attention of a batch whose rows all start with the same long prompt:
            its keys and values are held once, each row has a cache of its own
            for what follows (one query per row for decode, a chunk of queries
            for the rows' prompts);
``prompt``  causal attention of a prompt, which also adds each entry's attention
            weight (over all queries and the query heads of a group) to its score;
``scored``  one decode step of attention that adds the weights to the scores;
``append``  a decode step's raw projection rows to normalised, rotated queries and
            cache rows, in slots that are not the positions;
``evict``   a cache cut down to its budget: the first positions, the most recent
            ones and the entries of the largest scores stay.

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
EPS = 1e-6
THETA = 1e6


def listed():
    return [
        # a few short chats on one system prompt: the smallest call, where latency counts
        {"name": "shared_4x300", "kind": "shared", "batch": 4, "queries": 1, "prefix": 300, "context": 24,
         "hq": 32, "hkv": 4},
        # a decode batch on a long document
        {"name": "shared_32x8192", "kind": "shared", "batch": 32, "queries": 1, "prefix": 8192, "context": 512,
         "hq": 32, "hkv": 4},
        # the rows' own questions after the document, an odd number of tokens
        {"name": "shared_8x101q_2900", "kind": "shared", "batch": 8, "queries": 101, "prefix": 2900, "context": 101,
         "hq": 32, "hkv": 4},
        # the largest decode batch on a very long prefix
        {"name": "shared_64x32768", "kind": "shared", "batch": 64, "queries": 1, "prefix": 32768, "context": 1024,
         "hq": 32, "hkv": 4},
        # a prompt of the usual length
        {"name": "prompt_1x640", "kind": "prompt", "batch": 1, "queries": 640, "start": 0, "hq": 32, "hkv": 4},
        # two long prompts, one of them padded
        {"name": "prompt_2x4096", "kind": "prompt", "batch": 2, "queries": 4096, "start": 0, "hq": 32, "hkv": 4},
        # one sequence on a bounded cache
        {"name": "scored_1x1100", "kind": "scored", "batch": 1, "context": 1100, "hq": 32, "hkv": 4},
        # a batch of different lengths on bounded caches
        {"name": "scored_32x4160", "kind": "scored", "batch": 32, "context": 4160, "hq": 32, "hkv": 4},
        # one row appended, and a batch's
        {"name": "append_1", "kind": "append", "batch": 1, "slots": 1088, "hq": 32, "hkv": 4},
        {"name": "append_64", "kind": "append", "batch": 64, "slots": 576, "hq": 32, "hkv": 4},
        # a prompt's cache cut down into a bounded one
        {"name": "evict_2x4096_to_1024", "kind": "evict", "batch": 2, "context": 4096, "budget": 1024, "recent": 128,
         "sink": 4, "place": "other", "hkv": 4},
        # a decode batch's bounded caches, full again after 64 steps
        {"name": "evict_16x1088_to_1024", "kind": "evict", "batch": 16, "context": 1088, "budget": 1024,
         "recent": 128, "sink": 4, "place": "same", "hkv": 4},
    ]


HEADS = [(32, 4), (32, 4), (32, 4), (16, 4), (32, 8), (64, 4), (8, 8), (12, 4)]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random):
    kind = rng.choice(["shared", "shared", "shared", "prompt", "prompt", "scored", "scored", "append", "evict", "evict"])
    hq, hkv = rng.choice(HEADS)
    if kind == "shared":
        if rng.random() < 0.3:  # a chunk of queries
            batch = _log(rng, 1, 16)
            queries = _log(rng, 2, 512 // batch)
            return {"kind": kind, "batch": batch, "queries": queries, "prefix": _log(rng, 16, 4096),
                    "context": queries + rng.choice([0, 0, rng.randint(0, 300)]), "hq": hq, "hkv": hkv}
        batch = _log(rng, 1, 64)
        return {"kind": kind, "batch": batch, "queries": 1, "prefix": _log(rng, 16, 16384),
                "context": _log(rng, 1, 1024), "hq": hq, "hkv": hkv}
    if kind == "prompt":
        batch = _log(rng, 1, 8)
        return {"kind": kind, "batch": batch, "queries": _log(rng, 2, 2048 // batch),
                "start": rng.choice([0, 0, rng.randint(1, 1024)]), "hq": hq, "hkv": hkv}
    if kind == "scored":
        batch = _log(rng, 1, 64)
        return {"kind": kind, "batch": batch, "context": _log(rng, 1, min(8192, 65536 // batch)), "hq": hq, "hkv": hkv}
    if kind == "append":
        return {"kind": kind, "batch": _log(rng, 1, 64), "slots": _log(rng, 16, 600), "hq": hq, "hkv": hkv}
    context = _log(rng, 64, 8192)
    budget = rng.randint(context // 8, context)
    return {"kind": kind, "batch": _log(rng, 1, max(1, min(64, 32768 // context))), "context": context,
            "budget": budget, "recent": rng.randint(0, budget // 2), "sink": rng.choice([0, 1, 4]),
            "place": rng.choice(["same", "other"]), "hkv": hkv}


# ---------------------------------------------------------------------- inputs
def _spread(n, lo, hi):
    """``n`` lengths from ``lo`` to ``hi``, evenly: the case alone says their sum."""
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _contexts(case):
    """The cache entries that each row's first query sees."""
    if case["kind"] == "shared" and case["queries"] > 1:
        return [case["context"] - case["queries"] + 1] * case["batch"]
    return _spread(case["batch"], max(1, case["context"] // 4), case["context"])


def _lengths(case):
    """The queries of a prompt that are real (the rest is padding on the right)."""
    return _spread(case["batch"], max(1, case["queries"] * 5 // 6), case["queries"])


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, std=1.0, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="cuda").normal_(0.0, std, generator=g)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _weights_so_far(g, *shape):
    """Accumulated attention weights: a few entries hold most of them."""
    return torch.randn(*shape, generator=g, device="cuda").mul_(1.5).exp_()


def prepare(case, seed):
    g = _generator(seed)
    kind, b, hkv = case["kind"], case["batch"], case["hkv"]
    s = dict(case)
    if kind == "shared":
        cap = case["context"] + 64
        s["q"] = _normal(g, b * case["queries"], case["hq"], D, std=2.0)
        s["kp"], s["vp"] = _normal(g, hkv, case["prefix"], D), _normal(g, hkv, case["prefix"], D)
        s["k"], s["v"] = _normal(g, b, hkv, cap, D), _normal(g, b, hkv, cap, D)
        s["ctx"] = _ints(_contexts(case))[torch.randperm(b, generator=g, device="cuda")]
    elif kind == "prompt":
        n = case["start"] + case["queries"]
        s["q"] = _normal(g, b * case["queries"], case["hq"], D, std=2.0)
        s["k"], s["v"] = _normal(g, b, hkv, n + 1, D), _normal(g, b, hkv, n + 1, D)
        s["lengths"] = _ints(_lengths(case))[torch.randperm(b, generator=g, device="cuda")]
        s["scores"] = torch.zeros(b, hkv, n + 1, device="cuda")
        s["scores"][:, :, :case["start"]] = _weights_so_far(g, b, hkv, case["start"])
    elif kind == "scored":
        cap = case["context"] + 17
        s["q"] = _normal(g, b, case["hq"], D, std=2.0)
        s["k"], s["v"] = _normal(g, b, hkv, cap, D), _normal(g, b, hkv, cap, D)
        s["ctx"] = _ints(_contexts(case))[torch.randperm(b, generator=g, device="cuda")]
        s["scores"] = _weights_so_far(g, b, hkv, cap)
    elif kind == "append":
        cap = case["slots"]
        s["qkv"] = _normal(g, b, (case["hq"] + 2 * hkv) * D, std=1.5, dtype=torch.float32)
        s["qn"], s["kn"] = (1.0 + 0.1 * torch.randn(2, D, generator=g, device="cuda")).to(torch.bfloat16)
        inv = THETA ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        angle = torch.arange(8 * cap, dtype=torch.float64, device="cuda")[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        s["slots_of"] = torch.randint(0, cap, (b,), generator=g, device="cuda").int()
        s["positions"] = s["slots_of"] + torch.randint(0, 7 * cap, (b,), generator=g, device="cuda").int()
        s["k"], s["v"] = _normal(g, b, hkv, cap, D), _normal(g, b, hkv, cap, D)
        s["scores"] = _weights_so_far(g, b, hkv, cap)
        s["slot_pos"] = torch.arange(cap, dtype=torch.int32, device="cuda").repeat(b, hkv, 1)
    else:
        cap = case["context"]
        s["k"], s["v"] = _normal(g, b, hkv, cap, D), _normal(g, b, hkv, cap, D)
        s["scores"] = _weights_so_far(g, b, hkv, cap)
        s["ctx"] = _ints(_spread(b, max(1, cap * 3 // 4), cap))
        # a cache that was cut down before holds its positions out of order, and not all of them
        pos = torch.arange(cap, device="cuda").repeat(b, hkv, 1)
        if case["place"] == "same":
            pos = pos * 2 + (torch.rand(b, hkv, cap, generator=g, device="cuda") < 0.5)
            live = torch.arange(cap, device="cuda") < s["ctx"].view(b, 1, 1) - 64
            order = torch.where(live, torch.rand(b, hkv, cap, generator=g, device="cuda"), 2.0 + pos).argsort(-1)
            pos = pos.gather(-1, order)
        s["slot_pos"] = pos.int()
        s["scores"].masked_fill_(torch.arange(cap, device="cuda") >= s["ctx"].view(b, 1, 1), 0.0)
        n = case["budget"] + 64 if case["place"] == "other" else cap
        s["to"] = (torch.zeros(b, hkv, n, D, dtype=torch.bfloat16, device="cuda"),
                   torch.zeros(b, hkv, n, D, dtype=torch.bfloat16, device="cuda"),
                   torch.zeros(b, hkv, n, device="cuda"), torch.zeros(b, hkv, n, dtype=torch.int32, device="cuda"))
    return s


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


def _rows(q, b, s, hkv):
    """Queries [b*s, hq, D] as [b, hkv, s * group, D] in 32 bits."""
    group = q.shape[1] // hkv
    return q.float().view(b, s, hkv, group, D).permute(0, 2, 1, 3, 4).reshape(b, hkv, s * group, D)


def _back(o, b, s, hq):
    """[b, hkv, s * group, D] as bf16 [b*s, hq*D]."""
    hkv = o.shape[1]
    return o.view(b, hkv, s, hq // hkv, D).permute(0, 2, 1, 3, 4).reshape(b * s, hq * D).to(torch.bfloat16)


def _shared(st):
    b, s, hq, hkv = st["batch"], st["queries"], st["hq"], st["hkv"]
    if own:
        return _ops().attn_shared(st["q"], st["kp"], st["vp"], st["k"], st["v"], st["ctx"], b, s,
                                  max_ctx=st["context"])
    q = _rows(st["q"], b, s, hkv) / math.sqrt(D)
    rows, prefix, n = q.shape[2], st["prefix"], st["context"]
    flat = q.permute(1, 0, 2, 3).reshape(hkv, b * rows, D)
    lp = (flat @ st["kp"].float().transpose(1, 2)).view(hkv, b, rows, prefix).permute(1, 0, 2, 3)
    lo = q @ st["k"][:, :, :n].float().transpose(2, 3)
    sees = st["ctx"].view(b, 1) + torch.arange(s, device="cuda").repeat_interleave(rows // s)
    lo = lo.masked_fill(torch.arange(n, device="cuda") >= sees.view(b, 1, rows, 1), -math.inf)
    p = _softmax(torch.cat([lp, lo], -1))
    pp = p[..., :prefix].permute(1, 0, 2, 3).reshape(hkv, b * rows, prefix)
    o = (pp @ st["vp"].float()).view(hkv, b, rows, D).permute(1, 0, 2, 3) + p[..., prefix:] @ st["v"][:, :, :n].float()
    return _back(o, b, s, hq)


def _prompt(st):
    b, s, hq, hkv, start = st["batch"], st["queries"], st["hq"], st["hkv"], st["start"]
    if own:
        out = _ops().attn_prefill_scored(st["q"], st["k"], st["v"], st["scores"], b, s, start, lengths=st["lengths"])
        return out, st["scores"]
    n = start + s
    q = _rows(st["q"], b, s, hkv) / math.sqrt(D)
    at = torch.arange(s, device="cuda").repeat_interleave(hq // hkv)  # the query of each row
    x = q @ st["k"][:, :, :n].float().transpose(2, 3)
    p = _softmax(x.masked_fill_(torch.arange(n, device="cuda") > (start + at).view(-1, 1), -math.inf))
    real = (at < st["lengths"].view(b, 1)).float().view(b, 1, 1, -1)
    st["scores"][:, :, :n] += (real @ p).squeeze(2)
    return _back(p @ st["v"][:, :, :n].float(), b, s, hq), st["scores"]


def _scored(st):
    b, hq, hkv, n = st["batch"], st["hq"], st["hkv"], st["context"]
    if own:
        out = _ops().attn_decode_scored(st["q"], st["k"], st["v"], st["ctx"], st["scores"], max_ctx=n)
        return out, st["scores"]
    q = _rows(st["q"], b, 1, hkv) / math.sqrt(D)
    x = q @ st["k"][:, :, :n].float().transpose(2, 3)
    p = _softmax(x.masked_fill(torch.arange(n, device="cuda") >= st["ctx"].view(b, 1, 1, 1), -math.inf))
    st["scores"][:, :, :n] += p.sum(2)
    return _back(p @ st["v"][:, :, :n].float(), b, 1, hq), st["scores"]


def _append(st):
    b, hq, hkv = st["batch"], st["hq"], st["hkv"]
    if own:
        q = _ops().kv_append(st["qkv"], st["qn"], st["kn"], st["cos"], st["sin"], st["positions"], st["slots_of"],
                             hq, hkv, st["k"], st["v"], EPS, scores=st["scores"], slot_pos=st["slot_pos"])
        return q, st["k"], st["v"], st["scores"], st["slot_pos"]
    x = st["qkv"].view(b, hq + 2 * hkv, D)
    qk, v = x[:, :hq + hkv], x[:, hq + hkv:]
    qk = qk * torch.rsqrt(qk.square().mean(-1, keepdim=True) + EPS)
    qk = torch.cat([qk[:, :hq] * st["qn"].float(), qk[:, hq:] * st["kn"].float()], 1)
    pos, slot, row = st["positions"].long(), st["slots_of"].long(), torch.arange(b, device="cuda")
    c, sn = st["cos"][pos].unsqueeze(1), st["sin"][pos].unsqueeze(1)
    lo, hi = qk[..., :D // 2], qk[..., D // 2:]
    qk = torch.cat([lo * c - hi * sn, hi * c + lo * sn], -1).to(torch.bfloat16)
    st["k"][row, :, slot] = qk[:, hq:]
    st["v"][row, :, slot] = v.to(torch.bfloat16)
    st["scores"][row, :, slot] = 0.0
    st["slot_pos"][row, :, slot] = st["positions"].view(b, 1).expand(b, hkv)
    return qk[:, :hq].contiguous(), st["k"], st["v"], st["scores"], st["slot_pos"]


def _evict(st):
    b, hkv, budget = st["batch"], st["hkv"], st["budget"]
    k2, v2, sc2, pos2 = st["to"]
    if st["place"] == "same":  # the cache as it stands before the call: the call changes it
        for to, x in zip(st["to"], (st["k"], st["v"], st["scores"], st["slot_pos"])):
            to.copy_(x)
    if own:
        if st["place"] == "same":
            _ops().kv_evict(k2, v2, sc2, pos2, st["ctx"], budget, recent=st["recent"], sink=st["sink"])
        else:
            _ops().kv_evict(st["k"], st["v"], st["scores"], st["slot_pos"], st["ctx"], budget, recent=st["recent"],
                            sink=st["sink"], out=st["to"])
        return k2, v2, sc2, pos2
    n = st["context"]
    slot = torch.arange(n, device="cuda")
    live = slot < st["ctx"].view(b, 1, 1)
    pos = torch.where(live, st["slot_pos"].long(), -1)
    held = live & ((pos > pos.amax(-1, keepdim=True) - st["recent"]) | (pos < st["sink"]))
    rank = torch.where(held, math.inf, st["scores"]).masked_fill(~live, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :budget]
    keep = torch.zeros(b, hkv, n, dtype=torch.bool, device="cuda").scatter_(-1, order, True) & live
    hole = (live & ~keep)[..., :budget]
    movers = torch.sort((keep & (slot >= budget)).int(), dim=-1, descending=True, stable=True).indices
    src = torch.where(hole, movers.gather(-1, (hole.cumsum(-1) - 1).clamp_min(0)), slot[:budget])
    kept = live[..., :budget]
    src4, kept4 = src.unsqueeze(-1).expand(b, hkv, budget, D), kept.unsqueeze(-1)
    new = [torch.where(kept4, x.gather(2, src4), to[:, :, :budget]) for x, to in ((st["k"], k2), (st["v"], v2))]
    new_sc, new_pos = st["scores"].gather(-1, src), st["slot_pos"].gather(-1, src)
    k2[:, :, :budget], v2[:, :, :budget] = new[0], new[1]
    sc2.zero_()
    pos2.fill_(-1)
    sc2[:, :, :budget] = torch.where(kept, new_sc, 0.0)
    pos2[:, :, :budget] = torch.where(kept, new_pos, -1)
    return k2, v2, sc2, pos2


_RUN = {"shared": _shared, "prompt": _prompt, "scored": _scored, "append": _append, "evict": _evict}


# ---------------------------------------------------------------------- floors
def work(case):
    kind, b, hkv = case["kind"], case["batch"], case["hkv"]
    entry = 2 * D * 2  # a key and a value of one head
    if kind == "shared":
        s, hq, p = case["queries"], case["hq"], case["prefix"]
        seen = sum(c * s + s * (s - 1) // 2 for c in _contexts(case))
        held = sum(c + s - 1 for c in _contexts(case))
        return {"bytes": (p + held) * hkv * entry + 2 * b * s * hq * D * 2 + 4 * b,
                "flops": 4 * D * hq * (b * s * p + seen)}
    if kind == "prompt":
        s, hq, start = case["queries"], case["hq"], case["start"]
        seen = b * (s * start + s * (s + 1) // 2)
        return {"bytes": b * (start + s) * hkv * (entry + 8) + 2 * b * s * hq * D * 2,
                "flops": 4 * D * hq * seen}
    if kind == "scored":
        n = sum(_contexts(case))
        return {"bytes": n * hkv * (entry + 8) + 2 * b * case["hq"] * D * 2, "flops": 4 * D * case["hq"] * n}
    if kind == "append":
        heads = case["hq"] + 2 * hkv
        return {"bytes": b * heads * D * (4 + 2) + b * (D * 4 + hkv * 8), "flops": b * heads * D * 8}
    live, budget = _spread(b, max(1, case["context"] * 3 // 4), case["context"]), case["budget"]
    looked_at = hkv * sum(live) * 8  # the scores and positions
    if case["place"] == "same":  # with the copy that the pass starts from; then at most what is past the budget moves
        copied = hkv * b * case["context"] * 2 * (entry + 8)
        moved = hkv * sum(min(budget, max(0, c - budget)) for c in live) * 2 * (entry + 8)
        return {"bytes": looked_at + copied + moved, "flops": hkv * sum(live)}
    kept = hkv * sum(min(c, budget) for c in live) * 2 * (entry + 8)
    return {"bytes": looked_at + kept, "flops": hkv * sum(live)}


# ---------------------------------------------------------------------- in 64 bits
def _attend64(q, keys, values, sees):
    """q [rows, D], keys and values [n, D], sees [rows, n]: outputs and weights."""
    x = (q.double() @ keys.double().t()) / math.sqrt(D)
    e = torch.where(sees, torch.exp(x - x.amax(1, keepdim=True)), torch.zeros((), dtype=torch.float64, device="cuda"))
    total = e.sum(1, keepdim=True)
    w = torch.where(total > 0, e / total, torch.zeros_like(e))
    return w @ values.double(), w


def exact(case, seed):
    st = prepare(case, seed)
    kind, b, hkv = case["kind"], case["batch"], case["hkv"]
    if kind in ("shared", "prompt", "scored"):
        hq, s = case["hq"], case.get("queries", 1)
        group = hq // hkv
        q = st["q"].view(b, s, hq, D)
        out = torch.empty(b, s, hq, D, dtype=torch.float64, device="cuda")
        total = st["scores"].double() if "scores" in st else None
        for i in range(b):
            n = case["context"] if kind != "prompt" else case["start"] + s
            entry, query = torch.arange(n, device="cuda").view(1, n), torch.arange(s, device="cuda").view(s, 1)
            first = case["start"] + 1 if kind == "prompt" else int(st["ctx"][i])
            sees = (entry < first + query).expand(s, n)
            if kind == "shared":
                sees = torch.cat([torch.ones(s, case["prefix"], dtype=torch.bool, device="cuda"), sees], 1)
            for h in range(hkv):
                keys, values = st["k"][i, h, :n], st["v"][i, h, :n]
                if kind == "shared":
                    keys, values = torch.cat([st["kp"][h], keys]), torch.cat([st["vp"][h], values])
                for j in range(h * group, (h + 1) * group):
                    out[i, :, j], w = _attend64(q[i, :, j], keys, values, sees)
                    if kind == "prompt":
                        total[i, h, :n] += w[:int(st["lengths"][i])].sum(0)
                    elif kind == "scored":
                        total[i, h, :n] += w.sum(0)
        out = out.view(b * s, hq * D)
        return out if kind == "shared" else (out, total)
    if kind == "append":
        hq = case["hq"]
        rows = st["qkv"].double().view(b, hq + 2 * hkv, D)
        k, v = st["k"].double(), st["v"].double()
        q = torch.empty(b, hq, D, dtype=torch.float64, device="cuda")
        for i in range(b):
            p, at = int(st["positions"][i]), int(st["slots_of"][i])
            turn = torch.complex(st["cos"][p].double(), st["sin"][p].double())
            for j in range(hq + hkv):
                weight = (st["qn"] if j < hq else st["kn"]).double()
                x = rows[i, j] / torch.sqrt((rows[i, j] ** 2).sum() / D + EPS) * weight
                z = torch.complex(x[:D // 2], x[D // 2:]) * turn
                if j < hq:
                    q[i, j] = torch.cat([z.real, z.imag])
                else:
                    k[i, j - hq, at] = torch.cat([z.real, z.imag])
            v[i, :, at] = rows[i, hq + hkv:]
            st["scores"][i, :, at] = 0
        return q, k, v, st["scores"].double(), None
    return None  # what eviction returns is copied, not computed
