"""Plain 64-bit forms of the shared-prefix and bounded-cache operators, with the
error that their kernels' roundings allow."""

import math

import torch

D = 128
HALF_BF16 = torch.finfo(torch.bfloat16).eps / 2  # a rounding to bf16 is off by at most this, relative
F32 = 2.0 ** -24


def weights(q, keys, sees, scale):
    """Softmax weights ``[rows, n]`` of ``q[rows, D]`` over ``keys[n, D]`` where
    ``sees[rows, n]``, and the largest sum of |q_i k_i| * scale a row meets."""
    q, keys = q.double(), torch.where(sees.any(0)[:, None], keys.double(), 0.0)
    x = (q @ keys.t()) * scale
    x = torch.where(sees, x, torch.full_like(x, -math.inf))
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = e.sum(1, keepdim=True)
    mag = torch.where(sees, (q.abs() @ keys.abs().t()) * scale, 0.0).amax(1)
    return torch.where(total > 0, e / total, torch.zeros_like(e)), mag


def attend(q, keys, values, sees, scale):
    """Outputs ``[rows, D]``, the bound on a kernel's error in each, the weights
    and the bound on each weight's relative error ``[rows]``.

    A logit is a sum of 128 products in 32 bits: 128 * 2^-24 of the sum of the
    magnitudes; it enters a weight twice (numerator and row sum).  Exponentials,
    the row sum of n terms and the joins add up to (n + 64) * 2^-24, and 2^-20 for
    the exponential of a difference rounded at up to 16 log2 units.  The
    weights are rounded to bf16 once for the product with V, the result once
    for the output."""
    w, mag = weights(q, keys, sees, scale)
    values = torch.where(sees.any(0)[:, None], values.double(), 0.0)
    rel = 2 * D * F32 * mag + (keys.shape[0] + 64) * F32 + 2.0 ** -20
    size = w @ values.abs()
    bound = size * (rel[:, None] + HALF_BF16 * (1 + HALF_BF16)) + (w @ values).abs() * HALF_BF16
    return w @ values, bound + 1e-30, w, rel


def sees_first(counts, n):
    """``[rows, n]``: row r sees the first counts[r] of n entries."""
    return torch.arange(n, device=counts.device).view(1, n) < counts.view(-1, 1)


def shared(q, kp, vp, k, v, ctx, B, S, P, max_ctx, scale):
    """(outputs, bounds) ``[B*S, Hq*D]`` of the shared-prefix attention."""
    Hq, Hkv = q.shape[1], k.shape[1]
    G = Hq // Hkv
    out = torch.zeros(B * S, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, 1e-30)
    for b in range(B):
        counts = (int(ctx[b]) + torch.arange(S, device=q.device)).clamp(0, min(max_ctx, k.shape[2]))
        own = sees_first(counts, max(int(counts.max()), 0))
        sees = torch.cat([torch.ones(S, P, dtype=torch.bool, device=q.device), own], 1)
        for h in range(Hq):
            keys = torch.cat([kp[h // G, :P], k[b, h // G, :own.shape[1]]])
            vals = torch.cat([vp[h // G, :P], v[b, h // G, :own.shape[1]]])
            if keys.shape[0] == 0:
                continue
            o, e, _, _ = attend(q[b * S:(b + 1) * S, h], keys, vals, sees, scale)
            out[b * S:(b + 1) * S, h], bound[b * S:(b + 1) * S, h] = o, e
    return out.view(B * S, Hq * D), bound.view(B * S, Hq * D)


def scored(q, k, v, first, B, S, lengths, scale):
    """Causal or decode attention with accumulated weights: query s of row b sees
    ``first[b] + s`` entries.  (outputs, bounds, added scores, their bounds)."""
    Hq, Hkv, n_max = q.shape[1], k.shape[1], k.shape[2]
    G = Hq // Hkv
    out = torch.zeros(B * S, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, 1e-30)
    add = torch.zeros(B, Hkv, n_max, dtype=torch.float64, device=q.device)
    off = torch.full_like(add, 1e-30)
    for b in range(B):
        counts = (int(first[b]) + torch.arange(S, device=q.device)).clamp(0, n_max)
        n = int(counts.max())
        if n == 0:
            continue
        sees = sees_first(counts, n)
        for h in range(Hq):
            o, e, w, rel = attend(q[b * S:(b + 1) * S, h], k[b, h // G, :n], v[b, h // G, :n], sees, scale)
            out[b * S:(b + 1) * S, h], bound[b * S:(b + 1) * S, h] = o, e
            real = int(lengths[b]) if lengths is not None else S
            # the sum over the rows is in 32 bits too
            add[b, h // G, :n] += w[:real].sum(0)
            off[b, h // G, :n] += (w[:real] * (rel[:real, None] + (S * G + 64) * F32)).sum(0)
    return out.view(B * S, Hq * D), bound.view(B * S, Hq * D), add, off + 1e-30


def evict(k, v, scores, pos, ctx, budget, recent, sink, to=None):
    """Lists, one (row, head) at a time: the slots of the cache after eviction."""
    B, Hkv, S_max, _ = k.shape
    k2, v2, sc2, sp2 = [t.clone() for t in (to if to is not None else (k, v, scores, pos))]
    for b in range(B):
        n = min(max(int(ctx[b]), 0), S_max)
        for h in range(Hkv):
            p, s = pos[b, h].tolist(), scores[b, h].tolist()

            def rank(i):
                held = p[i] < sink or p[i] > max(p[:n]) - recent
                nan = s[i] != s[i]
                return (0 if held else 1, 0 if nan else 1, 0.0 if held or nan else -s[i], i)

            kept = sorted(sorted(range(n), key=rank)[:budget])
            stay = {i for i in kept if i < budget}
            holes = [i for i in range(min(n, budget)) if i not in stay]
            src = {i: i for i in stay}
            src.update(zip(holes, [i for i in kept if i >= budget]))
            for i, j in src.items():
                k2[b, h, i], v2[b, h, i] = k[b, h, j], v[b, h, j]
                sc2[b, h, i], sp2[b, h, i] = scores[b, h, j], pos[b, h, j]
            sc2[b, h, len(src):] = 0.0
            sp2[b, h, len(src):] = -1
    return k2, v2, sc2, sp2
