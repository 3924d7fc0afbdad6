"""Plain 64-bit forms of the windowed attention and of the cache in 4 bits, with the
error that their kernels' roundings allow."""

import math

import torch

import cache_ref

D = 128
BLOCK = 32
NUMBERS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


# ------------------------------------------------------------------ the format
def power_of(block):
    """The byte of a block (a list of Python floats)."""
    if any(math.isinf(x) or math.isnan(x) for x in block):
        return 255
    top = max(abs(x) for x in block)
    for p in range(7, 252):
        if top < 7 * 2.0 ** (p - 127):
            return p
    return 252


def code_of(x, power):
    if power == 255:
        return 0
    y = abs(x) / 2.0 ** (power - 127)
    best = min(range(8), key=lambda c: (abs(NUMBERS[c] - y), c % 2))  # ties: the even code
    return best + (8 if math.copysign(1.0, x) < 0 else 0)


def quantise_slow(row):
    """128 Python floats -> (64 bytes, 4 powers)."""
    codes, powers = [], []
    for i in range(0, D, BLOCK):
        p = power_of(row[i:i + BLOCK])
        powers.append(p)
        codes += [code_of(x, p) for x in row[i:i + BLOCK]]
    return [codes[i] + 16 * codes[i + 1] for i in range(0, D, 2)], powers


def two_to(power):
    """2^(power - 127) in 64 bits, by its bits (pow is off by a last place on some devices)."""
    return ((power.long() + (1023 - 127)) << 52).view(torch.float64)


def quantise(x):
    """``x[..., D]`` in 64 bits -> (codes u8 ``[..., D/2]``, powers u8 ``[..., D/32]``)."""
    x = x.double().reshape(*x.shape[:-1], D // BLOCK, BLOCK)
    top = x.abs().amax(-1)
    bad = ~torch.isfinite(x).all(-1)
    # top >= 7 * 2^(p - 127) asks for a power above p
    steps = 7.0 * two_to(torch.arange(7, 252, device=x.device))
    power = 7 + torch.bucketize(torch.where(bad, 0.0, top).contiguous(), steps, right=True)
    y = x.abs() / two_to(power).unsqueeze(-1)
    y = torch.where(bad.unsqueeze(-1), 0.0, y)
    # distances are exact, so ties are ties; of two nearest numbers the even code
    # comes first
    near, code = torch.full_like(y, math.inf), torch.zeros_like(y, dtype=torch.long)
    for c in (0, 2, 4, 6, 1, 3, 5, 7):
        off = (y - NUMBERS[c]).abs()
        code, near = torch.where(off < near, c, code), torch.minimum(off, near)
    code = code + 8 * torch.signbit(x) * (~bad.unsqueeze(-1))
    code = code.flatten(-2).to(torch.uint8)
    power = torch.where(bad, 255, power)
    return code[..., 0::2] + 16 * code[..., 1::2], power.to(torch.uint8)


def values(codes, powers):
    """What a cache's bytes stand for, in 64 bits (NaN in blocks of power 255)."""
    n = torch.tensor(NUMBERS + [-x for x in NUMBERS], dtype=torch.float64, device=codes.device)
    c = torch.stack([codes.long() & 15, codes.long() >> 4], -1).flatten(-2)
    scale = two_to(powers)
    scale = torch.where(powers == 255, torch.nan, scale).repeat_interleave(BLOCK, -1)
    return n[c] * scale


# ------------------------------------------------------------------ windows
def sees(ctx, S, S_max, max_ctx, window, sink):
    """``[S, S_max]``: what each query of one row sees."""
    p = min(ctx, S_max) - 1 + torch.arange(S).view(S, 1)
    e = torch.arange(S_max).view(1, S_max)
    return (e <= p) & (e < max_ctx) & ((e > p - (window or 1 << 40)) | (e < sink))


def window(q, k, v, ctx, B, S, window, sink, max_ctx, scale):
    """(outputs, bounds) ``[B*S, Hq*D]`` over ``k, v[B, Hkv, S_max, D]``."""
    Hq, Hkv, S_max = q.shape[1], k.shape[1], k.shape[2]
    G = Hq // Hkv
    out = torch.zeros(B * S, Hq, D, dtype=torch.float64, device=q.device)
    bound = torch.full_like(out, 1e-30)
    for b in range(B):
        see = sees(ctx[b], S, S_max, max_ctx, window, sink).to(q.device)
        used = see.any(0).nonzero().view(-1)
        if used.numel() == 0:
            continue
        see = see[:, used]
        for h in range(Hq):
            o, e, _, _ = cache_ref.attend(q[b * S:(b + 1) * S, h], k[b, h // G][used], v[b, h // G][used], see, scale)
            out[b * S:(b + 1) * S, h], bound[b * S:(b + 1) * S, h] = o, e
    return out.view(B * S, Hq * D), bound.view(B * S, Hq * D)


# ------------------------------------------------------------------ append
def append(qkv, qn, kn, cos, sin, positions, Hq, Hkv, eps):
    """Keys and values ``[T, Hkv, D]`` of raw projection rows, in 64 bits."""
    T = qkv.shape[0]
    x = qkv.double().view(T, Hq + 2 * Hkv, D)
    k = x[:, Hq:Hq + Hkv]
    k = k / torch.sqrt((k * k).mean(-1, keepdim=True) + eps) * kn.double()
    c, s = cos[positions.long()].double().unsqueeze(1), sin[positions.long()].double().unsqueeze(1)
    lo, hi = k[..., :D // 2], k[..., D // 2:]
    return torch.cat([lo * c - hi * s, hi * c + lo * s], -1), x[:, Hq + Hkv:]
