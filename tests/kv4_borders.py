"""Projection rows whose keys, normalised and rotated, lie next to a border: between two
numbers of a block, or between two powers of it."""

import torch

import kv4_ref as ref

D = 128
EPS = 1e-6


def keys(x, w, cos, sin):
    """Keys ``[n, D]`` of ``x[n, D]`` in the type of its arguments."""
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS)
    y = x * r * w
    lo, hi = y[:, :D // 2], y[:, D // 2:]
    return torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)


def rows(n, seed):
    """(x f32 ``[n, D]``, norm weight bf16 ``[D]``, cos, sin f32 ``[n, D / 2]``, the
    element of each row that is next to a border, its distance from that border
    relative to its size).  A row's element is moved until its key in 64 bits meets the
    border, then rounded to 32 bits: what is left is half a place of those, up to
    which 32-bit arithmetic is in doubt about the side."""
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(n, D, generator=g) * 1.5).double()
    w = (1.0 + 0.1 * torch.randn(D, generator=g)).to(torch.bfloat16)
    angle = torch.rand(n, D // 2, generator=g, dtype=torch.float64) * 0.5
    angle[::3] = 0.0  # position 0: no rotation
    cos, sin = angle.cos().float(), angle.sin().float()
    wide = (w.double(), cos.double(), sin.double())
    k = keys(x, *wide)
    blocks = k.abs().view(n, -1, ref.BLOCK)
    at_row = torch.arange(n)
    # every fourth row: the largest element of a block next to 7 times a power; the
    # others: some element next to a border of two numbers
    block = torch.randint(0, D // ref.BLOCK, (n,), generator=g)
    top, largest = blocks[at_row, block].max(-1)
    element = block * ref.BLOCK + torch.where(at_row % 4 == 0, largest, (largest + 1 + torch.randint(
        0, ref.BLOCK - 1, (n,), generator=g)) % ref.BLOCK)
    power = ref.quantise(k)[1][at_row, block]
    scale = ref.two_to(power)
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    size = k[at_row, element].abs()
    near = borders[(size[:, None] / scale[:, None] - borders).abs().argmin(1)] * scale
    up, down = 7.0 * scale, 3.5 * scale
    near = torch.where(at_row % 4 == 0, torch.where(up / size < size / down, up, down), near)
    target = torch.copysign(near, k[at_row, element])
    for _ in range(60):
        k = keys(x, *wide)
        r = 1.0 / torch.sqrt((x * x).mean(-1) + EPS)
        slope = r * w.double()[element] * cos.double()[at_row, element % (D // 2)]
        x[at_row, element] += (target - k[at_row, element]) / slope
    x = x.float()
    k = keys(x.double(), *wide)
    off = (k[at_row, element] - target) / target
    # rows that did not settle, or whose move changed the block's power, go; and those
    # that meet the border more closely than sums in 64 bits of any order agree
    after = ref.two_to(ref.quantise(k)[1][at_row, block])
    same = (after == scale) | (at_row % 4 == 0)
    keep = (off.abs() < 2.0 ** -22) & (off.abs() > 2.0 ** -36) & same
    return x[keep], w, cos[keep], sin[keep], element[keep], off[keep]
