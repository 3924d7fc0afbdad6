"""The 4-bit format's reference against itself: the fast form of the tests and the one
that follows the definition an element at a time."""

import math

import pytest
import torch

import kv4_ref as ref

F = torch.finfo(torch.bfloat16)


def _rows():
    g = torch.Generator().manual_seed(0)
    rows = [torch.randn(128, generator=g) * s for s in (1.0, 3e-3, 1e30, 1e-37, 1e-39)]
    rows.append(torch.zeros(128))
    rows.append(torch.full((128,), -0.0))
    rows.append(torch.full((128,), F.max))
    rows.append(torch.full((128,), -F.tiny / 64))
    borders = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 6.5, 6.96875]
    rows.append(torch.tensor([x * s for x in borders for s in (1, -1)] * 6 + [0.0] * 8))
    rows.append(torch.tensor([7.0, 1.0] * 64))      # the next power
    rows.append(torch.tensor([3.484375, 0.125] * 64))
    bad = torch.randn(128, generator=g)
    bad[5], bad[40], bad[100] = math.inf, math.nan, -math.inf
    rows.append(bad)
    return torch.stack(rows).to(torch.bfloat16)


@pytest.mark.parametrize("i", range(13))
def test_quantise_reference(i):
    row = _rows()[i]
    codes, powers = ref.quantise(row.double())
    slow_codes, slow_powers = ref.quantise_slow(row.double().tolist())
    assert powers.tolist() == slow_powers
    assert codes.tolist() == slow_codes
    v = ref.values(codes, powers)
    fine = torch.isfinite(row).view(4, 32).all(1).repeat_interleave(32)
    assert bool(torch.isnan(v[~fine]).all())
    # a number is off by at most half a step (1 above 4, where steps are 2), and
    # what is past 6 by the 1 that the power's rule leaves; the largest finite
    # values stop at 6 * 2^125
    scale = torch.pow(2.0, powers.double() - 127).repeat_interleave(32)
    off = (v - row.double())[fine].abs() / scale[fine]
    assert float(off.max() if off.numel() else 0.0) <= (2.0 if i == 7 else 1.0)


def test_window_of_a_query():
    see = ref.sees(5, 3, 10, 10, 2, 1)
    assert see.nonzero().tolist() == [[0, 0], [0, 3], [0, 4], [1, 0], [1, 4], [1, 5], [2, 0], [2, 5], [2, 6]]
    assert not bool(ref.sees(0, 1, 4, 4, 2, 4).any())
    assert ref.sees(3, 1, 4, 4, 0, 0).sum() == 3
