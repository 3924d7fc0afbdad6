"""The rows next to a border do what they are for: arithmetic in 32 bits puts some of
them on the wrong side."""

import torch

import kv4_borders
import kv4_ref as ref


def test_rows_next_to_a_border_need_64_bits():
    x, w, cos, sin, element, off = kv4_borders.rows(2400, 1)
    assert x.shape[0] >= 2048
    exact = ref.quantise(kv4_borders.keys(x.double(), w.double(), cos.double(), sin.double()))
    short = ref.quantise(kv4_borders.keys(x, w.float(), cos, sin))
    codes = (exact[0] != short[0]).any(1)
    powers = (exact[1] != short[1]).any(1)
    print(int(codes.sum()), int(powers.sum()), x.shape[0])
    assert int(codes.sum()) >= 100 and int(powers.sum()) >= 20
    # on both sides of the borders
    assert int((off > 0).sum()) >= 500 and int((off < 0).sum()) >= 500
    # and a next float of the moved element is on the other side of some
    step = torch.nextafter(x, torch.copysign(torch.full_like(x, 1e30), x))
    moved = x.clone()
    moved[torch.arange(x.shape[0]), element] = step[torch.arange(x.shape[0]), element]
    other = ref.quantise(kv4_borders.keys(moved.double(), w.double(), cos.double(), sin.double()))
    assert int(((exact[0] != other[0]).any(1) | (exact[1] != other[1]).any(1)).sum()) >= 200
