"""kv4_append of keys next to a border of two numbers, or of two powers."""

import pytest
import torch

import kv4_borders
import kv4_ref as ref
from gpu_util import announce
from qmoe import ops

pytestmark = pytest.mark.gpu

D = 128


@pytest.mark.parametrize("S", [1, 4])
def test_keys_next_to_a_border_land_on_the_right_side(dev, S):
    """Byte for byte the entries of keys in 64 bits: in 32 bits some of them are others."""
    announce(f"kv4_append, keys next to a border, {S} tokens a row")
    x, w, cos, sin, _, _ = (t.to(dev) for t in kv4_borders.rows(2400, 1))
    hq, hkv, T = 4, 4, 512
    B = T // S
    x, cos, sin = x[:T * hkv], cos[:T * hkv], sin[:T * hkv]
    want = ref.quantise(kv4_borders.keys(x.double(), w.double(), cos.double(), sin.double()))
    g = torch.Generator(device=dev).manual_seed(2)
    # heads of a token share its position, so token t has the rows 4 t .. 4 t + 3 in four
    # calls, one for each head's tables
    for head in range(hkv):
        qkv = torch.randn(T, hq + 2 * hkv, D, generator=g, device=dev)
        qkv[:, hq + head] = x[head::hkv]
        cache = ops.kv4_cache(B, hkv, S + 1, D, dev)
        at = torch.arange(T, dtype=torch.int32, device=dev)
        ops.kv4_append(qkv.view(T, -1), w, w, cos[head::hkv].contiguous(), sin[head::hkv].contiguous(), at, at % S, hq, hkv,
                       cache, 1e-6, S=S)
        torch.cuda.synchronize()
        for got, need, name in ((cache[0], want[0], "codes"), (cache[1], want[1], "powers")):
            got = got[:, head, :S].reshape(T, -1)
            wrong = (got != need[head::hkv]).any(1)
            assert not bool(wrong.any()), f"{name} of {int(wrong.sum())} rows of {T}"
