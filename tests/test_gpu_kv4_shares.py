"""Attention over a 4-bit cache with an even share of all keys for every workgroup
(long batches): the cut is found on the device from all rows' lengths, so it is
replayed with others, and with windows that differ within an item."""

import math

import pytest
import torch

import kv4_ref as ref
from gpu_util import announce, bf16_randn
from qmoe import ops

pytestmark = pytest.mark.gpu

D = 128
SCALE = 1.0 / math.sqrt(D)
STEP = 256  # keys of a workgroup's step
ROWS = 16   # query rows of an item


def _i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _places(dev):
    return 2 * torch.cuda.get_device_properties(dev).multi_processor_count


def _in_shares(ws, dev):
    """Whether a workspace is that of even shares: two records (m, l and O of 16 rows)
    for each place."""
    return ws is not None and ws.numel() * ws.element_size() == 2 * _places(dev) * (2 * ROWS + ROWS * D) * 4


def _filled(B, Hkv, S_max, g, dev):
    cache = ops.kv4_cache(B, Hkv, S_max, D, dev)
    for b in range(B):
        rows = [bf16_randn((1, Hkv, S_max, D), g, dev) for _ in range(2)]
        ops.kv4_store(*rows, tuple(t[b:b + 1] for t in cache))
    return cache


def _check_rows(got, q, cache, ctx, S, window, sink, which):
    for b in which:
        one = slice(b * S, (b + 1) * S)
        k, v = (ref.values(c[b:b + 1], p[b:b + 1]) for c, p in (cache[:2], cache[2:]))
        want, bound = ref.window(q[one], k, v, [ctx[b]], 1, S, window, sink, k.shape[2], SCALE)
        worst = float(((got[one].double() - want).abs() / bound).max())
        print(f"  row {b} of {ctx[b]}: worst error {worst:.3f} of the bound", flush=True)
        assert worst <= 1.0, b


def test_even_shares_with_a_window_and_several_queries(dev):
    """The first and the last query of an item see different windows."""
    S, Hq, Hkv, window, sink = 3, 16, 4, 33000, 4
    S_max = 34000
    steps = -(-(window + sink + S - 1 + 3) // STEP)
    B = -(-16 * _places(dev) // (Hkv * steps))
    announce(f"even shares, {B} x {S} queries, window {window}")
    assert _in_shares(ops.attn_kv4_workspace(B, S, Hq, Hkv, D, window, sink, S_max, dev), dev)
    g = torch.Generator(device=dev).manual_seed(3)
    cache = _filled(B, Hkv, S_max, g, dev)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    ctx = ([34000, 1, -1, 33001, 33990, 33002, 20000, 33500] * B)[:B]
    got = ops.attn_kv4(q, cache, _i32(ctx, dev), B, S, window, sink)
    again = ops.attn_kv4(q, cache, _i32(ctx, dev), B, S, window, sink)
    torch.cuda.synchronize()
    assert torch.equal(got, again) and not bool(torch.isnan(got).any())
    _check_rows(got, q, cache, ctx, S, window, sink, sorted({*range(min(B, 8)), B - 1}))


def test_graph_replays_of_even_shares(dev):
    """A step and a windowed chunk in even shares, on one workspace, captured once and
    replayed with other lengths and eager work between; every replay as the eager
    call, and rows of it against 64 bits."""
    B, Hq, Hkv, S = 40, 32, 4, 2
    S_max = (-(-16 * _places(dev) // (B * Hkv)) + 2) * STEP - 37
    window, sink = S_max - 2 * STEP, 4
    announce(f"even shares in a graph, {B} rows of up to {S_max}")
    ws = ops.attn_kv4_workspace(B, 1, Hq, Hkv, D, 0, 0, S_max, dev)
    assert _in_shares(ws, dev)
    assert _in_shares(ops.attn_kv4_workspace(B, S, Hq, Hkv, D, window, sink, S_max, dev), dev)
    g = torch.Generator(device=dev).manual_seed(9)
    cache = _filled(B, Hkv, S_max, g, dev)
    q = bf16_randn((B * S, Hq, D), g, dev, 2.0)
    ctx = _i32([1] * B, dev)
    outs = [torch.zeros(n, Hq * D, dtype=torch.bfloat16, device=dev) for n in (B, B * S)]

    def calls(outs, ws):
        ops.attn_kv4(q[:B], cache, ctx, B, 1, workspace=ws, out=outs[0])
        ops.attn_kv4(q, cache, ctx, B, S, window, sink, workspace=ws, out=outs[1])

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        calls(outs, ws)
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        calls(outs, ws)
    eager = [torch.zeros_like(o) for o in outs]
    for rep, (top, less) in enumerate([(S_max, 290), (1, 0), (5000, 290), (0, 0), (S_max, 0), (S_max - 1, 3 * S_max),
                                       (257, 7)]):
        lengths = [max(-S, top - less * i) for i in range(B)]
        ctx.copy_(_i32(lengths, dev))
        q.normal_(0.0, 2.0, generator=g)
        graph.replay()
        torch.cuda.synchronize()
        calls(eager, None)
        torch.cuda.synchronize()
        for a, b in zip(outs, eager):
            assert torch.equal(a, b), rep
            assert not bool(torch.isnan(a).any())
        if rep in (0, 5):
            _check_rows(outs[0], q[:B], cache, lengths, 1, 0, 0, (0, 1, B - 1))
            _check_rows(outs[1], q, cache, lengths, S, window, sink, (0, 1, B - 1))
