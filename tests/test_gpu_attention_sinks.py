"""Gradients of attention's first keys that stay visible, on the GPU, over packs of many
sequences: those whose window items go on for their sinks, those with items of their
own, and both in one pack. Against the float64 restatement, by the tolerances of
test_gpu_attention_window.py."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gpu_attention_window import check, inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(1, 1), (3, 130), (9, 33), (475, 1000)])
@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 4, 2, 64), ("f16", 3, 1, 32)])
def test_many_short_sequences(dev, window, sinks, ty, heads, kv, dim):
    rng = np.random.default_rng(window)
    q_lens = [int(x) for x in rng.integers(0, 40, 300)]
    k_lens = [max(0, n + int(x)) for n, x in zip(q_lens, rng.integers(-5, 25, 300))]
    q, k, v, do = inputs(("short", window, ty), sum(q_lens), sum(k_lens), heads, kv, dim, ty)
    check(dev, q, k, v, do, q_lens, k_lens, ty, window, sinks)


@pytest.mark.parametrize("ty,heads,kv,dim", [("bf16", 4, 2, 64), ("f16", 5, 1, 128)])
@pytest.mark.parametrize("sinks", [3, 130, 700])
@pytest.mark.parametrize("window", [1, 70])
def test_sequences_about_the_length_of_items_of_their_own(dev, ty, heads, kv, dim, sinks, window):
    """255 to 257 queries past the window of the first key, one of them alone over a
    longer memory, and none."""
    q_lens = [window + 255, window + 256, window + 257, 257, 256, window, 300]
    k_lens = [window + 255, window + 256, window + 257, window + 600, 900, window, 100]
    q, k, v, do = inputs(("near", window, sinks, ty), sum(q_lens), sum(k_lens), heads, kv, dim, ty)
    check(dev, q, k, v, do, q_lens, k_lens, ty, window, sinks)


@pytest.mark.parametrize("heads,kv", [(10, 2), (8, 1), (3, 3)])
def test_runs_of_some_of_the_heads(dev, heads, kv):
    """Enough tokens for runs of several heads' tiles, even and uneven, beside sequences
    that have none and one whose heads are cut."""
    q_lens = [420, 700, 60, 5, 0, 200, 2600, 800] + [510] * 16
    n = sum(q_lens)
    q, k, v, do = inputs(("some", heads), n, n, heads, kv, 16, "bf16")
    check(dev, q, k, v, do, q_lens, q_lens, "bf16", 50, 300)


def test_one_sequence_of_sinks_alone(dev):
    """More sinks than a window leaves out, in items and in place."""
    for n, window, sinks in ((1500, 1, 1500), (900, 300, 899), (300, 20, 300)):
        q, k, v, do = inputs(("alone", n), n, n, 4, 2, 64, "f16")
        check(dev, q, k, v, do, [n], [n], "f16", window, sinks)


@pytest.mark.parametrize("tokens,sequences,heads,dim,window,sinks", [
    (32768, 2048, 32, 64, 475, 130), (32768, 512, 32, 64, 475, 1000), (16320, 1024, 32, 32, 475, 500)])
def test_packs_of_thousands_of_sequences(dev, tokens, sequences, heads, dim, window, sinks):
    """The first, middle and last sequences of two heads against the restatement."""
    from metal_gauss_amd import attention
    from oracle import token_ref
    from test_gpu_attention_window import UNIT, host

    rng = np.random.default_rng(sequences)
    at = np.sort(rng.choice(np.arange(1, tokens), sequences - 1, replace=False))
    off = np.concatenate([[0], at, [tokens]])
    q, k, v, do = inputs(("thousands", sequences), tokens, tokens, heads, heads, dim, "bf16")
    leaves = [t.to(dev).requires_grad_(True) for t in (q, k, v)]
    o = attention(*leaves, torch.tensor(off, dtype=torch.int32, device=dev), causal=True,
                  window=window, sinks=sinks)
    got = [o, *torch.autograd.grad(o, leaves, do.to(dev))]
    for s in (0, 1, sequences // 2, sequences - 2, sequences - 1):
        lo, hi = int(off[s]), int(off[s + 1])
        for h in (0, heads - 1):
            part = [host(t[lo:hi, h:h + 1]) for t in (q, k, v, do)]
            want, bound = token_ref.attention(*part[:3], [0, hi - lo], [0, hi - lo], True,
                                              dim ** -0.5, part[3], UNIT["bf16"], window, sinks)
            for a, w, b in zip(got, want, bound):
                a = host(a[lo:hi, h:h + 1])
                assert (np.abs(a - w) <= b * (1.0 + 2.0 ** -14 / UNIT["bf16"]) * 1.05 + 1e-30).all()


@pytest.mark.parametrize("sinks", [4, 130])
def test_items_of_their_own_in_a_graph_and_on_another_stream(dev, sinks):
    """Replayed with other inputs and other lengths, some sequences gaining items of
    their own and some losing them, against the eager result."""
    from metal_gauss_amd import attention

    q, k, v, do = (t.to(dev) for t in inputs(("graph", sinks), 1400, 1400, 4, 2, 64, "bf16"))
    off = torch.tensor([0, 700, 740, 1400], dtype=torch.int32, device=dev)
    leaves = [t.requires_grad_(True) for t in (q, k, v)]

    def step():
        o = attention(*leaves, off, causal=True, window=60, sinks=sinks)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lens in ([0, 700, 740, 1400], [0, 100, 200, 1400], [0, 300, 620, 940], [0, 0, 1399, 1400]):
        with torch.no_grad():
            off.copy_(torch.tensor(lens, dtype=torch.int32))
            for i, t in enumerate(leaves):
                t.copy_(inputs(("again", lens[1], i), 1400, 1400, 4, 2, 64, "bf16")[min(i, 1)])
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))
