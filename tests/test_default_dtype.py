"""Buffers that kernels write have float32 by name: torch's default type is the
caller's, and with a shorter one the kernels would write past them."""

from __future__ import annotations

import ast
from pathlib import Path

import pytest
import torch

PACKAGE = Path(__file__).resolve().parents[1] / "metal-gauss_amd"
MAKERS = {"empty", "zeros", "ones", "full", "empty_strided"}


def untyped(source: str) -> list[int]:
    """Lines of torch.empty(...) and its like without a dtype."""
    found = []
    for node in ast.walk(ast.parse(source)):
        if isinstance(node, ast.Call) and isinstance(node.func, ast.Attribute) \
                and isinstance(node.func.value, ast.Name) and node.func.value.id == "torch" \
                and node.func.attr in MAKERS and not any(k.arg == "dtype" for k in node.keywords):
            found.append(node.lineno)
    return found


# scenes.py makes random scenes on the CPU, which no kernel writes.
@pytest.mark.parametrize("name", sorted(p.name for p in PACKAGE.glob("*.py")
                                        if p.name != "scenes.py"))
def test_buffers_name_their_type(name):
    assert not untyped((PACKAGE / name).read_text())


def test_the_check_finds_one_without():
    assert untyped("a = torch.empty(3, device=d)\nb = torch.empty(3, dtype=torch.int32)") == [1]


@pytest.mark.gpu
@pytest.mark.parametrize("default", [torch.bfloat16, torch.float64])
def test_results_do_not_go_by_the_default_type(dev, default):
    from metal_gauss_amd import attention, dropout, layer_norm, norm_rotary, render
    from metal_gauss_amd import rotary_frequencies, shared_attention

    g = torch.Generator().manual_seed(5)
    rand = lambda *shape: torch.randn(*shape, generator=g, dtype=torch.float32).to(dev)  # noqa: E731
    qkv = [rand(300, h, 64).bfloat16().requires_grad_(True) for h in (4, 2, 2)]
    do, x, w, b = rand(300, 4, 64).bfloat16(), rand(300, 256), rand(256), rand(256)
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    dx, qw = rand(300, 256), rand(64)
    pos = torch.arange(300, device=dev)
    freq = rotary_frequencies(64, device=dev)
    seed = 7
    n = 400
    scene = [(rand(n, 3) * 0.6 + torch.tensor([0.0, 0.0, 4.0], device=dev, dtype=torch.float32)),
             rand(n, 4), rand(n, 3).abs() * 0.1 + 0.03, rand(n).sigmoid(), rand(n, 16, 3) * 0.25]
    scene = [t.detach().requires_grad_(True) for t in scene]
    K = torch.tensor([[51.2, 0, 32], [0, 51.2, 24], [0, 0, 1]], dtype=torch.float32)
    vm = torch.eye(4, dtype=torch.float32)

    def run():
        out = []
        for kw in (dict(causal=True), dict(causal=True, window=30, sinks=4)):
            o = attention(*qkv, **kw)
            out += [o, *torch.autograd.grad(o, qkv, do)]
        with torch.no_grad():
            out += [shared_attention(*qkv, qkv[1], qkv[2]), attention(qkv[0][:2], *qkv[1:])]
        y = layer_norm(x, w, b)
        out += [y, *torch.autograd.grad(y, leaves, dx)]
        out.append(dropout(x, 0.3, seed).detach())
        out += list(norm_rotary(qkv[0].detach(), qkv[1].detach(), qw, qw, pos, freq))
        rgb, alpha, _ = render(*scene, K, vm, 64, 48, sh_degree=3)
        out += [rgb, alpha]
        grads = torch.autograd.grad(rgb.square().sum(), scene)
        return [t.detach() for t in out], grads

    want, want_grads = run()
    before = torch.get_default_dtype()
    torch.set_default_dtype(default)
    try:
        got, grads = run()
    finally:
        torch.set_default_dtype(before)
    for a, b_ in zip(got, want):
        assert a.dtype == b_.dtype and torch.equal(a, b_)
    # The renderer's gradients are added up by atomics, in any order.
    for a, b_ in zip(grads, want_grads):
        assert a.dtype == b_.dtype
        assert float((a - b_).norm()) <= 1e-4 * float(b_.norm())
