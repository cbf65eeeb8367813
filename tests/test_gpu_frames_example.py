"""The network of examples/patch_splats.py over frames: heads normed and turned, a
window with first tokens that stay visible, dropout onto the residual, and views
over a memory that they share, together as they would be used."""

from __future__ import annotations

import importlib.util
import math

import pytest
import torch
import torch.nn.functional as F

from conftest import ROOT
from oracle import token_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("patch_splats",
                                                  ROOT / "examples" / "patch_splats.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def path(example, frames, seed, size=64):
    images, cams = example.make_scene(frames, size, seed)
    tokens, positions, rays = example.tokens_of(images[:-1], cams[:-1], size)
    return tokens, example.with_frames(positions, (size // example.PATCH) ** 2), rays


class Plain:
    """The operators in elementary torch operations, float64."""

    def __init__(self, mg):
        self.mg = mg

    def layer_norm(self, x, w, b):
        c = x - x.mean(-1, keepdim=True)
        return c / (c.square().mean(-1, keepdim=True) + 1e-5).sqrt() * w + b

    def norm_rotary(self, q, k, qw, kw, positions, frequencies, sections):
        axes = torch.tensor(token_ref.axes_of(sections, "runs"), device=q.device)
        t = (positions[:, axes].double() * frequencies)[:, None]

        def one(x, w):
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w
            a, b = x.chunk(2, -1)
            return torch.cat([a * t.cos() - b * t.sin(), b * t.cos() + a * t.sin()], -1)

        return one(q, qw), one(k, kw)

    def attention(self, q, k, v, q_offsets, k_offsets, causal, window, sinks):
        assert k_offsets is None and causal
        out, bounds = [], q_offsets.tolist()
        for a, b in zip(bounds[:-1], bounds[1:]):
            seen = torch.from_numpy(token_ref.sees(b - a, b - a, True, window, sinks)).to(q.device)
            for h in range(q.shape[1]):
                kh = h * k.shape[1] // q.shape[1]
                s = q[a:b, h] @ k[a:b, kh].T / math.sqrt(q.shape[2])
                out.append(s.masked_fill(~seen, -math.inf).softmax(1) @ v[a:b, kh])
            out[-q.shape[1]:] = [torch.stack(out[-q.shape[1]:], 1)]
        return torch.cat(out)

    def dropout(self, x, p, seed, residual, site):
        # Which elements are kept is tested by itself, against the generator.
        kept = self.mg.dropout(torch.ones_like(x, dtype=torch.float32), p, seed, site=site)
        return residual + x * kept.double()


def test_gradients_of_the_whole_network(dev, example, monkeypatch):
    """Against the same network in float64. Its bfloat16 operators and products round some
    20 times in a row, 2^-8 each at most, were they all alike in sign: an error of
    20 * 2^-8 of a gradient's norm."""
    net = example.Network(seed=2, frames=True, window=20, sinks=3, drop=0.2)
    parts = [path(example, n, s) for n, s in ((3, 0), (2, 1))]
    tokens, positions, _ = (torch.cat(t) for t in zip(*parts))
    offsets = example.offsets_of([p[0].shape[0] for p in parts])
    seed = torch.tensor([77], device=dev)
    g = torch.Generator().manual_seed(5)
    names = list(net.params)
    out = net(tokens, positions, offsets, causal=True, seed=seed)
    dy = torch.randn(out.shape, generator=g).to(dev)
    got = torch.autograd.grad(out, list(net.params.values()), dy)
    mg, plain = example.mg, Plain(example.mg)
    for name in ("layer_norm", "norm_rotary", "attention", "dropout"):
        monkeypatch.setattr(mg, name, getattr(plain, name))
    plain.mg = type("Drawn", (), {"dropout": staticmethod(
        importlib.import_module("metal_gauss_amd.dropout").dropout)})
    net.params = {n: p.detach().double().requires_grad_(True) for n, p in net.params.items()}
    monkeypatch.setattr(example.Network, "_product",
                        lambda self, x, name: F.linear(x, self.params[name]))
    monkeypatch.setattr(torch.Tensor, "float", lambda t: t)
    want = net(tokens.double(), positions, offsets, causal=True, seed=seed)
    exact = torch.autograd.grad(want, list(net.params.values()), dy.double())
    monkeypatch.undo()
    allowed = 20 * 2.0 ** -8
    assert float((out.double() - want).norm() / want.norm()) < allowed
    for name, a, b in zip(names, got, exact):
        assert a.shape == b.shape and bool(a.isfinite().all())
        assert float((a.double() - b).norm() / b.norm()) < allowed, name


def test_training_steps_run(dev, example):
    """Steps through the renderer, each with draws of its own."""
    net = example.Network(seed=1, frames=True, window=24, sinks=2, drop=0.1)
    mg = example.mg
    images, cams = example.make_scene(3, 64, 4)
    tokens, positions, rays = example.tokens_of(images[:-1], cams[:-1], 64)
    positions = example.with_frames(positions, 16)
    offsets = example.offsets_of([tokens.shape[0]])
    opt = mg.FusedAdam([{"params": list(net.params.values())}], lr=1e-3, eps=1e-8)
    window = mg.gaussian_kernel(device=dev, groups=15)
    seed, before = torch.tensor([5], device=dev), {n: p.clone() for n, p in net.params.items()}
    for _ in range(3):
        prediction = net(tokens, positions, offsets, causal=True, seed=seed)
        means, quats, log_scales, logits, colors = example.splats_of(prediction, rays)
        K, vm = cams[-1]
        rgb, _, _ = mg.render(means, quats, log_scales, logits, None, K, vm, 64, 64,
                              colors=colors, activations=True)
        loss = mg.photometric_loss(rgb, images[-1], window)[0]
        opt.zero_grad(set_to_none=True)
        loss.backward()
        for name, p in net.params.items():
            assert bool(p.grad.isfinite().all()), name
        opt.step()
        seed.add_(1)
        assert math.isfinite(float(loss.detach()))
    assert all(not torch.equal(p, before[n]) for n, p in net.params.items())


def test_views_over_a_shared_memory(dev, example):
    """Each candidate is what it is added to the scene alone. The products' tiles may
    differ with the number of rows: bfloat16 rounding (2^-8) of activations of size
    one, through two blocks."""
    net = example.Network(seed=3, frames=True)
    tokens, positions, _ = path(example, 4, 6)
    n = 32
    views = [(tokens[n:n + 16], positions[n:n + 16]), (tokens[n + 16:], positions[n + 16:]),
             (tokens[5:6], positions[5:6])]
    got = example.candidates(net, tokens[:n], positions[:n], views)
    for (t, at), view in zip(views, got):
        alone = example.extend(net, torch.cat([tokens[:n], t]), torch.cat([positions[:n], at]), n)
        assert view.shape == alone.shape
        assert float((view - alone).abs().max()) < 0.1


def test_views_of_a_network_with_a_window_are_refused(dev, example):
    net = example.Network(seed=3, frames=True, window=20)
    tokens, positions, _ = path(example, 4, 6)
    with pytest.raises(ValueError, match="seen whole"):
        example.candidates(net, tokens[:32], positions[:32], [(tokens[32:], positions[32:])])


def test_a_window_over_the_memory(dev, example):
    """New tokens over kept keys and values see what they see in the whole path."""
    net = example.Network(seed=4, frames=True, window=20, sinks=4)
    tokens, positions, _ = path(example, 4, 7)
    n = tokens.shape[0]
    with torch.no_grad():
        whole = net(tokens, positions, example.offsets_of([n]), causal=True)
    for old in (1, 30, n - 1):
        new = example.extend(net, tokens, positions, old)
        assert float((new - whole[old:]).abs().max()) < 0.1
