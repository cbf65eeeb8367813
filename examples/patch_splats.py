"""Predict splats from posed images with a small network over patch tokens, and
train it through the renderer.

Each 16 x 16 patch of each input view is a token; the views of a scene are one
sequence, and scenes of different numbers of views are packed one after the
other. A block is layer norm, a projection to queries, keys and values, rotary
positions (the patch's column and row), attention within the scene, and a small
perceptron. Each token predicts a few Gaussians along its patch's ray, which
``render`` draws from a view that was not among the inputs; the photometric loss
against that view trains everything through FusedAdam.

With ``causal=True`` a token sees the views before its own and the tokens before
it, so that a new view can be added to a scene already seen: ``extend`` runs the
new tokens alone over the keys and values kept of the old ones, and ``candidates``
runs several views at once, each by itself, over the one memory that they share.

For the frames of a camera path a network takes ``frames=True``: heads are normed
and turned by frame, column and row; ``window`` and ``sinks``: a token sees the last
tokens and the path's first ones alone; and ``drop``: the branches are dropped out
as they are added to the residual.

    python examples/patch_splats.py [--steps 60] [--seed 0]

Views are synthetic: random coloured balls drawn by the renderer itself.
"""

from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import torch
import torch.nn.functional as F

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

import metal_gauss_amd as mg  # noqa: E402

PATCH = 16
PER_TOKEN = 4            # Gaussians a token predicts
OUT = PER_TOKEN * 14     # offset 3, log scale 3, quaternion 4, opacity 1, colour 3


class Network:
    """Parameters (float32, as FusedAdam keeps them) and the forward pass; matrix
    products and attention run in bfloat16, norms and the residual in float32."""

    def __init__(self, width=128, heads=4, kv_heads=2, blocks=2, seed=0, device="cuda",
                 frames=False, window=None, sinks=0, drop=0.0):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.blocks = heads, kv_heads, width // heads, blocks
        self.window, self.sinks, self.drop = window, sinks, drop

        def matrix(rows, cols, gain=1.0):
            return torch.randn(rows, cols, generator=g) * (gain / math.sqrt(cols))

        p = {"embed": matrix(width, PATCH * PATCH * 3 + 6), "out": matrix(OUT, width, 0.1)}
        for b in range(blocks + 1):
            for n in ("a", "b") if b < blocks else ("a",):
                p[f"{b}.norm_{n}.w"], p[f"{b}.norm_{n}.b"] = torch.ones(width), torch.zeros(width)
            if b < blocks:
                p[f"{b}.qkv"] = matrix((heads + 2 * kv_heads) * self.dim, width)
                p[f"{b}.join"] = matrix(width, width, 0.5)
                p[f"{b}.up"] = matrix(4 * width, width)
                p[f"{b}.down"] = matrix(width, 4 * width, 0.5)
                if frames:
                    p[f"{b}.q_norm"], p[f"{b}.k_norm"] = torch.ones(self.dim), torch.ones(self.dim)
        self.params = {k: v.to(device).requires_grad_(True) for k, v in p.items()}
        self.sections = None
        if frames:                   # a quarter of the pairs for the frame
            pairs = self.dim // 2
            self.sections = (pairs // 4, (pairs - pairs // 4) // 2,
                             pairs - pairs // 4 - (pairs - pairs // 4) // 2)
        self.frequencies = mg.rotary_frequencies(self.dim, base=100.0, axes=1 if frames else 2,
                                                 device=device)

    def _product(self, x, name):
        return F.linear(x.bfloat16(), self.params[name].bfloat16())

    def _norm(self, x, name):
        return mg.layer_norm(x, self.params[name + ".w"], self.params[name + ".b"])

    def _turned(self, q, k, positions, block):
        if self.sections is None:
            return mg.rotary(q, k, positions, self.frequencies)
        return mg.norm_rotary(q, k, self.params[f"{block}.q_norm"], self.params[f"{block}.k_norm"],
                              positions, self.frequencies, sections=self.sections)

    def _add(self, x, branch, seed, site):
        if seed is None or self.drop == 0.0:
            return x + branch.float()
        return mg.dropout(branch, self.drop, seed, residual=x, site=site)

    def __call__(self, tokens, positions, q_offsets, k_offsets=None, causal=False, memory=None,
                 shared=None, seed=None):
        """tokens (n, patch and ray), positions (n, 2; of frames 3) -> (n, PER_TOKEN, 14).

        ``memory``: per block (keys, values) of the tokens seen before; the new
        ones' are joined to them, and k_offsets bounds the result. ``shared``: the
        same, which all sequences see beside their own. ``seed`` of the step's
        dropout; None (serving): none."""
        if shared is not None and self.window is not None:
            raise ValueError("a shared memory is seen whole: the network's window does not apply")
        H, Hk, D = self.heads, self.kv_heads, self.dim
        x = self._product(tokens, "embed").float()
        for b in range(self.blocks):
            qkv = self._product(self._norm(x, f"{b}.norm_a"), f"{b}.qkv").view(-1, H + 2 * Hk, D)
            q, k = self._turned(qkv[:, :H], qkv[:, H:H + Hk], positions, b)
            v = qkv[:, H + Hk:]
            if memory is not None:
                if b < len(memory):
                    k, v = torch.cat([memory[b][0], k]), torch.cat([memory[b][1], v])
                    memory[b] = (k, v)
                else:
                    memory.append((k, v))
            if shared is not None:
                o = mg.shared_attention(q, k, v, *shared[b], q_offsets, causal=causal)
            else:
                o = mg.attention(q, k, v, q_offsets, k_offsets, causal=causal,
                                 window=self.window, sinks=self.sinks)
            x = self._add(x, self._product(o.reshape(-1, H * D), f"{b}.join"), seed, 2 * b)
            up = F.gelu(self._product(self._norm(x, f"{b}.norm_b"), f"{b}.up"))
            x = self._add(x, self._product(up, f"{b}.down"), seed, 2 * b + 1)
        out = self._product(self._norm(x, f"{self.blocks}.norm_a"), "out").float()
        return out.view(-1, PER_TOKEN, 14)


def camera(angle, size, distance=4.0, device="cpu"):
    """(K, world to camera) of a camera on a circle around the origin."""
    c, s = math.cos(angle), math.sin(angle)
    R = torch.tensor([[c, 0.0, -s], [0.0, 1.0, 0.0], [s, 0.0, c]])
    vm = torch.eye(4)
    vm[:3, :3], vm[2, 3] = R, distance
    f = 0.9 * size
    return torch.tensor([[f, 0, size / 2], [0, f, size / 2], [0, 0, 1.0]]).to(device), vm


def make_scene(views, size, seed, device="cuda"):
    """Random balls drawn from views + 1 cameras; the last is the target."""
    g = torch.Generator().manual_seed(seed)
    n = 40
    means = (torch.rand(n, 3, generator=g) * 2.0 - 1.0).to(device)
    quats = torch.randn(n, 4, generator=g).to(device)
    scales = (torch.rand(n, 3, generator=g) * 0.15 + 0.1).to(device)
    colors = torch.rand(n, 3, generator=g).to(device)
    opacity = torch.full((n,), 0.9, device=device)
    angles = torch.rand(views + 1, generator=g) * 0.8 - 0.4
    cams = [camera(float(a), size) for a in angles]
    with torch.no_grad():
        images = [mg.render(means, quats, scales, opacity, None, K, vm, size, size,
                            colors=colors)[0] for K, vm in cams]
    return images, cams


def tokens_of(images, cams, size):
    """Patches with their rays, positions (column, row), and each token's ray
    origin and direction."""
    side = size // PATCH
    dev = images[0].device
    row, col = torch.meshgrid(torch.arange(side), torch.arange(side), indexing="ij")
    at = torch.stack([col, row], -1).view(-1, 2)
    out, rays = [], []
    for image, (K, vm) in zip(images, cams):
        patch = image.view(side, PATCH, side, PATCH, 3).permute(0, 2, 1, 3, 4)
        patch = patch.reshape(side * side, -1) - 0.5
        centre = (at.float() + 0.5) * PATCH
        d = torch.stack([(centre[:, 0] - K[0, 2].cpu()) / K[0, 0].cpu(),
                         (centre[:, 1] - K[1, 2].cpu()) / K[1, 1].cpu(),
                         torch.ones(side * side)], 1) @ vm[:3, :3]
        o = (-vm[:3, :3].T @ vm[:3, 3]).expand(side * side, 3)
        ray = torch.cat([o, d], 1).to(dev)
        out.append(torch.cat([patch, ray], 1))
        rays.append(ray)
    positions = at.to(dev, torch.int32).repeat(len(images), 1)
    return torch.cat(out), positions, torch.cat(rays)


def splats_of(prediction, rays, distance=4.0):
    """Gaussians around the point of each token's ray nearest the origin's depth."""
    start = (rays[:, :3] + distance * rays[:, 3:])[:, None]
    p = prediction
    means = (start + 0.5 * p[..., :3]).reshape(-1, 3)
    log_scales = (p[..., 3:6] - 1.8).reshape(-1, 3)
    quats = (p[..., 6:10] + torch.tensor([1.0, 0, 0, 0], device=p.device)).reshape(-1, 4)
    return means, quats, log_scales, p[..., 10].reshape(-1), p[..., 11:].sigmoid().reshape(-1, 3)


def offsets_of(lengths, device="cuda"):
    return torch.tensor([0, *torch.tensor(lengths).cumsum(0).tolist()], dtype=torch.int32,
                        device=device)


def extend(net, scene_tokens, positions, old, device="cuda"):
    """The prediction of tokens `old` .. of one scene, run in two parts: the first
    `old` tokens, then the rest over the memory of their keys and values."""
    memory, n = [], scene_tokens.shape[0]
    with torch.no_grad():
        net(scene_tokens[:old], positions[:old], offsets_of([old], device), causal=True,
            memory=memory)
        return net(scene_tokens[old:], positions[old:], offsets_of([n - old], device),
                   offsets_of([n], device), causal=True, memory=memory)


def candidates(net, scene_tokens, positions, views, device="cuda"):
    """The predictions of several views, (tokens, positions) each, of one scene: each
    view over the scene's memory, read once for all, and none seeing another."""
    memory, n = [], scene_tokens.shape[0]
    with torch.no_grad():
        net(scene_tokens, positions, offsets_of([n], device), causal=True, memory=memory)
        tokens, at = (torch.cat(t) for t in zip(*views))
        lengths = [t.shape[0] for t, _ in views]
        out = net(tokens, at, offsets_of(lengths, device), causal=True, shared=memory)
    return out.split(lengths)


def with_frames(positions, length):
    """(frame, column, row) of the tokens of frames of `length` tokens each."""
    frame = torch.arange(positions.shape[0], device=positions.device) // length
    return torch.cat([frame[:, None].to(positions), positions], 1)


def train(steps=60, size=64, views=(2, 4, 3), seed=0, lr=2e-3, device="cuda", log=print):
    """Returns (network, losses, packed inputs)."""
    scenes = [make_scene(v, size, seed + i, device) for i, v in enumerate(views)]
    packed = [tokens_of(images[:-1], cams[:-1], size) for images, cams in scenes]
    tokens, positions, rays = (torch.cat(t) for t in zip(*packed))
    lengths = [p[0].shape[0] for p in packed]
    offsets = offsets_of(lengths, device)
    net = Network(seed=seed, device=device)
    opt = mg.FusedAdam([{"params": list(net.params.values())}], lr=lr, eps=1e-8)
    window = mg.gaussian_kernel(device=device, groups=15)
    losses = []
    for step in range(steps):
        prediction = net(tokens, positions, offsets, causal=True)
        loss = 0.0
        at = 0
        for n, (images, cams) in zip(lengths, scenes):
            means, quats, log_scales, logits, colors = splats_of(prediction[at:at + n],
                                                                 rays[at:at + n])
            at += n
            K, vm = cams[-1]
            rgb, _, _ = mg.render(means, quats, log_scales, logits, None, K, vm, size, size,
                                  colors=colors, activations=True)
            loss = loss + mg.photometric_loss(rgb, images[-1], window)[0] / len(scenes)
        opt.zero_grad(set_to_none=True)
        loss.backward()
        opt.step()
        losses.append(float(loss.detach()))
        if step % 10 == 0 or step == steps - 1:
            log(f"step {step:4d}  loss {losses[-1]:.4f}")
    return net, losses, (tokens, positions, lengths)


def main():
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--steps", type=int, default=60)
    ap.add_argument("--seed", type=int, default=0)
    a = ap.parse_args()
    net, _, (tokens, positions, lengths) = train(a.steps, seed=a.seed)
    n = lengths[0]
    with torch.no_grad():
        whole = net(tokens[:n], positions[:n], offsets_of([n]), causal=True)
    new = extend(net, tokens[:n], positions[:n], n // 2)
    print(f"a view added over the memory: {float((new - whole[n // 2:]).abs().max()):.4f} from "
          "the whole scene's prediction at once")


if __name__ == "__main__":
    main()
