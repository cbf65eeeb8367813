"""The patch network of examples/patch_splats.py: layer norm, rotary positions and
attention with their gradients, the renderer, its loss and FusedAdam together."""

from __future__ import annotations

import importlib.util

import pytest
import torch

from conftest import ROOT

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("patch_splats",
                                                  ROOT / "examples" / "patch_splats.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def test_training_lowers_the_loss_and_scenes_stay_apart(dev, example):
    net, losses, (tokens, positions, lengths) = example.train(steps=40, log=lambda s: None)
    assert all(x == x for x in losses)
    assert losses[-1] < 0.7 * losses[0], losses
    # A scene predicted alone is the scene predicted among others.
    n = lengths[0]
    with torch.no_grad():
        packed = net(tokens, positions, example.offsets_of(lengths), causal=True)
        alone = net(tokens[:n], positions[:n], example.offsets_of([n]), causal=True)
    # The products' tiles may differ with the number of rows: bfloat16 rounding
    # (2^-8) of activations of size one, through two blocks.
    assert float((packed[:n] - alone).abs().max()) < 0.1


def test_new_tokens_over_the_memory(dev, example):
    net = example.Network(seed=3)
    images, cams = example.make_scene(3, 64, 5)
    tokens, positions, _ = example.tokens_of(images, cams, 64)
    n = tokens.shape[0]
    with torch.no_grad():
        whole = net(tokens, positions, example.offsets_of([n]), causal=True)
    for old in (1, n // 2, n - 1):
        new = example.extend(net, tokens, positions, old)
        assert new.shape == whole[old:].shape
        assert float((new - whole[old:]).abs().max()) < 0.1
