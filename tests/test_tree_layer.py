"""A layer's drafted-tree pass and the example that runs it end to end."""

from __future__ import annotations

import os
import sys

import numpy as np
import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")


def make_layer(seed=0, capacity=256):
    from insitu_b200 import AttentionLayer, QuantConfig
    rng = np.random.default_rng(seed)
    w = lambda *s: rng.standard_normal(s, dtype=np.float32) * 0.05
    return AttentionLayer(w(256, 256), w(128, 256), w(128, 256), w(256, 256), hidden=256, num_heads=4, num_kv_heads=2,
                          quant=QuantConfig(key_bits=4, value_bits=2), capacity=capacity, max_position=1024)


@pytest.mark.gpu
def test_verify_and_accept_give_the_layer_decoded_token_by_token():
    """A tree's accepted path leaves the cache that decoding the path's inputs
    one at a time leaves, byte for byte; the outputs agree with the
    fixed-point layer within 2^-6 (bf16 attention outputs, 2^-15 fixed-point
    probabilities, then the same fp16 projection)."""
    from insitu_b200.tree import DraftTree
    rng = np.random.default_rng(5)
    xs = rng.standard_normal((40, 256)).astype(np.float32)
    parents = [-1, 0, 0, 1, 1, 3, 2]
    path = [0, 1, 3, 5]
    drafted = rng.standard_normal((7, 256)).astype(np.float32)
    tree_layer, plain = make_layer(), make_layer()
    for layer in (tree_layer, plain):
        layer.forward(xs)
    y, out = tree_layer.verify(drafted, DraftTree([parents]))
    assert y.shape == (7, 256) and out.shape == (7, 4, 64) and out.dtype == torch.bfloat16
    tree_layer.accept(path)
    want = torch.cat([plain.forward(drafted[i:i + 1])[0] for i in path])
    for layer in (tree_layer, plain):
        layer.dec.pc.status()
        assert layer.dec.pc.length(0) == 44
    assert torch.equal(tree_layer.dec.pc.rows([0]), plain.dec.pc.rows([0]))
    err = float((y[path] - want).norm() / want.norm())
    assert err <= 2.0 ** -6, err
    tree_layer.close()
    plain.close()


@pytest.mark.gpu
def test_verify_and_accept_refuse_what_does_not_fit():
    from insitu_b200.tree import DraftTree
    layer = make_layer()
    x = np.zeros((3, 256), np.float32)
    with pytest.raises(RuntimeError):
        layer.accept([0])
    with pytest.raises(ValueError):
        layer.verify(x, DraftTree([[-1, 0]]))
    with pytest.raises(ValueError):
        layer.verify(x, DraftTree([[-1], [-1, 0]]))
    with pytest.raises(ValueError):
        layer.verify(x, DraftTree.from_mask([np.eye(3, dtype=bool)]))
    layer.verify(x, DraftTree([[-1, 0, 0]]))
    with pytest.raises(ValueError):
        layer.accept([2, 1])
    layer.accept([0, 2])
    assert layer.dec.pc.length(0) == 2
    layer.verify(x, DraftTree([[-1, 0, 0]]))
    layer.forward(x[:1])
    with pytest.raises(RuntimeError):
        layer.accept([0])
    layer.close()


@pytest.mark.gpu
def test_the_example_draws_the_tokens_of_decoding_one_at_a_time(capsys):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import tree_decode
    assert tree_decode.main(["--tokens", "48"]) == 0
    said = capsys.readouterr().out
    passes = [int(line.split(" passes")[0].split()[-1]) for line in said.splitlines() if "passes" in line]
    assert passes[0] < passes[1] == 48, said
