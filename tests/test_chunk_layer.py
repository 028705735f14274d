"""Layers that attend in floating point, and a run of the operators together."""

from __future__ import annotations

import os
import sys

import numpy as np
import pytest

from conftest import ROOT

torch = pytest.importorskip("torch")


def make_layer(seed=0, capacity=1024, **kw):
    from insitu_b200 import AttentionLayer, QuantConfig
    rng = np.random.default_rng(seed)
    w = lambda *s: rng.standard_normal(s, dtype=np.float32) * 0.05
    return AttentionLayer(w(256, 256), w(128, 256), w(128, 256), w(256, 256), hidden=256, num_heads=4, num_kv_heads=2,
                          quant=QuantConfig(key_bits=4, value_bits=2), capacity=capacity, max_position=1024, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 300])
def test_a_float_layer_agrees_with_the_fixed_point_one(n):
    """The same cache, byte for byte, and outputs within 2^-6 (the fixed-point
    scan's 2^-15 probabilities and the bf16 attention output, then the same
    fp16 projection)."""
    rng = np.random.default_rng(5)
    xs = rng.standard_normal((n, 256)).astype(np.float32)
    one, two = make_layer(softmax="float"), make_layer(softmax="two_pass")
    y, out = one.forward(xs)
    want, _ = two.forward(xs)
    assert out.dtype == torch.bfloat16 and out.shape == (n, 256)
    assert torch.equal(one.dec.pc.rows([0]), two.dec.pc.rows([0]))
    assert float((y - want).norm() / want.norm()) <= 2.0 ** -6
    one.close()
    two.close()


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(None, 0), (100, 4), (1, 0)])
def test_chunks_of_any_size_leave_one_cache_and_like_outputs(window, sinks):
    """Rows are written token by token whatever the chunk; outputs are those of
    other roundings, each within bf16's 2^-9 and the projection of them."""
    rng = np.random.default_rng(6)
    xs = rng.standard_normal((420, 256)).astype(np.float32)
    whole = make_layer(softmax="float", window=window, sinks=sinks)
    want, _ = whole.forward(xs)
    for chunk in (1, 33, 200):
        layer = make_layer(softmax="float", window=window, sinks=sinks)
        got = torch.cat([layer.forward(xs[i:i + chunk])[0] for i in range(0, 420, chunk)])
        assert torch.equal(layer.dec.pc.rows([0]), whole.dec.pc.rows([0]))
        assert float((got - want).norm() / want.norm()) <= 2.0 ** -6
        layer.close()
    whole.close()


@pytest.mark.gpu
def test_layer_refusals():
    for kw in (dict(softmax="exact"), dict(window=5), dict(softmax="online", sinks=2),
               dict(softmax="float", window=0), dict(softmax="float", window=5, sinks=-1)):
        with pytest.raises(ValueError):
            make_layer(**kw)
    from insitu_b200 import DraftTree
    layer = make_layer(softmax="float", window=5)
    with pytest.raises(ValueError):
        layer.verify(np.zeros((1, 256), np.float32), DraftTree([[-1]]))
    layer.close()


@pytest.mark.gpu
def test_the_example_runs(capsys):
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    import chunked_prompt
    assert chunked_prompt.main(["--prompt", "300", "--tokens", "12"]) == 0
    said = capsys.readouterr().out
    assert said.count("12 tokens") == 3 and "NOT as" not in said, said
