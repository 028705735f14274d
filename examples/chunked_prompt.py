"""A long prompt in chunks, then tokens under penalties and a grammar.

    python examples/chunked_prompt.py --prompt 600 --tokens 32 --window 256

Every layer attends its compressed cache in floating point, under a window and
a few first tokens (``AttentionLayer(softmax="float")``). The prompt goes through
in chunks of several sizes, which leave the same caches; then each token is
drawn from logits that ``Penalties`` has changed: repeated tokens cost, and a
mask allows every second half of the vocabulary in turn.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from insitu_b200 import AttentionLayer, Penalties, QuantConfig, Sampler  # noqa: E402


class Model:
    """Embedding, attention layers with residuals, a head; random weights."""

    def __init__(self, layers: int, vocab: int, capacity: int, window: int | None, sinks: int, seed: int = 0):
        rng = np.random.default_rng(seed)
        hidden, heads, kv = 256, 4, 2
        w = lambda *s: rng.standard_normal(s, dtype=np.float32) * 0.05
        self.layers = [AttentionLayer(w(heads * 64, hidden), w(kv * 64, hidden), w(kv * 64, hidden),
                                      w(hidden, heads * 64), hidden=hidden, num_heads=heads, num_kv_heads=kv,
                                      quant=QuantConfig(key_bits=4, value_bits=2), max_position=capacity,
                                      capacity=capacity, softmax="float", window=window, sinks=sinks)
                       for _ in range(layers)]
        self.embed = torch.from_numpy(rng.standard_normal((vocab, hidden), dtype=np.float32)).cuda()
        self.head = torch.from_numpy(w(vocab, hidden)).cuda()

    def __call__(self, tokens) -> torch.Tensor:
        """Logits after the last of the tokens, which join the caches."""
        x = self.embed[torch.as_tensor(tokens, device="cuda")]
        for layer in self.layers:
            x = x + layer.forward(x)[0]
        return x[-1:] @ self.head.T

    def close(self) -> None:
        for layer in self.layers:
            layer.close()


def allowed(vocab: int, i: int) -> torch.Tensor:
    """The mask of the i-th drawn token: one half of the vocabulary."""
    ids = np.arange(-(-vocab // 32) * 32)
    bits = (ids < vocab) & ((ids < vocab // 2) == (i % 2 == 0))
    return torch.from_numpy(np.packbits(bits, bitorder="little").view(np.int32).copy()).cuda()


def generate(model: Model, prompt: list, n: int, chunk: int, uniform: torch.Tensor, vocab: int) -> list:
    penalties, sampler = Penalties(repetition=1.2, presence=0.3, frequency=0.2), Sampler(temperature=0.8, top_k=40)
    tokens = torch.full((1, len(prompt) + n), -1, dtype=torch.int64, device="cuda")
    tokens[0, :len(prompt)] = torch.tensor(prompt)
    prompts = torch.tensor([len(prompt)], dtype=torch.int32, device="cuda")
    for i in range(0, len(prompt), chunk):
        logits = model(prompt[i:i + chunk])
    for i in range(n):
        logits = penalties(logits, tokens, prompts=prompts, mask=allowed(vocab, i))
        token, _ = sampler(logits, uniform[i:i + 1])
        tokens[0, len(prompt) + i] = token[0]
        logits = model(token)
    return tokens[0, len(prompt):].tolist()


def main(argv=None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=600)
    ap.add_argument("--tokens", type=int, default=32)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=1000)
    ap.add_argument("--window", type=int, default=256)
    ap.add_argument("--sinks", type=int, default=4)
    a = ap.parse_args(argv)
    g = torch.Generator("cuda").manual_seed(1)
    uniform = torch.rand((a.tokens, a.vocab), generator=g, device="cuda")
    prompt = np.random.default_rng(2).integers(0, a.vocab, a.prompt).tolist()
    for chunk in (a.prompt, 100, 7):
        model = Model(a.layers, a.vocab, a.prompt + a.tokens, a.window or None, a.sinks)
        tokens = generate(model, prompt, a.tokens, chunk, uniform, a.vocab)
        rows = [layer.dec.pc.dense([0], dtype=torch.float32) for layer in model.layers]
        model.close()
        half = [int(t >= a.vocab // 2) for t in tokens]
        print(f"chunks of {chunk}: {len(tokens)} tokens, {len(set(tokens))} of them different, "
              f"{'as' if half == [i % 2 for i in range(len(half))] else 'NOT as'} the masks allow; "
              f"keys of the first layer: mean {float(rows[0][0].mean()):+.4f}")
    return 0


if __name__ == "__main__":
    sys.exit(main())
