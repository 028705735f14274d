"""Speculative decoding over the compressed cache, on a small random model.

    python examples/tree_decode.py [--tokens 64] [--layers 2] [--temperature 0.7]

Each step drafts a tree of tokens from what followed the last token before,
runs all of its nodes through the layers in one pass (AttentionLayer.verify:
one tree attention a layer), samples the next token at every node, keeps the
path that the samples confirm (DraftTree.accept) and drops the other nodes'
cached rows (AttentionLayer.accept). The random numbers belong to positions,
so the tokens are those that decoding one at a time draws, which the second
run does.
"""

from __future__ import annotations

import argparse
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
from insitu_b200 import AttentionLayer, DraftTree, QuantConfig, Sampler  # noqa: E402


class Model:
    """Embedding, attention layers with residuals, a tied head. Weights are
    random, with a token's successor made likely, as text is."""

    def __init__(self, layers: int, vocab: int, capacity: int, seed: int = 0):
        rng = np.random.default_rng(seed)
        hidden, heads, kv = 256, 4, 2
        w = lambda *s: rng.standard_normal(s, dtype=np.float32) * 0.02
        self.layers = [AttentionLayer(w(heads * 64, hidden), w(kv * 64, hidden), w(kv * 64, hidden),
                                      w(hidden, heads * 64), hidden=hidden, num_heads=heads, num_kv_heads=kv,
                                      quant=QuantConfig(key_bits=4, value_bits=2), max_position=capacity,
                                      capacity=capacity) for _ in range(layers)]
        self.embed = torch.from_numpy(rng.standard_normal((vocab, hidden), dtype=np.float32)).cuda()
        follows = torch.from_numpy(rng.permutation(vocab)).cuda()
        self.head = torch.empty_like(self.embed)
        self.head[follows] = self.embed * 0.05

    def logits(self, tokens, tree: DraftTree) -> torch.Tensor:
        """Logits after each node of the tree; its rows stay in the caches."""
        x = self.embed[torch.as_tensor(tokens, device="cuda")]
        for layer in self.layers:
            x = x + layer.verify(x, tree)[0]
        return x @ self.head.T

    def keep(self, path) -> None:
        for layer in self.layers:
            layer.accept(path)

    def close(self) -> None:
        for layer in self.layers:
            layer.close()


def draft(last: int, seen: dict, depth: int, width: int):
    """A tree of guesses: the last token, then what followed each token
    before, the latest first. Returns (tokens, parents)."""
    tokens, parents, level = [last], [-1], [0]
    for _ in range(depth):
        nxt = []
        for node in level:
            for t in seen.get(tokens[node], [])[-1:-1 - width:-1]:
                nxt.append(len(tokens))
                tokens.append(t)
                parents.append(node)
        level = nxt[:4]
    return tokens, parents


def generate(model: Model, first: int, n: int, uniform: torch.Tensor, sampler: Sampler, *, depth: int = 4,
             width: int = 2):
    """n tokens after `first`; depth 0 decodes one at a time. Returns the
    tokens and the number of passes."""
    out, seen, passes = [first], {}, 0
    while len(out) <= n:
        tokens, parents = draft(out[-1], seen, depth, width)
        tree = DraftTree([parents])
        logits = model.logits(tokens, tree)
        # the node at depth d stands at position len(out) + d - 2 and draws the token after it
        at = torch.as_tensor(len(out) - 1 + tree.depths - 1, device="cuda")
        sampled = sampler(logits, uniform[at])[0].tolist()
        path, extra = tree.accept(0, tokens, sampled, first=out[-1])
        model.keep(path)
        new = [tokens[i] for i in path[1:]] + [extra]
        for a, b in zip([out[-1]] + new, new):
            seen[a] = [t for t in seen.get(a, []) if t != b] + [b]
        out += new
        passes += 1
    return out[1:n + 1], passes


def main(argv=None) -> int:
    ap = argparse.ArgumentParser()
    ap.add_argument("--tokens", type=int, default=64)
    ap.add_argument("--layers", type=int, default=2)
    ap.add_argument("--vocab", type=int, default=64)
    ap.add_argument("--temperature", type=float, default=0.7)
    a = ap.parse_args(argv)
    g = torch.Generator("cuda").manual_seed(1)
    uniform = torch.rand((a.tokens + 16, a.vocab), generator=g, device="cuda")
    sampler = Sampler(temperature=a.temperature, top_k=20, top_p=0.95)
    runs = []
    for depth in (4, 0):
        model = Model(a.layers, a.vocab, capacity=a.tokens + 64)
        tokens, passes = generate(model, 3, a.tokens, uniform, sampler, depth=depth)
        model.close()
        runs.append(tokens)
        print(f"{'drafted trees' if depth else 'one at a time'}: {len(tokens)} tokens in {passes} passes")
    print("the same tokens" if runs[0] == runs[1] else f"they part at token "
          f"{next(i for i, (x, y) in enumerate(zip(*runs)) if x != y)}")
    return 0 if runs[0] == runs[1] else 1


if __name__ == "__main__":
    sys.exit(main())
