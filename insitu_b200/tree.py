"""Trees of drafted tokens: which node descends from which.

    from insitu_b200.tree import DraftTree
    tree = DraftTree([[-1, 0, 0, 1]])       # one sequence: a root, two children, a grandchild
    out = cache.tree_scan([0], q_rot, tree)
    path = tree.accept(0, drafted, sampled)

A tree is a list of parents: node i's parent is an earlier node, or -1 for a
node that follows the context's last token. ``DraftTree`` holds one tree for
each sequence of a batch; it depends on no cache and no length, so the same
object serves every step that drafts the same shape.
"""

from __future__ import annotations

import numpy as np
import torch

MAX_NODES = 256


class DraftTree:
    """Drafted trees of a batch of sequences, node after node.

    ``counts``: nodes of each tree; ``offsets``: the first node of each in the
    batch; ``depths``: each node's distance from the context (1 for a node
    whose parent is -1), so its position is context + depth - 1."""

    def __init__(self, parents):
        self.parents = [[int(p) for p in tree] for tree in parents]
        rows, depths = [], []
        for b, tree in enumerate(self.parents):
            if len(tree) > MAX_NODES:
                raise ValueError(f"tree {b} holds {len(tree)} nodes; at most {MAX_NODES}")
            seen, deep = [], []
            for i, p in enumerate(tree):
                if not -1 <= p < i:
                    raise ValueError(f"tree {b}: node {i}'s parent {p} is not -1 or an earlier node")
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
                deep.append((deep[p] if p >= 0 else 0) + 1)
            rows += seen
            depths += deep
        self._set(rows, [len(t) for t in self.parents])
        self.depths = np.asarray(depths, dtype=np.int64)

    @classmethod
    def from_mask(cls, masks) -> "DraftTree":
        """From each sequence's (nodes, nodes) truth values instead: row i
        names the drafted tokens that node i attends (any set; a node that
        attends none sees the context only). Such a tree has no parents."""
        self = cls.__new__(cls)
        rows, counts = [], []
        for b, m in enumerate(masks):
            m = np.asarray(m, dtype=bool)
            if m.ndim != 2 or m.shape[0] != m.shape[1] or m.shape[0] > MAX_NODES:
                raise ValueError(f"mask {b} must be (nodes, nodes) with at most {MAX_NODES} nodes, got {m.shape}")
            rows += [sum(1 << int(j) for j in np.flatnonzero(r)) for r in m]
            counts.append(len(m))
        self.parents = self.depths = None
        self._set(rows, counts)
        return self

    def _set(self, rows, counts):
        self.counts = counts
        self.offsets = np.concatenate([[0], np.cumsum(counts)]).astype(np.int64).tolist()
        words = max(1, -(-max(counts, default=1) // 64))
        host = np.array([[(r >> 64 * w) & (2 ** 64 - 1) for w in range(words)] for r in rows],
                        dtype=np.uint64).reshape(len(rows), words)
        self._mask = torch.from_numpy(host.view(np.int64).copy())

    def __len__(self) -> int:
        """Nodes of all trees."""
        return self.offsets[-1]

    def mask(self, device) -> torch.Tensor:
        """The nodes' masks, (nodes, words) int64 bit patterns, on ``device``.
        They are copied once (the host waits for it), and then ready for calls
        on every stream."""
        if self._mask.device != torch.device(device):
            self._mask = self._mask.to(device)
        return self._mask

    def accept(self, b: int, drafted, sampled, first: int) -> tuple[list, int]:
        """The path of tree ``b`` that sampling confirms. ``drafted``: the
        tokens of its nodes; ``sampled``: the token drawn at each node (what
        follows it); ``first``: the token drawn after the context itself. Walks
        from the context to the child whose drafted token is the drawn one, as
        far as there is one. Returns the path's nodes and the token drawn after
        its last (the step's extra token): exactly the tokens that drawing one
        at a time gives."""
        tree = self.parents[b]
        if len(drafted) != len(tree) or len(sampled) != len(tree):
            raise ValueError(f"tree {b} holds {len(tree)} nodes; drafted {len(drafted)}, sampled {len(sampled)}")
        path, at, token = [], -1, int(first)
        for i, p in enumerate(tree):          # a child comes after its parent
            if p == at and int(drafted[i]) == token:
                path.append(i)
                at, token = i, int(sampled[i])
        return path, token
