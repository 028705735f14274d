"""Tree attention where it once went wrong."""

from __future__ import annotations

import numpy as np
import pytest

from test_tree import make, random_rows, random_tree

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 12, 64])
def test_a_dropped_trees_mask_stays_while_another_stream_reads_it(nodes):
    """The tree is dropped and its memory asked for again while the scan of
    another stream has not begun."""
    from insitu_b200 import DraftTree
    rng = np.random.default_rng(nodes)
    pc = make(4, 2, 2, 4, 64, 700, 1)
    pc.put_rows([0], [nodes], torch.from_numpy(random_rows(rng, pc, nodes)).to(pc.device))
    q = torch.from_numpy(np.rint(rng.standard_normal((nodes, 8, 64)) * 16384).astype(np.int32)).to(pc.device)
    parents, other = [random_tree(rng, nodes)], torch.cuda.Stream()
    want = pc.tree_scan([0], q, DraftTree(parents))
    tree = DraftTree(parents)
    tree.mask(pc.device)
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        torch.cuda._sleep(200_000_000)
        got = pc.tree_scan([0], q, tree)
    del tree
    zeros = [torch.zeros(nodes, dtype=torch.int64, device="cuda") for _ in range(200)]
    torch.cuda.synchronize()
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
    del zeros
    pc.close()
