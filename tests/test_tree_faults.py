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


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 3, 6, 24, 64])
@pytest.mark.parametrize("tile", [0, 1, 21])
def test_a_wait_for_rows_that_runs_out_is_reported_and_the_context_survives(nodes, tile):
    """One tile's copies are announced 16 bytes larger than they are, so the
    wait for them cannot complete: it gives up after the lowered limit, the
    launch ends, the status is INS_ETIMEOUT, and the next scan is what it was.
    Every copy lands; nothing faults."""
    from insitu_b200 import DraftTree
    from insitu_b200._lib import DeviceTimeout
    rng = np.random.default_rng(nodes)
    pc = make(4, 2, 8, 4, 256, 60160, 1)
    pc.put_rows([0], [60001], torch.from_numpy(random_rows(rng, pc, 60001)).to(pc.device))
    q = torch.from_numpy(np.rint(rng.standard_normal((nodes, 32, 64)) * 16384).astype(np.int32)).to(pc.device)
    tree = DraftTree([random_tree(rng, nodes)])
    want = pc.tree_scan([0], q, tree)
    pc.status()
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    for cta in (0, 77):
        pc.set_wait_test(poll_limit=4096, item=cta, chunk=tile)
        begin.record()
        pc.tree_scan([0], q, tree)
        end.record()
        with pytest.raises(DeviceTimeout):
            pc.status()
        print(f"{nodes} nodes, tile {tile} of CTA {cta}: {begin.elapsed_time(end):.2f} ms")
        pc.set_wait_test()
        assert torch.equal(pc.tree_scan([0], q, tree).view(torch.int16), want.view(torch.int16))
        pc.status()
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("then", ["forward", "verify"])
def test_drafted_nodes_that_no_accept_kept_are_not_context(then):
    """A verify whose nodes all fell, then the next step without an accept of
    nothing: the siblings' rows are no tokens of the sequence."""
    from insitu_b200 import DraftTree
    from test_tree_layer import make_layer
    rng = np.random.default_rng(8)
    xs, drafted, x = (rng.standard_normal((n, 256)).astype(np.float32) for n in (40, 5, 1))
    layer, plain = make_layer(), make_layer()
    for m in (layer, plain):
        m.forward(xs)
    layer.verify(drafted, DraftTree([[-1, 0, 0, -1, 3]]))
    if then == "forward":
        got, want = layer.forward(x)[0], plain.forward(x)[0]
    else:
        one = DraftTree([[-1]])
        got, want = layer.verify(x, one)[0], plain.verify(x, one)[0]
        layer.accept([0])
        plain.accept([0])
    assert layer.dec.pc.length(0) == 41
    assert torch.equal(got, want) and torch.equal(layer.dec.pc.rows([0]), plain.dec.pc.rows([0]))
    layer.close()
    plain.close()


@pytest.mark.gpu
def test_a_verify_whose_scan_fails_leaves_no_rows_behind(monkeypatch):
    """Its rows are appended before the scan: an error there (no memory for the
    partial sums) must not make them context."""
    from insitu_b200 import DraftTree
    from test_tree_layer import make_layer
    rng = np.random.default_rng(8)
    xs, drafted, x = (rng.standard_normal((n, 256)).astype(np.float32) for n in (40, 5, 1))
    layer, plain = make_layer(), make_layer()
    for m in (layer, plain):
        m.forward(xs)

    def no_memory(*args):
        raise torch.cuda.OutOfMemoryError("no memory")

    monkeypatch.setattr(layer.dec.pc, "tree_scan", no_memory)
    with pytest.raises(torch.cuda.OutOfMemoryError):
        layer.verify(drafted, DraftTree([[-1, 0, 0, -1, 3]]))
    monkeypatch.undo()
    got, want = layer.forward(x)[0], plain.forward(x)[0]
    assert layer.dec.pc.length(0) == 41
    assert torch.equal(got, want) and torch.equal(layer.dec.pc.rows([0]), plain.dec.pc.rows([0]))
    layer.close()
    plain.close()


@pytest.mark.gpu
def test_a_refusal_has_its_own_error():
    """A tree of more nodes than the sequence has rows is a matter of length,
    as the scans' lengths are; a sequence that is not there is an argument."""
    from insitu_b200 import DraftTree
    from insitu_b200._lib import ArgumentError, CapacityError
    pc = make(4, 2, 2, 4, 16, 64, 2)
    pc.put_rows([0], [2], torch.zeros((2, 2, 52), dtype=torch.uint8, device=pc.device))
    q = torch.zeros((3, 8, 64), dtype=torch.int32, device=pc.device)
    tree = DraftTree([[-1, 0, 1]])
    with pytest.raises(CapacityError, match="fewer than its tree"):
        pc.tree_scan([0], q, tree)
    with pytest.raises(ArgumentError, match="out of range"):
        pc.tree_scan([5], q, tree)
    pc.close()
