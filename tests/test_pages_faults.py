"""Calls of the page operations that once went wrong: each is refused, or
gives what its definition says, and the pool's bookkeeping stays whole."""

from __future__ import annotations

import numpy as np
import pytest

from test_pages import append, check, make, random_rows

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("spare", [0, 1, 5])
def test_a_fork_whose_source_is_also_a_target_is_refused(spare):
    """Sequence 1 is empty when the call is checked and a copy of sequence 0
    when its own fork would run: its page was never counted (with none to spare
    the free list ran empty), and its rows were read while being written."""
    pc = make(4, 2, 2, 16, capacity=64, max_seqs=4, n_pages=2 + spare)
    rows = random_rows(np.random.default_rng(spare), pc, 20)
    append(pc, 0, rows)
    for src, dst, lens in (([0, 1], [1, 2], None), ([1, 0], [2, 1], None), ([0, 1], [1, 2], [16, 0]),
                           ([0, 1, 2], [1, 2, 3], None), ([1], [1], None), ([0], [0], None)):
        with pytest.raises(ValueError):
            pc.fork(src, dst, lens)
    check(pc, {0: rows})
    assert [pc.length(s) for s in (1, 2, 3)] == [0, 0, 0] and pc.free_pages == spare
    pc.fork([0, 0], [1, 2], [16, 0])               # two targets of one source
    check(pc, {0: rows, 1: rows[:16]})
    pc.truncate([0, 1], 0)
    assert pc.free_pages == 2 + spare
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("change", ["truncate", "compact", "reset"])
def test_a_context_split_does_not_outlive_its_rows(change):
    """Between the phases rows are dropped and as many others appended: the
    maxima are of rows that are gone, so the second phase is refused. Changes
    of other sequences, and rows only added, leave it."""
    from insitu_b200 import Geometry, PagedCache, QuantConfig
    rng = np.random.default_rng(3)
    pc = PagedCache(QuantConfig(key_bits=4, value_bits=2), geo=Geometry(2, 4, 64), max_seqs=3, capacity=4096)
    wire = lambda s, *shape: torch.from_numpy(np.rint(rng.standard_normal(shape) * s * 65536).astype(np.int32)).cuda()
    q = wire(0.25, 1, 8, 64)
    for s in (0, 1):
        pc.ingress([s] * 3000, wire(1, 3000, 2, 64), wire(1, 3000, 2, 64))
    maxima = pc.scan_maxima([0], q, lengths=[3000])
    pc.truncate([1], 2000)
    pc.compact([1], [list(range(0, 2000, 3))])
    pc.fork([0], [2])
    pc.ingress([0] * 10, wire(1, 10, 2, 64), wire(1, 10, 2, 64))
    want = pc.scan_part([0], torch.full_like(maxima, pc.S_LO), lengths=[3000])
    maxima = pc.scan_maxima([0], q, lengths=[3000])
    if change == "truncate":
        pc.truncate([0], 2900)
    elif change == "compact":
        pc.compact([0], [[i for i in range(3010) if i % 50]])
    else:
        pc.reset(0)
    pc.ingress([0] * 3010, wire(1, 3010, 2, 64), wire(1, 3010, 2, 64)) if change == "reset" else \
        pc.ingress([0] * 200, wire(1, 200, 2, 64), wire(1, 200, 2, 64))
    with pytest.raises(ValueError):
        pc.scan_part([0], torch.full_like(maxima, pc.S_LO), lengths=[3000])
    again = pc.scan_maxima([2], q, lengths=[3000])          # the fork has kept the rows
    got = pc.scan_part([2], torch.full_like(again, pc.S_LO), lengths=[3000])
    torch.cuda.synchronize()
    assert got.shape == want.shape
    pc.status()
    pc.close()
