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
