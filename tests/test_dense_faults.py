"""Spans of rows that are not there are refused before anything of their size is allocated."""

from __future__ import annotations

import numpy as np
import pytest

from test_tree import make, random_rows

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("read", ["dense", "rows"])
def test_more_rows_than_memory_holds_are_refused_as_any_that_are_not_cached(read):
    """2^31 - 1 rows of a sequence of 10 would be hundreds of gigabytes."""
    from insitu_b200._lib import ArgumentError, CapacityError
    pc = make(4, 2, 2, 4, 16, 64, 2)
    pc.put_rows([0], [10], torch.from_numpy(random_rows(np.random.default_rng(1), pc, 10)).to(pc.device))
    call = getattr(pc, read)
    call([0], 0, 10)
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    for args in (([0], 0, 11), ([0], 0, 2 ** 31 - 1), ([0, 0, 1], 0, [10, 2 ** 31 - 1, 0]), ([0], 0, 2 ** 40),
                 ([0], 2 ** 40, 0), ([0], -1, 5), ([0], 4, -1), ([0, 1], [0, 0], [10, 1])):
        with pytest.raises(CapacityError):
            call(*args)
    for seq in (2, -1):
        with pytest.raises(ArgumentError):
            call([seq], 0, 2 ** 31 - 1)
    assert torch.cuda.max_memory_allocated() == before
    pc.close()
    with pytest.raises((ValueError, RuntimeError)):
        call([0], 0, 10)
