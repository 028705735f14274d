"""Waits for copies give up after about a second by default: what would never
complete ends in seconds, with a status and without a fault."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu


def timed(call):
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    call()
    end.record()
    torch.cuda.synchronize()
    return begin.elapsed_time(end) / 1000


@pytest.mark.parametrize("operator", ["scan", "tree"])
def test_a_wait_for_copies_lasts_about_a_second(operator):
    """Twice that in all: the wait, and the one for the copies in flight."""
    from insitu_b200 import DraftTree, Geometry, PagedCache, QuantConfig
    from insitu_b200._lib import DeviceTimeout
    rng = np.random.default_rng(1)
    pc = PagedCache(QuantConfig(key_bits=4, value_bits=2), geo=Geometry(8, 4, 64), max_seqs=1, capacity=40000)
    pc.put_rows([0], [40000], torch.from_numpy(rng.integers(0, 256, (40000, 8, 52), dtype=np.uint8)).to(pc.device))
    q = torch.from_numpy(np.rint(rng.standard_normal((1, 32, 64)) * 8192).astype(np.int32)).to(pc.device)
    tree = DraftTree([[-1]])
    call = (lambda: pc.scan([0], q)) if operator == "scan" else (lambda: pc.tree_scan([0], q, tree))
    call()
    pc.status()
    pc.set_wait_test(item=3, chunk=2, head=0)
    seconds = timed(call)
    with pytest.raises(DeviceTimeout):
        pc.status()
    pc.set_wait_test()
    assert 0.2 < seconds < 6
    call()
    pc.status()
    pc.close()
