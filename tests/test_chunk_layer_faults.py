"""A chunk whose attention is refused or fails leaves the cache as it was."""

from __future__ import annotations

import numpy as np
import pytest

from test_chunk_layer import make_layer

torch = pytest.importorskip("torch")


class FakeCache:
    """What chunk_attend calls of a PagedCache, with a scan that fails once."""

    def __init__(self):
        self.len, self.fails = 7, 1

    def length(self, seq):
        return self.len

    def ingress(self, ids, k, v, q):
        self.len += len(ids)
        return q

    def chunk_scan(self, ids, q, n, window=None, sinks=0):
        self.fails -= 1
        if self.fails >= 0:
            raise torch.OutOfMemoryError("no room for a workspace")
        return q

    def truncate(self, ids, lengths):
        (self.len,) = lengths


def test_rows_of_a_chunk_whose_scan_fails_are_dropped():
    """Called again, the same tokens would else be in the context twice."""
    from insitu_b200.decode import DecodeAttention
    dec = DecodeAttention.__new__(DecodeAttention)
    dec.pc = FakeCache()
    q, k = torch.zeros(3, 8, 64), torch.zeros(3, 2, 64)
    with pytest.raises(torch.OutOfMemoryError):
        dec.chunk_attend(0, q, k, k)
    assert dec.pc.len == 7
    assert dec.chunk_attend(0, q, k, k) is q and dec.pc.len == 10


@pytest.mark.gpu
def test_a_refused_chunk_leaves_the_cache_and_the_next_one_is_what_it_was():
    rng = np.random.default_rng(6)
    xs = rng.standard_normal((60, 256)).astype(np.float32)
    layer, whole = make_layer(softmax="float"), make_layer(softmax="float")
    want = torch.cat([whole.forward(xs[i:i + 20])[0] for i in (0, 20, 40)])
    got = [layer.forward(xs[:20])[0]]
    layer.window = 0                                            # which chunk_scan refuses, after the rows went in
    with pytest.raises(ValueError):
        layer.forward(xs[20:40])
    layer.window = None
    assert layer.dec.pc.length(0) == 20
    got += [layer.forward(xs[i:i + 20])[0] for i in (20, 40)]
    assert torch.equal(torch.cat(got), want)
    assert torch.equal(layer.dec.pc.rows([0]), whole.dec.pc.rows([0]))
    for x in (layer, whole):
        x.close()
