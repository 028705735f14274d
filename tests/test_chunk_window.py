"""Chunks of many query rows under a window without sinks: the later tokens of a
row tile see nothing of its first tiles, whatever their scores.

The bound is that of test_tree.py with the output's rounding in full: bf16 keeps 8
bits, so a value in [2^e, 2^(e+1)) lies within half of its step 2^(e-7), which is
2^-8 of the value and not 2^-9 (1.07413 and 1.07422 round to numbers 0.0078 apart).

Some scores are shifted as a whole. Every key holds the same value in channel 0
(one code, one norm), so its product with a query is one number, rounded once and
alike for every key, and the softmax does not depend on it: the reference leaves
channel 0 out. What is left of a shift of S nats is the fp32 sum of 64 products,
at most 68 additions of 2^-23 of the largest partial sum: with z = sum|q k| of the
other channels a score is off by 2^-16 (S + z) at most, a weight by twice that
relatively (numerator and denominator)."""

from __future__ import annotations

import numpy as np
import pytest

from test_chunk import visible
from test_tree import decode, make, random_rows, reference

torch = pytest.importorskip("torch")


def attend(context, n, n_kv, groups, window, scores, kb=4, vb=2, sinks=0, page=64, step=128):
    seed = context + n + 7 * window + 31 * groups
    rng = np.random.default_rng(seed)
    pc = make(kb, vb, n_kv, groups, page, context + n, 1)
    rows = random_rows(rng, pc, context + n)
    spread, shift, own, rise = scores
    level = lambda i: float(pc.tables.k_centroids[i]) / 32768  # noqa: E731
    top = (1 << kb) - 1
    if shift:
        rows[..., 0] |= top
        rows[..., -4:-2] = np.frombuffer(np.array(512, "<i2").tobytes(), np.uint8)
    if rise:
        code = np.arange(context + n) * (top + 1) // (context + n)
        rows[..., 0] = (rows[..., 0] & ~np.uint8(top)) | code[:, None].astype(np.uint8)
    k, v = decode(pc, rows)
    # scores of `spread` nats' deviation: 64 products with keys of mean square 1
    q = rng.standard_normal((n, n_kv, groups, 64)) * spread / 8
    last = k[context:, :, None]
    if own:                                                    # a token's own key, so many nats up
        q += own * last / (last ** 2).sum(-1, keepdims=True)
    if shift:
        q[..., 0] = shift / level(top)
    if rise:
        q[..., 0] = rise / (level(top) - level(0))
    q = np.rint(q * 65536).astype(np.int32)
    pc.put_rows([0], [context + n], torch.from_numpy(rows).to(pc.device))
    got = pc.chunk_scan([0], torch.from_numpy(q.reshape(n, -1, 64)).to(pc.device), n, window=window, sinks=sinks)
    pc.status()
    got = got.float().cpu().numpy().reshape(q.shape)
    pc.close()
    x = q / 65536.0
    if shift:
        x[..., 0] = 0.0
    see = visible(context, n, window, sinks)
    reach = np.abs(v).max()
    for a in range(0, n, step):
        b = min(n, a + step)
        lo = max(0, context + a - window + 1) if not sinks else 0
        want, bound = reference(x[a:b], k[lo:], v[lo:], see[a:b, lo:])
        bound = bound + 2.0 ** -9 * np.abs(want)
        if shift:
            z = np.abs(x[a:b]).sum(-1, keepdims=True) * np.abs(k).max()
            bound = bound + 2 * 2.0 ** -16 * (abs(shift) + z) * reach
        off = np.abs(got[a:b] - want)
        assert (off <= bound).all(), f"tokens {a} on: {(~(off <= bound)).any(-1).sum()} rows off, by {(off - bound).max()}"
        assert np.linalg.norm(off) <= 2.0 ** -8 * np.linalg.norm(want) + 1e-7


# (deviation, shift, own key, rise) in nats
SCORES = [(0.0, 0, 0, 0), (0.16, 0, 0, 0), (0.5, 0, 0, 0), (1.0, 0, 0, 0), (2.0, 0, 0, 0), (0.5, 0, 4, 0), (1.0, 0, 4, 0),
          (0.5, -30, 0, 0), (0.5, -100, 0, 0), (0.5, 60, 0, 0), (0.5, 0, 0, 6), (0.5, 0, 0, -6)]


@pytest.mark.gpu
@pytest.mark.parametrize("scores", SCORES)
@pytest.mark.parametrize("context,n,n_kv,groups,window", [
    (2000, 256, 2, 4, 1000), (3001, 520, 2, 2, 1500), (8191, 600, 1, 1, 1024), (5003, 1024, 2, 1, 2000),
    (1000, 200, 3, 8, 129), (0, 1300, 2, 2, 300), (5003, 300, 1, 8, 2000)])
def test_rows_that_see_nothing_of_their_first_tiles(context, n, n_kv, groups, window, scores):
    """Row tiles whole and in pieces, of 32 to 256 tokens."""
    attend(context, n, n_kv, groups, window, scores)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", SCORES[2:9])
@pytest.mark.parametrize("kb,vb", [(3, 3), (2, 4)])
def test_other_widths(kb, vb, scores):
    attend(2500, 260, 2, 4, 700, scores, kb, vb)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", SCORES[2:9])
@pytest.mark.parametrize("sinks", [0, 4])
def test_a_long_window_in_pieces(sinks, scores):
    attend(8192, 512, 8, 4, 4000, scores, sinks=sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("scores", SCORES[2:9])
@pytest.mark.parametrize("n", [1, 9, 60, 128])
def test_short_chunks(n, scores):
    attend(2000, n, 2, 4, 700, scores)
