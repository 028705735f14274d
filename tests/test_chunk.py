"""Attention of chunks of new tokens (causal, window, sinks) against its
definition in float64. The bound of one output is that of test_tree.py: the
products' operands (query, key, weight, value) are rounded to fp16 once each,
sums are fp32, the output is rounded to bf16."""

from __future__ import annotations

import numpy as np
import pytest

from test_tree import decode, make, random_rows, reference

torch = pytest.importorskip("torch")


def visible(context, n, window, sinks):
    """(n, context + n) truth values from the definition."""
    p = context + np.arange(n)[:, None]
    t = np.arange(context + n)[None]
    see = t <= p
    if window is not None:
        see &= (t > p - window) | (t < sinks)
    return see


def queries(rng, pc, n, scale=0.25):
    q = np.rint(rng.standard_normal((n, pc.geo.num_heads, 64)) * scale * 65536)
    return torch.from_numpy(np.clip(q, -2 ** 31, 2 ** 31 - 1).astype(np.int64).astype(np.int32)).to(pc.device)


def check(pc, seqs, rows, counts, q, window=None, sinks=0, near=True, step=512):
    """chunk_scan of `seqs` against the reference; rows[i] are the packed rows of seqs[i]."""
    g = pc.geo
    got = pc.chunk_scan(seqs, q, counts, window=window, sinks=sinks)
    assert got.dtype == torch.bfloat16 and got.shape == q.shape
    pc.status()
    got = got.float().cpu().numpy()
    lo = 0
    for r, n in zip(rows, counts):
        if n:
            k, v = decode(pc, r)
            see = visible(len(r) - n, n, window, sinks)
            qi = q[lo:lo + n].cpu().numpy().astype(np.float64).reshape(n, g.n_kv_heads, g.kv_groups, 64) / 65536
            for a in range(0, n, step):
                b = min(n, a + step)
                want, bound = reference(qi[a:b], k, v, see[a:b])
                have = got[lo + a:lo + b].reshape(want.shape)
                worst = (np.abs(have - want) - bound).max()
                assert worst <= 0, f"{n} tokens from {a} on of {len(r)}: {worst} over the bound"
                if near:
                    assert np.linalg.norm(have - want) <= 2.0 ** -8 * np.linalg.norm(want) + 1e-7
        lo += n


def run(kb, vb, n_kv, groups, page, contexts, counts, window=None, sinks=0, seed=0, scale=0.25, wild=False):
    rng = np.random.default_rng(seed)
    lens = [c + n for c, n in zip(contexts, counts)]
    pc = make(kb, vb, n_kv, groups, page, max(16, *lens), len(lens))
    rows = [random_rows(rng, pc, n, wild) for n in lens]
    for i in rng.permutation(len(lens)):
        if lens[i]:
            pc.put_rows([int(i)], [lens[i]], torch.from_numpy(rows[i]).to(pc.device))
    check(pc, list(range(len(lens))), rows, counts, queries(rng, pc, sum(counts), scale), window, sinks,
          near=scale <= 0.25 and not wild)
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kb,vb", [(4, 2), (3, 3), (1, 1), (2, 4), (5, 3), (8, 8)])
@pytest.mark.parametrize("n", [1, 3, 8, 21, 64, 130, 300])
def test_every_width(kb, vb, n):
    run(kb, vb, 2, 4, 64, [517], [n], seed=kb * 100 + n)
    run(kb, vb, 2, 4, 64, [517], [n], window=100, sinks=3, seed=kb * 100 + n + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 2, 4, 8])
@pytest.mark.parametrize("n", [1, 2, 5, 17, 33, 129, 257])
def test_every_group(groups, n):
    run(4, 2, 3, groups, 256, [1000], [n], seed=groups * 100 + n)
    run(4, 2, 3, groups, 256, [1000], [n], window=40, sinks=1, seed=groups * 100 + n)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("context", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 2051])
def test_context_lengths_around_every_boundary(page, context):
    run(4, 2, 1, 4, page, [context], [1], seed=context)
    run(3, 3, 1, 4, page, [context], [7], seed=context)
    run(4, 2, 2, 4, page, [context], [50], seed=context)
    run(4, 2, 1, 4, page, [context], [140], seed=context)


@pytest.mark.gpu
@pytest.mark.parametrize("sinks", [0, 1, 4, 127, 128, 129, 300])
@pytest.mark.parametrize("window", [1, 2, 31, 63, 64, 65, 127, 128, 129, 250, 1000])
def test_windows_and_sinks_around_every_boundary(window, sinks):
    for n in (1, 5, 40, 200):
        run(4, 2, 1, 4, 48, [900], [n], window=window, sinks=sinks, seed=window + sinks)
    run(4, 2, 1, 2, 48, [0], [700], window=window, sinks=sinks, seed=window + sinks)


@pytest.mark.gpu
@pytest.mark.parametrize("counts", [(1,) * 40, (5, 0, 64, 1, 17), (256, 130, 65), (700, 1, 0, 300), (8,) * 70])
@pytest.mark.parametrize("window", [None, 200])
def test_ragged_batches(counts, window):
    rng = np.random.default_rng(len(counts))
    contexts = [int(x) for x in np.exp(rng.uniform(0, np.log(5000), len(counts)))]
    contexts[0] = 0
    run(4, 2, 2, 4, 256, contexts, list(counts), window=window, sinks=4, seed=len(counts))
    run(3, 3, 2, 2, 32, contexts, list(counts), window=window, sinks=4, seed=len(counts) + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("n,groups", [(1, 4), (9, 4), (40, 8), (520, 2)])
@pytest.mark.parametrize("window", [None, 5000, 100_000])
def test_long_contexts(n, groups, window):
    run(4, 2, 1, groups, 256, [150_001], [n], window=window, sinks=5, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("kb,vb", [(4, 2), (2, 4)])
@pytest.mark.parametrize("context,n,window", [(0, 4500, None), (700, 3300, None), (3000, 2500, 300), (0, 3000, 64)])
def test_more_row_tiles_than_the_gpu_has_room_for(kb, vb, context, n, window):
    """Each SM takes many units, of a few tiles and of many."""
    run(kb, vb, 4, 4, 256, [context, 5], [n, 1200], window=window, sinks=4, seed=n)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 12, 60, 400])
@pytest.mark.parametrize("scale", [0.0, 4.0, 60.0])
def test_peaked_and_flat_scores(n, scale):
    run(4, 2, 2, 4, 64, [2000], [n], seed=n, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 12, 60, 400])
def test_any_norms(n):
    run(4, 2, 2, 4, 64, [700], [n], seed=n, scale=0.05, wild=True)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40, 400])
def test_pages_beyond_four_gigabytes(n):
    rng = np.random.default_rng(2)
    filler = 12 * 10 ** 6 // 256 * 256
    pc = make(4, 2, 8, 4, 256, filler, 2, n_pages=filler // 256 + 8)
    pc.put_rows([0], [filler], torch.zeros((filler, 8, 52), dtype=torch.uint8, device=pc.device))
    rows = random_rows(rng, pc, 900)
    pc.put_rows([1], [900], torch.from_numpy(rows).to(pc.device))
    check(pc, [1], [rows], [n], queries(rng, pc, n), window=700, sinks=2)
    check(pc, [1], [rows], [n], queries(rng, pc, n))
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20, 64, 500])
def test_it_is_the_tree_scan_of_a_chain(n):
    """The same definition: within both forms' roundings of one another."""
    from insitu_b200.tree import DraftTree
    rng = np.random.default_rng(n)
    pc = make(4, 2, 4, 4, 256, 4000, 1)
    rows = random_rows(rng, pc, 3500)
    pc.put_rows([0], [3500], torch.from_numpy(rows).to(pc.device))
    m = min(n, 200)
    q = queries(rng, pc, n)
    got = pc.chunk_scan([0], q, n)[n - m:]
    want = pc.tree_scan([0], q[n - m:], DraftTree([list(range(-1, m - 1))]))
    assert float((got.double() - want.double()).norm() / want.double().norm()) <= 2.0 ** -7
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20, 64, 500])
def test_runs_repeat_on_another_stream_and_in_a_graph(n):
    rng = np.random.default_rng(n)
    pc = make(4, 2, 8, 4, 256, 9000, 1)
    rows = random_rows(rng, pc, 8000)
    pc.put_rows([0], [8000], torch.from_numpy(rows).to(pc.device))
    q = queries(rng, pc, n)
    call = lambda: pc.chunk_scan([0], q, n, window=6000, sinks=4)
    first = call()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = [call() for _ in range(5)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = call()
    for _ in range(3):
        held.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again.append(held.clone())
    for x in again:
        assert torch.equal(first.view(torch.int16), x.view(torch.int16))
    pc.close()


@pytest.mark.gpu
def test_a_sequence_named_twice_and_forked_pages():
    rng = np.random.default_rng(8)
    pc = make(4, 2, 2, 4, 32, 700, 3)
    rows = random_rows(rng, pc, 600)
    pc.put_rows([0], [600], torch.from_numpy(rows).to(pc.device))
    pc.fork([0], [2], [555])
    check(pc, [0, 2, 0], [rows, rows[:555], rows], [3, 40, 600], queries(rng, pc, 643), window=123, sinks=9)
    pc.close()


@pytest.mark.gpu
def test_refusals():
    pc = make(4, 2, 2, 4, 16, 64, 2)
    rng = np.random.default_rng(1)
    pc.put_rows([0], [10], torch.from_numpy(random_rows(rng, pc, 10)).to(pc.device))
    q = torch.zeros((3, 8, 64), dtype=torch.int32, device=pc.device)
    assert torch.isfinite(pc.chunk_scan([0], q, 3)).all()
    for seqs, qq, counts, kw in (([1], q, 3, {}), ([2], q, 3, {}), ([-1], q, 3, {}), ([0, 1], q, [3, 0, 0], {}),
                                 ([0], q[:2], 3, {}), ([0], q[:, :4], 3, {}), ([0], q, 4, {}), ([0], q, [-3], {}),
                                 ([0], q, 3, {"window": 0}), ([0], q, 3, {"window": -4}),
                                 ([0], q, 3, {"window": 4, "sinks": -1}), ([0], q, 3, {"window": 1 << 40}),
                                 ([0], torch.zeros((11, 8, 64), dtype=torch.int32, device="cuda"), 11, {})):
        with pytest.raises(ValueError):
            pc.chunk_scan(seqs, qq, counts, **kw)
    with pytest.raises(TypeError):
        pc.chunk_scan([0], q.float(), 3)
    assert pc.chunk_scan([], q[:0], []).shape == (0, 8, 64)
    assert pc.chunk_scan([0, 1], q[:0], 0).shape == (0, 8, 64)
    pc.close()
    with pytest.raises((ValueError, RuntimeError)):
        pc.chunk_scan([0], q, 3)


def test_the_c_entry_checks_its_arguments():
    from insitu_b200 import _lib
    L = _lib.lib()
    assert L.ins_chunk_workspace(None, 1, None, None, 0, 0) == -1
    assert L.ins_chunk_scan(None, 1, None, None, 0, 0, None, None, None, 0, None) == _lib.INS_EINVAL
