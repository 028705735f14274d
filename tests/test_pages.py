"""Page operations of the cache (fork, compact, truncate, rows, put_rows):
every sequence's packed rows against a plain list of rows that the same
operations are applied to, and the pool's free pages against a count of the
pages that are held."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def make(kb=4, vb=2, n_kv=2, page=16, capacity=160, max_seqs=6, n_pages=None):
    from insitu_b200 import Geometry, PagedCache, QuantConfig
    return PagedCache(QuantConfig(key_bits=kb, value_bits=vb), geo=Geometry(n_kv, 1, 64), max_seqs=max_seqs,
                      capacity=capacity, page_tokens=page, n_pages=n_pages)


def random_rows(rng, pc, n):
    return rng.integers(0, 256, (n, pc.geo.n_kv_heads, pc.row_bytes), dtype=np.uint8)


def append(pc, seq, rows):
    pc.put_rows([seq], [len(rows)], torch.from_numpy(rows).to(pc.device))


def check(pc, held):
    """held: {sequence: its rows}."""
    for seq, rows in held.items():
        assert pc.length(seq) == len(rows)
    ids = list(held)
    got = pc.rows(ids).cpu().numpy()
    np.testing.assert_array_equal(got, np.concatenate([held[s] for s in ids]))


@pytest.mark.gpu
@pytest.mark.parametrize("kb,vb,n_kv,page", [(4, 2, 8, 256), (3, 3, 1, 16), (1, 1, 3, 48), (8, 8, 9, 32), (5, 7, 2, 16)])
def test_rows_are_the_exported_bytes_and_put_rows_brings_them_back(kb, vb, n_kv, page):
    pc = make(kb, vb, n_kv, page, capacity=4 * page, max_seqs=3)
    rng = np.random.default_rng(kb * 10 + vb)
    n = 3 * page + 5
    rows = random_rows(rng, pc, n)
    pc.import_rows(0, rows)
    np.testing.assert_array_equal(pc.rows([0]).cpu().numpy(), rows)
    np.testing.assert_array_equal(pc.rows([0], page - 1, 2).cpu().numpy(), rows[page - 1:page + 1])
    assert pc.rows([0], 7, 0).shape[0] == 0
    both = pc.rows([0, 0], [3, page], [1, page + 9])
    np.testing.assert_array_equal(both.cpu().numpy(), np.concatenate([rows[3:4], rows[page:2 * page + 9]]))
    append(pc, 1, rows[:3])                       # a partial page, then more rows after it
    append(pc, 1, rows[3:])
    for h in range(n_kv):
        np.testing.assert_array_equal(pc.export(1, h), rows[:, h])
    pc.close()


@pytest.mark.gpu
def test_random_operations_match_a_list_of_rows():
    """Forks of forks, compactions that start inside shared pages, truncations
    to zero, one and page boundaries, appends after each of them."""
    rng = np.random.default_rng(11)
    page = 16
    pc = make(4, 2, 2, page, capacity=10 * page, max_seqs=6, n_pages=200)
    held = {s: np.zeros((0, 2, pc.row_bytes), np.uint8) for s in range(6)}
    for step in range(150):
        op = rng.integers(0, 5)
        if op == 0:
            s = int(rng.integers(0, 6))
            n = int(rng.choice([1, 2, page, page + 1, 37]))
            rows = random_rows(rng, pc, n)
            if len(held[s]) + n > pc.capacity:
                with pytest.raises(ValueError):
                    append(pc, s, rows)
            else:
                append(pc, s, rows)
                held[s] = np.concatenate([held[s], rows])
        elif op == 1:
            empty = [s for s in held if len(held[s]) == 0]
            if not empty:
                continue
            dst = [int(x) for x in rng.permutation(empty)[:2]]
            src = [int(rng.integers(0, 6)) for _ in dst]
            if any(s in dst for s in src):
                continue
            n = [int(rng.integers(0, len(held[s]) + 1)) for s in src]
            pc.fork(src, dst, n)
            for s, d, k in zip(src, dst, n):
                held[d] = held[s][:k].copy()
        elif op in (2, 3):
            ids = [int(x) for x in rng.permutation(6)[:rng.integers(1, 5)]]
            bases, keeps = [], []
            for s in ids:
                base = int(rng.integers(0, len(held[s]) + 1))
                among = len(held[s]) - base
                m = int(rng.integers(0, among + 1))
                if rng.random() < 0.2:
                    keep = np.arange(m)               # nothing moves
                else:
                    keep = np.sort(rng.permutation(among)[:m])
                bases.append(base)
                keeps.append(keep)
            pc.compact(ids, keeps, bases)
            for s, base, keep in zip(ids, bases, keeps):
                held[s] = np.concatenate([held[s][:base], held[s][base:][keep]])
        else:
            ids = [int(x) for x in rng.permutation(6)[:2]]
            n = [int(rng.choice([0, len(held[s]), len(held[s]) // page * page, rng.integers(0, len(held[s]) + 1)]))
                 for s in ids]
            pc.truncate(ids, n)
            for s, k in zip(ids, n):
                held[s] = held[s][:k]
        check(pc, held)
    pc.status()
    pc.truncate(list(held), 0)
    assert pc.free_pages == 200
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("forked", [False, True])
@pytest.mark.parametrize("spare", [0, 400])
def test_long_compaction(forked, spare):
    """Thousands of kept rows, in the sequence's own pages (no page to spare:
    in order) and into new ones (in parallel)."""
    rng = np.random.default_rng(5)
    n, page = 5003, 16
    pages = -(-n // page)
    pc = make(4, 2, 2, page, capacity=pages * page, max_seqs=2, n_pages=pages + spare + (pages if forked else 0))
    rows = random_rows(rng, pc, n)
    pc.put_rows([0], [n], torch.from_numpy(rows).to(pc.device))
    seq = 0
    if forked:
        pc.fork([0], [1])
        seq = 1
    keep = np.sort(rng.permutation(n)[:2601])
    pc.compact([seq], [keep])
    np.testing.assert_array_equal(pc.rows([seq]).cpu().numpy(), rows[keep])
    if forked:
        np.testing.assert_array_equal(pc.rows([0]).cpu().numpy(), rows)
    pc.truncate([0, 1], 0)
    assert pc.free_pages == pages + spare + (pages if forked else 0)
    pc.close()


@pytest.mark.gpu
def test_fork_shares_pages_and_appends_stay_apart():
    """A fork of a sequence takes one page (its last, partial one); rows that
    either side appends, by ingress too, do not reach the other."""
    from insitu_b200 import DecodeAttention, Geometry, QuantConfig
    rng = np.random.default_rng(3)
    wire = lambda *s: torch.from_numpy(rng.integers(-(1 << 17), 1 << 17, s).astype(np.int32))
    dec = DecodeAttention(QuantConfig(key_bits=4, value_bits=2), geo=Geometry(2, 4, 64), max_seqs=3, capacity=64,
                          page_tokens=16)
    k, v = wire(40, 2, 64), wire(40, 2, 64)
    dec.prefill(0, k, v)
    free = dec.pc.free_pages
    dec.pc.fork([0, 0], [1, 2], [40, 32])
    assert free - dec.pc.free_pages == 1
    q = wire(1, 8, 64)
    outs = []
    for s in (1, 0, 2):
        k1, v1 = wire(1, 2, 64), wire(1, 2, 64)
        out, _ = dec.step(q, k1, v1, [s])
        ref = DecodeAttention(QuantConfig(key_bits=4, value_bits=2), geo=Geometry(2, 4, 64), max_seqs=1, capacity=64,
                              page_tokens=16)
        n = 32 if s == 2 else 40
        ref.prefill(0, k[:n], v[:n])
        want, _ = ref.step(q, k1, v1, [0])
        np.testing.assert_array_equal(out.cpu().numpy(), want.cpu().numpy())
        outs.append(out)
        ref.close()
    dec.pc.reset()
    assert dec.pc.free_pages == 3 * 4
    dec.close()


@pytest.mark.gpu
def test_refusals_change_nothing():
    pc = make(4, 2, 2, 16, capacity=64, max_seqs=3, n_pages=4)
    rng = np.random.default_rng(1)
    rows = random_rows(rng, pc, 40)
    append(pc, 0, rows)
    free = pc.free_pages
    append(pc, 2, rows[:3])                        # the pool's last page
    for call in (lambda: pc.fork([0], [2]),                      # not empty
                 lambda: pc.fork([0], [1], [41]),                # longer than the source
                 lambda: pc.fork([0], [1]),                      # no page left for the partial one
                 lambda: pc.fork([0, 0], [1, 1]),                # the same target twice
                 lambda: pc.fork([0], [3]), lambda: pc.fork([-1], [1]), lambda: pc.fork([0], [1, 2]),
                 lambda: pc.compact([0], [[3, 2]]), lambda: pc.compact([0], [[2, 2]]),
                 lambda: pc.compact([0], [[-1]]), lambda: pc.compact([0], [[40]]),
                 lambda: pc.compact([0], [[0]], 41), lambda: pc.compact([0], [[5]], 35),
                 lambda: pc.compact([0, 0], [[0], [1]]), lambda: pc.compact([0], []),
                 lambda: pc.truncate([0], 41), lambda: pc.truncate([0], -1), lambda: pc.truncate([7], 0),
                 lambda: pc.rows([0], 39, 2), lambda: pc.rows([0], -1, 1), lambda: pc.rows([3], 0, 1),
                 lambda: pc.put_rows([1], [1], torch.zeros((2, 2, pc.row_bytes), dtype=torch.uint8, device="cuda")),
                 lambda: pc.put_rows([1], [1], torch.zeros((1, 2, 3), dtype=torch.uint8, device="cuda")),
                 lambda: pc.put_rows([1], [1], torch.zeros((1, 2, pc.row_bytes), dtype=torch.uint8)),
                 lambda: append(pc, 1, rows[:1]), lambda: append(pc, 0, rows[:30])):
        with pytest.raises(ValueError):
            call()
    check(pc, {0: rows, 2: rows[:3]})
    assert pc.length(1) == 0 and pc.free_pages == free - 1
    pc.fork([0], [1], [32])                        # whole pages only: no page needed
    with pytest.raises(ValueError):                # a shared page to be written, and none to replace it
        pc.compact([1], [[1]])
    check(pc, {0: rows, 1: rows[:32], 2: rows[:3]})
    pc.close()


def test_null_handles_and_missing_arrays_are_errors():
    from insitu_b200 import _lib
    L = _lib.lib()
    assert L.ins_cache_free_pages(None) == -1
    assert L.ins_cache_fork(None, 0, None, None, None, None) == _lib.INS_EINVAL
    assert L.ins_cache_compact(None, 1, None, None, None, None, None) == _lib.INS_EINVAL
    assert L.ins_cache_truncate(None, 1, None, None, None) == _lib.INS_EINVAL
    assert L.ins_cache_rows(None, 1, None, None, None, None, None) == _lib.INS_EINVAL
    assert L.ins_cache_put_rows(None, 1, None, None, None, None) == _lib.INS_EINVAL
