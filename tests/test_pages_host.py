"""The page operations' bookkeeping on the host, run without a GPU: pages.cu
built against a runtime whose allocations can be made to fail and whose copies
and launches do nothing (tests/native)."""

from __future__ import annotations

import ctypes as C
import os
import subprocess

import numpy as np
import pytest

from insitu_b200 import _lib

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "native")
P, SEQS, PAGES_PER_SEQ = 16, 6, 1024


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    d = tmp_path_factory.mktemp("pages_host")
    so, fake = str(d / "pages_host.so"), str(d / "fake_cuda.o")
    cuda = os.path.join(os.path.dirname(os.path.dirname(_lib.nvcc())), "include")
    subprocess.run(["g++", "-O1", "-fPIC", f"-I{cuda}", "-c", "-o", fake, os.path.join(HERE, "fake_cuda.cpp")], check=True)
    subprocess.run([_lib.nvcc(), "-gencode", "arch=compute_100a,code=sm_100a", "-O1", "-std=c++17", "-Xcompiler", "-fPIC",
                    "-shared", "-cudart", "none", "-Xlinker", "-Bsymbolic", "-o", so,
                    os.path.join(HERE, "pages_host.cu"), fake], check=True)
    L = C.CDLL(so)
    L.host_create.restype = C.c_void_p
    L.host_error.restype = C.c_char_p
    for name in ("host_table", "host_lengths", "host_refs"):
        getattr(L, name).restype = C.POINTER(C.c_int32)
    return L


class Cache:
    """The handle, its calls (status returned) and what the host knows."""

    def __init__(self, L, n_pages):
        self.L, self.n_pages = L, n_pages
        self.h = C.c_void_p(L.host_create(2, P, SEQS, PAGES_PER_SEQ, n_pages))

    def close(self):
        self.L.host_destroy(self.h)

    def _call(self, name, ids, *arrays, rows=False):
        i32 = lambda v: np.ascontiguousarray(v, np.int32).ctypes.data_as(C.c_void_p)
        arrays = [None if a is None else np.ascontiguousarray(a, np.int32 if name == "fork" and i == 0 else np.int64)
                  for i, a in enumerate(arrays)]
        args = [None if a is None else a.ctypes.data_as(C.c_void_p) for a in arrays]
        ids = np.ascontiguousarray(ids, np.int32)
        tail = [C.c_void_p(64)] if rows else []
        return getattr(self.L, f"ins_cache_{name}")(self.h, len(ids), i32(ids), *args, *tail, None)

    def put(self, ids, n):
        return self._call("put_rows", ids, n, rows=True)

    def fork(self, src, dst, lengths=None):
        return self._call("fork", src, dst, lengths)

    def compact(self, ids, base, keep):
        flat = np.concatenate([np.asarray(k, np.int64) for k in keep] or [np.zeros(0, np.int64)])
        return self._call("compact", ids, base, [len(k) for k in keep], flat)

    def truncate(self, ids, n):
        return self._call("truncate", ids, n)

    def state(self):
        free = np.zeros(self.n_pages, np.int32)
        n = self.L.host_free(self.h, free.ctypes.data_as(C.c_void_p))
        view = lambda f, k: np.ctypeslib.as_array(f(self.h), (k,)).copy()
        return (view(self.L.host_table, SEQS * PAGES_PER_SEQ).reshape(SEQS, -1), view(self.L.host_lengths, SEQS),
                view(self.L.host_refs, self.n_pages), sorted(free[:n].tolist()))

    def check(self):
        """Every page is free or held as often as it is counted; every sequence
        has the pages of its length; the page that the next row goes to is its own."""
        table, lengths, refs, free = self.state()
        held = np.zeros(self.n_pages, int)
        for s in range(SEQS):
            n = -(-int(lengths[s]) // P)
            assert (table[s, :n] >= 0).all() and (table[s, n:] == -1).all()
            assert len(set(table[s, :n])) == n
            np.add.at(held, table[s, :n], 1)
            if lengths[s] % P:
                assert refs[table[s, n - 1]] == 1
        assert (held == refs).all() and free == np.flatnonzero(held == 0).tolist()
        return lengths


def same(a, b):
    return all(np.array_equal(x, y) for x, y in zip(a, b))


@pytest.fixture
def cache(host):
    made = []
    yield lambda n_pages: made.append(Cache(host, n_pages)) or made[-1]
    host.host_allow(-1)
    for c in made:
        c.close()


CALLS = {
    "compact in place": lambda c: c.compact([0], [0], [range(1, 16000, 3)]),
    "compact into new pages": lambda c: c.compact([1], [8000], [range(0, 8000, 2)]),
    "compact several": lambda c: c.compact([0, 1], [10, 0], [range(3, 9000), range(1, 4000)]),
    "fork": lambda c: c.fork([0, 1, 1], [2, 3, 4], [16000, 15999, 7]),
    "put rows": lambda c: c.put([2, 3], [16000, 5]),
}


@pytest.mark.parametrize("call", CALLS)
@pytest.mark.parametrize("allowed", range(8))
def test_a_call_whose_upload_buffers_cannot_be_had_changes_nothing(host, cache, call, allowed):
    """Its plan does not fit the kernel's parameter; one of the four buffer
    pairs' allocations fails."""
    c = cache(2001 if "in place" in call else 4200)
    for s in (0, 1):
        for _ in range(50):                      # in steps whose plans are small
            assert c.put([s], [320]) == 0
    before = c.state()
    host.host_allow(allowed)
    assert CALLS[call](c) == _lib.INS_ENOMEM
    host.host_allow(-1)
    assert same(c.state(), before)
    c.check()
    assert CALLS[call](c) == 0
    c.check()


def test_random_operations_keep_the_books(cache):
    rng = np.random.default_rng(4)
    c = cache(90)
    refused = 0
    for _ in range(3000):
        lengths = c.check()
        op, before = rng.integers(0, 4), c.state()
        ids = rng.permutation(SEQS)[:rng.integers(1, 4)].tolist()
        if op == 0:
            rc = c.put(ids, [int(rng.choice([0, 1, P - 1, P, 37, 300])) for _ in ids])
        elif op == 1:
            src = rng.integers(0, SEQS, len(ids)).tolist()
            rc = c.fork(src, ids, [int(rng.integers(0, lengths[s] + 1)) for s in src] if rng.random() < 0.6 else None)
            if set(src) & set(ids):
                assert rc == _lib.INS_EINVAL
        elif op == 2:
            base = [int(rng.integers(0, lengths[s] + 1)) for s in ids]
            keep = [np.sort(rng.permutation(int(lengths[s]) - b)[:rng.integers(0, lengths[s] - b + 1)])
                    for s, b in zip(ids, base)]
            rc = c.compact(ids, base, keep)
            if rc == 0:
                assert c.check()[ids].tolist() == [b + len(k) for b, k in zip(base, keep)]
        else:
            n = [int(rng.choice([0, lengths[s] // P * P, rng.integers(0, lengths[s] + 1)])) for s in ids]
            rc = c.truncate(ids, n)
        if rc:
            refused += 1
            assert same(c.state(), before)
    assert 100 < refused < 2500
    assert c.truncate(range(SEQS), [0] * SEQS) == 0
    assert len(c.state()[3]) == 90
