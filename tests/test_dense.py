"""Cached rows read back as keys and values, against float64.

A vector as it is held is one product of two exact numbers, norm and centroid:
two fp32 roundings at most and that of the type, half a unit each. Turned back,
a sum of 64 centroids is taken in six stages of fp32 additions (2^-24 of the
partial sums each, which the sum of the magnitudes bounds), and scaled."""

from __future__ import annotations

import numpy as np
import pytest

from test_tree import decode, make, random_rows

torch = pytest.importorskip("torch")

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def want_of(pc, rows, rotated):
    """((k, v), (sum of magnitudes behind each)) in float64."""
    out, size = [], []
    scale = 512.0 / 2 ** pc.quant.norm_frac
    for x in decode(pc, rows):
        x = x * scale
        s = np.abs(x)
        if not rotated:
            from insitu_b200 import Rotation
            r = Rotation.for_quant(pc.quant, 64).matrix()
            s = np.repeat(np.abs(x).sum(-1, keepdims=True), 64, -1) / 8 * max(1, 8 ** (pc.quant.rot_rounds - 1))
            x = x @ r                                  # rows hold R x; R^T = R^-1
            if pc.quant.rot_rounds == 0:
                s = np.abs(x)
        out.append(x)
        size.append(s)
    return out, size


def check(pc, rows, got, dtype, rotated):
    want, size = want_of(pc, rows, rotated)
    half = torch.finfo(dtype).eps / 2
    # below the type's normal range half its smallest step
    floor = torch.finfo(dtype).smallest_normal * half
    for g, w, s in zip(got, want, size):
        assert g.dtype == dtype and tuple(g.shape) == w.shape
        # fp32: six additions a round, the product, the scale
        err = s * 2.0 ** -24 * (6 * max(1, pc.quant.rot_rounds) + 2)
        off = np.abs(g.double().cpu().numpy() - w)
        assert (off <= err + half * (np.abs(w) + err) + floor).all(), (off - err - half * np.abs(w)).max()


@pytest.mark.gpu
@pytest.mark.parametrize("kb,vb", [(4, 2), (3, 3), (1, 1), (2, 4), (5, 3), (8, 8), (7, 1)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rotated", [True, False])
def test_every_width_and_type(kb, vb, dtype, rotated):
    rng = np.random.default_rng(kb * 10 + vb)
    for n_kv, page, n in ((1, 16, 37), (3, 48, 101), (8, 256, 300)):
        pc = make(kb, vb, n_kv, 4, page, 512, 2)
        rows = random_rows(rng, pc, n, wild=dtype != torch.float16)
        pc.put_rows([1], [n], torch.from_numpy(rows).to(pc.device))
        check(pc, rows, pc.dense([1], dtype=dtype, rotated=rotated), dtype, rotated)
        check(pc, rows[5:n - 3], pc.dense([1], 5, n - 8, dtype=dtype, rotated=rotated), dtype, rotated)
        pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("rounds", [0, 1, 2, 3])
def test_rounds_of_the_rotation(rounds):
    from insitu_b200 import Geometry, PagedCache, QuantConfig
    rng = np.random.default_rng(rounds)
    pc = PagedCache(QuantConfig(key_bits=4, value_bits=2, rot_rounds=rounds, seed=7), geo=Geometry(2, 2, 64),
                    capacity=64, page_tokens=16)
    rows = random_rows(rng, pc, 50)
    pc.put_rows([0], [50], torch.from_numpy(rows).to(pc.device))
    check(pc, rows, pc.dense([0], dtype=torch.float32), torch.float32, False)
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("norm_frac", [1, 5, 12, 15])
def test_norm_formats(norm_frac):
    from insitu_b200 import Geometry, PagedCache, QuantConfig
    rng = np.random.default_rng(norm_frac)
    pc = PagedCache(QuantConfig(key_bits=4, value_bits=2, norm_frac=norm_frac), geo=Geometry(2, 2, 64), capacity=64,
                    page_tokens=16)
    rows = random_rows(rng, pc, 50, wild=True)
    pc.put_rows([0], [50], torch.from_numpy(rows).to(pc.device))
    for rotated in (True, False):
        check(pc, rows, pc.dense([0], dtype=torch.bfloat16, rotated=rotated), torch.bfloat16, rotated)
    pc.close()


@pytest.mark.gpu
def test_batches_spans_and_order():
    """Ragged spans of several sequences, one twice, one empty, one over a
    long range of pages."""
    rng = np.random.default_rng(4)
    lens = [700, 1, 33, 20_000]
    pc = make(4, 2, 2, 4, 32, 20_000, 4)
    rows = [random_rows(rng, pc, n) for n in lens]
    for i, n in enumerate(lens):
        pc.put_rows([i], [n], torch.from_numpy(rows[i]).to(pc.device))
    spans = [(3, 11, 19_000), (0, 31, 2), (1, 0, 1), (2, 33, 0), (0, 0, 700), (2, 1, 31)]
    got = pc.dense([s for s, _, _ in spans], [a for _, a, _ in spans], [n for _, _, n in spans], dtype=torch.float32)
    check(pc, np.concatenate([rows[s][a:a + n] for s, a, n in spans]), got, torch.float32, False)
    many = [(i % 4, 0, 1) for i in range(300)]
    got = pc.dense([s for s, _, _ in many], 0, 1, dtype=torch.float32, rotated=True)
    check(pc, np.concatenate([rows[s][:1] for s, _, _ in many]), got, torch.float32, True)
    pc.close()


@pytest.mark.gpu
def test_pages_and_outputs_beyond_four_gigabytes():
    rng = np.random.default_rng(2)
    filler = 12 * 10 ** 6 // 256 * 256
    pc = make(4, 2, 8, 4, 256, filler, 2, n_pages=filler // 256 + 8)
    pc.put_rows([0], [filler], torch.zeros((filler, 8, 52), dtype=torch.uint8, device=pc.device))
    rows = random_rows(rng, pc, 900)
    pc.put_rows([1], [900], torch.from_numpy(rows).to(pc.device))
    k, v = pc.dense([0, 1], [0, 0], [5 * 10 ** 6, 900])           # 5.1 GB each before the second sequence
    check(pc, rows, (k[-900:], v[-900:]), torch.bfloat16, False)
    pc.close()


@pytest.mark.gpu
def test_keys_and_values_that_went_in_come_back():
    """What an ingress wrote is read back within the codebook's own error. With
    y = R x, norm its root mean square and u = y / norm, a channel's code is its
    nearest centroid (boundaries lie halfway), off by d = min |u - c|. The norm
    is held to 2^-10 (half of 2^-9), the wire and the rotation's floors add
    2^-15 to y, a code chosen across a boundary by these is no further than d
    plus as much again. So ||got - x|| <= norm ||d + 2^-9 (2 + |u|)||, which a
    channel beyond the last centroid (a few in 25,600 Gaussian ones) can make
    some per cent of x."""
    from insitu_b200 import Geometry, PagedCache, QuantConfig, Rotation
    rng = np.random.default_rng(3)
    pc = PagedCache(QuantConfig(key_bits=8, value_bits=8), geo=Geometry(4, 2, 64), capacity=128, page_tokens=16)
    k, v = (rng.standard_normal((100, 4, 64)) for _ in range(2))
    wire = lambda x: torch.from_numpy(np.rint(x * 65536).astype(np.int32)).cuda()
    pc.ingress([0] * 100, wire(k), wire(v))
    r = Rotation.for_quant(pc.quant, 64).matrix()
    for got, x, cent in zip(pc.dense([0], dtype=torch.float32), (k, v), (pc.tables.k_centroids, pc.tables.v_centroids)):
        y = x @ r.T
        norm = np.sqrt((y ** 2).mean(-1))
        u = y / norm[..., None]
        d = np.abs(u[..., None] - np.asarray(cent) / 32768.0).min(-1)
        limit = norm * np.linalg.norm(d + 2.0 ** -9 * (2 + np.abs(u)), axis=-1)
        assert (np.linalg.norm(got.cpu().numpy() - x, axis=-1) <= limit).all()
    pc.close()


@pytest.mark.gpu
def test_another_stream_and_a_graph():
    rng = np.random.default_rng(5)
    pc = make(4, 2, 4, 4, 64, 4000, 1)
    rows = random_rows(rng, pc, 3000)
    pc.put_rows([0], [3000], torch.from_numpy(rows).to(pc.device))
    first = pc.dense([0])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        other = pc.dense([0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = pc.dense([0])
    for x in held:
        x.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for a, b, c in zip(first, other, held):
        assert torch.equal(a, b) and torch.equal(a, c)
    pc.close()


@pytest.mark.gpu
def test_refusals():
    pc = make(4, 2, 2, 4, 16, 64, 2)
    rng = np.random.default_rng(1)
    pc.put_rows([0], [10], torch.from_numpy(random_rows(rng, pc, 10)).to(pc.device))
    for args in (([2],), ([-1],), ([0], 11), ([0], -1), ([0], 0, 11), ([0], 5, 6), ([0], 0, -1), ([1], 0, 1)):
        with pytest.raises(ValueError):
            pc.dense(*args)
    with pytest.raises(ValueError):
        pc.dense([0], dtype=torch.float64)
    for x in pc.dense([], 0, 0) + pc.dense([0, 1], 0, 0) + pc.dense([1]):
        assert x.shape == (0, 2, 64)
    pc.close()


def test_the_c_entry_checks_its_arguments():
    from insitu_b200 import _lib
    assert _lib.lib().ins_cache_dense(None, 1, None, None, None, None, None, 0, 0, None) == _lib.INS_EINVAL
