"""Waits of the chunk attention that run out, and formats at its products' edges."""

from __future__ import annotations

import numpy as np
import pytest

from test_chunk import check, queries, visible
from test_tree import make, random_rows

torch = pytest.importorskip("torch")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 24, 64, 700])
@pytest.mark.parametrize("tile", [0, 1, 9])
def test_a_wait_for_rows_that_runs_out_is_reported_and_the_context_survives(n, tile):
    """One tile's copies are announced 16 bytes larger than they are, so the
    wait for them cannot complete: it gives up after the lowered limit, the
    launch ends, the status is INS_ETIMEOUT, and the next scan is what it was.
    Every copy lands; nothing faults."""
    from insitu_b200._lib import DeviceTimeout
    rng = np.random.default_rng(n)
    pc = make(4, 2, 8, 4, 256, 60160, 1)
    pc.put_rows([0], [60001], torch.from_numpy(random_rows(rng, pc, 60001)).to(pc.device))
    q = queries(rng, pc, n)
    want = pc.chunk_scan([0], q, n)
    pc.status()
    for cta in (0, 77):
        pc.set_wait_test(poll_limit=4096, item=cta, chunk=tile)
        pc.chunk_scan([0], q, n)
        with pytest.raises(DeviceTimeout):
            pc.status()
        pc.set_wait_test()
        assert torch.equal(pc.chunk_scan([0], q, n).view(torch.int16), want.view(torch.int16))
        pc.status()
    pc.close()


def reference_rows(pc, q, rows, window, sinks):
    """Float64 over the operands unrounded: (n, heads, 64)."""
    from insitu_b200 import KVQuantizer
    kv = KVQuantizer(64, pc.quant, pc.fmt).unpack(rows)
    real = lambda cent, idx, norm: torch.as_tensor(  # noqa: E731
        cent[idx] / 2.0 ** pc.fmt.centroid_frac * (norm.astype(np.float64) / 2.0 ** pc.quant.norm_frac)[..., None]).cuda()
    k, v = real(pc.tables.k_centroids, kv.k_idx, kv.k_norm), real(pc.tables.v_centroids, kv.v_idx, kv.v_norm)
    g, n = pc.geo, len(q)
    x = q.double().reshape(n, g.n_kv_heads, g.kv_groups, 64) / 2.0 ** pc.fmt.qk_frac
    see = torch.as_tensor(visible(len(rows) - n, n, window, sinks)).cuda()
    s = torch.einsum("nhgd,thd->nhgt", x, k).masked_fill(~see[:, None, None], -torch.inf)
    a = torch.softmax(s, -1)
    reach = torch.einsum("nhgt,thd->nhgd", a, v.abs())
    size = torch.einsum("nhgd,thd->nhgt", x.abs(), k.abs()).masked_fill(~see[:, None, None], 0).amax(-1, keepdim=True)
    out = torch.einsum("nhgt,thd->nhgd", a, v)
    # the bound of test_tree.py: four roundings to 11 bits in scores, three in terms, the output's
    bound = 2.0 ** -9 * out.abs() + 2.0 ** -11 * (4 * size + 3) * reach + 1e-7 * float(v.abs().max())
    return out.reshape(q.shape), bound.reshape(q.shape)


@pytest.mark.gpu
@pytest.mark.parametrize("norm_frac,qk_frac", [(9, 16), (1, 16), (3, 12), (9, 8), (15, 20), (12, 16), (9, 24)])
@pytest.mark.parametrize("n", [1, 30, 400])
def test_formats(norm_frac, qk_frac, n):
    """Powers of two between the products' fixed units and the formats, where
    they stand in queries, keys, scores and outputs."""
    from insitu_b200 import FixedFormat, Geometry, PagedCache, QuantConfig
    rng = np.random.default_rng(norm_frac * 100 + qk_frac + n)
    pc = PagedCache(QuantConfig(key_bits=4, value_bits=2, norm_frac=norm_frac), FixedFormat(qk_frac=qk_frac),
                    Geometry(2, 4, 64), capacity=1024, page_tokens=64)
    norms = np.clip(np.rint(2.0 ** norm_frac * (1 + 0.1 * rng.standard_normal((900, 2, 2)))), 1, 32767)
    rows = rng.integers(0, 256, (900, 2, pc.row_bytes), dtype=np.uint8)
    rows[..., -4:] = np.ascontiguousarray(norms.astype("<i2")).view(np.uint8).reshape(900, 2, 4)
    pc.put_rows([0], [900], torch.from_numpy(rows).to(pc.device))
    q = torch.from_numpy(np.rint(rng.standard_normal((n, 8, 64)) * 2.0 ** qk_frac / 4).astype(np.int32)).to(pc.device)
    got = pc.chunk_scan([0], q, n, window=300, sinks=3)
    pc.status()
    want, bound = reference_rows(pc, q, rows, 300, 3)
    worst = float(((got.double() - want).abs() - bound).max())
    assert worst <= 0, worst
    pc.close()


@pytest.mark.gpu
def test_formats_that_the_products_do_not_cover_are_refused():
    from insitu_b200 import FixedFormat, Geometry, PagedCache, QuantConfig
    pc = PagedCache(QuantConfig(key_bits=4, value_bits=2), FixedFormat(qk_frac=-1), Geometry(2, 4, 64), capacity=64)
    pc.put_rows([0], [4], torch.zeros((4, 2, 52), dtype=torch.uint8, device=pc.device))
    with pytest.raises(ValueError):
        pc.chunk_scan([0], torch.zeros((4, 8, 64), dtype=torch.int32, device=pc.device), 4)
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [2, 40, 600])
def test_a_masked_row_of_the_largest_values_changes_nothing(n):
    """Rows outside the window hold the largest norms there are: their scores
    are hidden before any maximum or sum."""
    rng = np.random.default_rng(n)
    pc = make(4, 2, 2, 4, 64, 3000, 1)
    rows = random_rows(rng, pc, 2500)
    rows[:2500 - n - 40, :, -4:] = np.frombuffer(np.array([32767, 32767], "<i2").tobytes(), np.uint8)
    pc.put_rows([0], [2500], torch.from_numpy(rows).to(pc.device))
    check(pc, [0], [rows], [n], queries(rng, pc, n), window=40, sinks=0)
    pc.close()
