"""Tree attention over the compressed cache against its definition in float64.

The bound for one output, derived before the first run: with u = 2^-11 (half
a unit of fp16's 11 bits), the query and the key each carry a relative error
of u, so a score is off by at most 2u sum|q k|, a weight by twice that
relatively (numerator and denominator); the weight and the value carry u each
more; then one rounding to bf16 (2^-9). So

    |out - ref| <= 2^-9 |ref| + (4u max_r sum|q k_r| + 3u) sum_r a_r |v_r| + tiny

and, since the errors are independent roundings, the whole tensor is within
2^-8 of the reference in the 2-norm wherever scores are moderate."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

U = 2.0 ** -11


def make(kb, vb, n_kv, groups, page, capacity, max_seqs, n_pages=None):
    from insitu_b200 import Geometry, PagedCache, QuantConfig
    return PagedCache(QuantConfig(key_bits=kb, value_bits=vb), geo=Geometry(n_kv, groups, 64), max_seqs=max_seqs,
                      capacity=capacity, page_tokens=page, n_pages=n_pages)


def random_rows(rng, pc, n, wild=False):
    """Random codes; norms near 1 (512), or (wild) any 16-bit number."""
    rows = rng.integers(0, 256, (n, pc.geo.n_kv_heads, pc.row_bytes), dtype=np.uint8)
    if not wild:
        norms = np.clip(np.rint(512 + 60 * rng.standard_normal((n, pc.geo.n_kv_heads, 2))), 1, 32767).astype("<i2")
        rows[..., -4:] = norms.view(np.uint8).reshape(n, pc.geo.n_kv_heads, 4)
    return rows


def decode(pc, rows):
    """(k, v): (n, n_kv, 64) float64 in real units, by this package's row codec."""
    from insitu_b200 import KVQuantizer
    kv = KVQuantizer(64, pc.quant).unpack(rows)
    k = pc.tables.k_centroids[kv.k_idx] / 32768.0 * (kv.k_norm.astype(np.float64) / 512)[..., None]
    v = pc.tables.v_centroids[kv.v_idx] / 32768.0 * (kv.v_norm.astype(np.float64) / 512)[..., None]
    return k, v


def reference(q, k, v, see):
    """q (n, n_kv, g, 64), k and v (T, n_kv, 64), see (n, T) -> out, the bound, both (n, n_kv, g, 64)."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    q, k, v, see = (torch.as_tensor(x, device=dev) for x in (q, k, v, see))
    s = torch.einsum("nhgd,thd->nhgt", q, k)
    s = torch.where(see[:, None, None], s, -torch.inf)
    some = see.any(1)
    m = torch.where(some[:, None, None], s.amax(-1), 0.0)
    a = torch.exp(s - m[..., None])
    a = a / a.sum(-1, keepdim=True).clamp(min=1e-300)
    out = torch.einsum("nhgt,thd->nhgd", a, v)
    reach = torch.einsum("nhgt,thd->nhgd", a, v.abs())
    size = torch.einsum("nhgd,thd->nhgt", q.abs(), k.abs())
    size = torch.where(see[:, None, None], size, 0.0).amax(-1, keepdim=True)
    bound = 2.0 ** -9 * out.abs() + (4 * U * size + 3 * U) * reach + 1e-7
    return out.cpu().numpy(), bound.cpu().numpy()


def check(pc, seqs, tree, rows, contexts, q, near=True):
    """tree_scan of `seqs` against the reference; rows[i] are sequence i's packed rows."""
    g = pc.geo
    got = pc.tree_scan(seqs, q, tree)
    assert got.dtype == torch.bfloat16 and got.shape == q.shape
    pc.status()
    got = got.float().cpu().numpy()
    masks = tree.mask("cpu").numpy().view(np.uint64)
    tree.mask(pc.device)
    for i, ctx in enumerate(contexts):
        lo, n = tree.offsets[i], tree.counts[i]
        if n == 0:
            continue
        k, v = decode(pc, rows[i])
        bits = (masks[lo:lo + n, :, None] >> np.arange(64, dtype=np.uint64)) & np.uint64(1)
        see = np.concatenate([np.ones((n, ctx), bool), bits.reshape(n, -1)[:, :n].astype(bool)], 1)
        qi = q[lo:lo + n].cpu().numpy().astype(np.float64).reshape(n, g.n_kv_heads, g.kv_groups, 64) / 65536
        want, bound = reference(qi, k, v, see)
        have = got[lo:lo + n].reshape(want.shape)
        worst = (np.abs(have - want) - bound).max()
        assert worst <= 0, f"sequence {i}: {worst} over the bound"
        if near:
            assert np.linalg.norm(have - want) <= 2.0 ** -8 * np.linalg.norm(want) + 1e-7


def random_tree(rng, n, roots=0.1):
    return [-1 if i == 0 or rng.random() < roots else int(rng.integers(max(0, i - 9), i)) for i in range(n)]


def run(kb, vb, n_kv, groups, page, contexts, nodes, seed=0, scale=0.25, wild=False, tree=None):
    from insitu_b200.tree import DraftTree
    rng = np.random.default_rng(seed)
    lens = [c + n for c, n in zip(contexts, nodes)]
    pc = make(kb, vb, n_kv, groups, page, max(16, *lens), len(lens))
    rows = [random_rows(rng, pc, n, wild) for n in lens]
    for i in rng.permutation(len(lens)):
        pc.put_rows([int(i)], [lens[i]], torch.from_numpy(rows[i]).to(pc.device))
    tree = tree or DraftTree([random_tree(rng, n) for n in nodes])
    q = torch.from_numpy(np.rint(rng.standard_normal((sum(nodes), n_kv * groups, 64)) * scale * 65536).astype(np.int32))
    check(pc, list(range(len(lens))), tree, rows, contexts, q.to(pc.device), near=scale <= 0.25 and not wild)
    pc.close()


@pytest.mark.gpu
@pytest.mark.parametrize("kb,vb", [(4, 2), (3, 3), (1, 1), (2, 4), (5, 3), (8, 8)])
@pytest.mark.parametrize("nodes", [1, 3, 8, 21, 64])
def test_every_width(kb, vb, nodes):
    run(kb, vb, 2, 4, 64, [517], [nodes], seed=kb * 100 + nodes)


@pytest.mark.gpu
@pytest.mark.parametrize("groups", [1, 2, 4, 8])
@pytest.mark.parametrize("nodes", [1, 2, 5, 16, 17, 33])
def test_every_group(groups, nodes):
    run(4, 2, 3, groups, 256, [1000], [nodes], seed=groups * 100 + nodes)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 48, 256])
@pytest.mark.parametrize("context", [0, 1, 15, 16, 17, 47, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257, 4099])
def test_context_lengths_around_every_boundary(page, context):
    run(4, 2, 1, 4, page, [context], [1], seed=context)
    run(3, 3, 1, 4, page, [context], [7], seed=context)
    run(4, 2, 2, 4, page, [context], [50], seed=context)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [(1,) * 9, (5, 0, 64, 1, 17), (256, 130, 65), (8,) * 40])
def test_ragged_batches(nodes):
    rng = np.random.default_rng(len(nodes))
    contexts = [int(x) for x in np.exp(rng.uniform(0, np.log(6000), len(nodes)))]
    run(4, 2, 2, 4, 256, contexts, list(nodes), seed=len(nodes))
    run(3, 3, 2, 2, 32, contexts, list(nodes), seed=len(nodes) + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes,groups", [(1, 4), (1, 8), (9, 4), (40, 8)])
def test_long_contexts(nodes, groups):
    run(4, 2, 1, groups, 256, [150_001], [nodes], seed=nodes)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 12, 60])
@pytest.mark.parametrize("scale", [0.0, 4.0, 60.0])
def test_peaked_and_flat_scores(nodes, scale):
    """Queries up to the wire format's limits: one token takes all the weight,
    maxima rise late and often; and zero queries: the plain mean."""
    run(4, 2, 2, 4, 64, [3000], [nodes], seed=nodes, scale=scale)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 12, 60])
def test_any_norms(nodes):
    """Rows of random bytes: norms of either sign up to 64."""
    run(4, 2, 2, 4, 64, [700], [nodes], seed=nodes, scale=0.05, wild=True)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [3, 20, 70])
def test_any_mask_and_nodes_that_see_nothing(n):
    from insitu_b200.tree import DraftTree
    rng = np.random.default_rng(n)
    masks = [rng.random((n, n)) < 0.3, np.zeros((n, n), bool)]
    masks[0][0] = False
    masks[0][-1] = False
    masks[0][-1, -1] = True
    run(4, 2, 2, 4, 64, [0, 5], [n, n], seed=n, tree=DraftTree.from_mask(masks))


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 40])
def test_pages_beyond_four_gigabytes(nodes):
    """The sequence's pages lie after 5 GB of another one's."""
    from insitu_b200.tree import DraftTree
    rng = np.random.default_rng(2)
    filler = 12 * 10 ** 6 // 256 * 256
    pc = make(4, 2, 8, 4, 256, filler, 2, n_pages=filler // 256 + 8)
    pc.put_rows([0], [filler], torch.zeros((filler, 8, 52), dtype=torch.uint8, device=pc.device))
    rows = random_rows(rng, pc, 900)
    pc.put_rows([1], [900], torch.from_numpy(rows).to(pc.device))
    np.testing.assert_array_equal(pc.rows([1]).cpu().numpy(), rows)
    q = torch.from_numpy(np.rint(rng.standard_normal((nodes, 32, 64)) * 16384).astype(np.int32)).to(pc.device)
    check(pc, [1], DraftTree([random_tree(rng, nodes)]), [rows], [900 - nodes], q)
    pc.close()


@pytest.mark.gpu
def test_a_chain_agrees_with_the_fixed_point_scan():
    """Eight tokens as a chain in one call, and one at a time through the
    bit-exact scan: within the bound above plus the fixed-point form's own
    resolution (2^-15 probabilities, Q16 outputs)."""
    from insitu_b200 import DecodeAttention, Geometry, QuantConfig
    from insitu_b200.tree import DraftTree
    rng = np.random.default_rng(6)
    wire = lambda s, *shape: torch.from_numpy(np.rint(rng.standard_normal(shape) * s * 65536).astype(np.int32)).cuda()
    quant, geo = QuantConfig(key_bits=4, value_bits=2), Geometry(8, 4, 64)
    one, dec = (DecodeAttention(quant, geo=geo, max_seqs=1, capacity=1024) for _ in range(2))
    k, v, q = wire(1, 600, 8, 64), wire(1, 600, 8, 64), wire(0.25, 8, 32, 64)
    one.prefill(0, k[:592], v[:592])
    dec.prefill(0, k[:592], v[:592])
    want = torch.cat([one.step(q[i:i + 1], k[592 + i:593 + i], v[592 + i:593 + i], mode="two_pass")[0] for i in range(8)])
    q_rot = dec.pc.ingress([0] * 8, k[592:], v[592:], q)
    got = dec.pc.tree_scan([0], q_rot, DraftTree([list(range(-1, 7))]))
    want = want.double() / 65536
    assert float((got.double() - want).norm() / want.norm()) <= 2.0 ** -7
    one.close()
    dec.close()


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 20, 64])
def test_runs_repeat_on_another_stream(nodes):
    from insitu_b200.tree import DraftTree
    rng = np.random.default_rng(nodes)
    pc = make(4, 2, 8, 4, 256, 9000, 1)
    rows = random_rows(rng, pc, 8000)
    pc.put_rows([0], [8000], torch.from_numpy(rows).to(pc.device))
    tree = DraftTree([random_tree(rng, nodes)])
    q = torch.from_numpy(np.rint(rng.standard_normal((nodes, 32, 64)) * 16384).astype(np.int32)).to(pc.device)
    first = pc.tree_scan([0], q, tree)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = [pc.tree_scan([0], q, tree) for _ in range(5)]
    torch.cuda.synchronize()
    for x in again:
        assert torch.equal(first.view(torch.int16), x.view(torch.int16))
    pc.close()


@pytest.mark.gpu
def test_refusals():
    from insitu_b200.tree import DraftTree
    pc = make(4, 2, 2, 4, 16, 64, 2)
    rng = np.random.default_rng(1)
    pc.put_rows([0], [10], torch.from_numpy(random_rows(rng, pc, 10)).to(pc.device))
    q = torch.zeros((3, 8, 64), dtype=torch.int32, device=pc.device)
    tree = DraftTree([[-1, 0, 1]])
    assert torch.isfinite(pc.tree_scan([0], q, tree)).all()
    for seqs, queries, t in (([1], q, tree), ([2], q, tree), ([-1], q, tree), ([0, 1], q, tree), ([0], q[:2], tree),
                             ([0], q[:, :4], tree), ([0], torch.zeros((11, 8, 64), dtype=torch.int32, device="cuda"),
                                                     DraftTree([list(range(-1, 10))]))):
        with pytest.raises(ValueError):
            pc.tree_scan(seqs, queries, t)
    with pytest.raises(TypeError):
        pc.tree_scan([0], q.float(), tree)
    assert pc.tree_scan([], q[:0], DraftTree([])).shape == (0, 8, 64)
    assert pc.tree_scan([0], q[:0], DraftTree([[]])).shape == (0, 8, 64)
    pc.close()


def test_trees_are_checked_and_hold_their_ancestors():
    from insitu_b200.tree import DraftTree
    for bad in ([[0]], [[-1, 1]], [[-2]], [[-1] * 257]):
        with pytest.raises(ValueError):
            DraftTree(bad)
    with pytest.raises(ValueError):
        DraftTree.from_mask([np.zeros((2, 3), bool)])
    t = DraftTree([[-1, 0, 0, 1, -1], [], list(range(-1, 129))])
    assert t.counts == [5, 0, 130] and t.offsets == [0, 5, 5, 135] and len(t) == 135
    assert t.depths[:5].tolist() == [1, 2, 2, 3, 1] and t.depths[-1] == 130
    m = t.mask("cpu").numpy().view(np.uint64)
    assert m.shape == (135, 3)
    assert m[:5, 0].tolist() == [1, 3, 5, 11, 16]
    assert m[-1].tolist() == [2 ** 64 - 1, 2 ** 64 - 1, 3]


def test_accept_walks_the_drawn_tokens():
    from insitu_b200.tree import DraftTree
    t = DraftTree([[-1, -1, 1, 1, 3]])
    drafted = [5, 7, 8, 9, 4]
    assert t.accept(0, drafted, [0, 9, 0, 4, 6], first=7) == ([1, 3, 4], 6)
    assert t.accept(0, drafted, [0, 9, 0, 3, 6], first=7) == ([1, 3], 3)
    assert t.accept(0, drafted, [2, 0, 0, 0, 0], first=5) == ([0], 2)
    assert t.accept(0, drafted, [2, 0, 0, 0, 0], first=6) == ([], 6)
    with pytest.raises(ValueError):
        t.accept(0, drafted[:4], [0] * 5, 1)


def test_the_c_entry_checks_its_arguments():
    from insitu_b200 import _lib
    L = _lib.lib()
    assert L.ins_tree_workspace(None, 1, None, None) == -1
    assert L.ins_tree_scan(None, 1, None, None, None, 1, None, None, None, 0, None) == _lib.INS_EINVAL
