"""Tree attention against a float64 computation over the operands that the
kernels round to fp16, so that the bound stays near the output's own rounding
whatever the scores' size.

What is rounded before the products (q' = fp16(q log2(e)), c = fp16(centroid),
and for more than 64 query rows a KV head K = fp16(c hi + fp16(c lo)) with the
norm's halves hi + lo, V likewise) is rounded here the same way, in the units
that the kernels use: q/2^16 and norm/2^9, and the power of two that the cache's
formats need beyond these on the scores (more than 64 rows: on the queries, or
up to 2^5 on the keys) and on the output. Left over, for
one output of T tokens seen with weights a_r and values v_r:

* a score is a sum of 64 products in fp32, by tensor cores that may truncate:
  at most 68 additions of 2^-23 of the largest partial sum, then two fp32
  roundings; d_r = 2^-16 sum|q' k_r| covers them, and the weight's relative
  error is e_r = 2^d_r - 1 + 2^-21 (the exponential's 2^-22 twice);
* P (up to 64 rows: weight times value norm) is rounded to fp16: 2^-11 of each
  term, and 2^-25 where it is below fp16's normal range, in units of 2^9 /
  2^norm_frac and of a sum that is at least 1 (many rows: of 2^-7 of that);
* the sums over tokens are fp32 in steps of 16: (T / 16 + 64) 2^-23 each.

So the sum that is rounded to bf16 lies within err = 1.1 (sum a (e + s) |v|
+ |ref| sum a (e + s)) + 2^-11 sum a |v| + floor of ref, with s the sums' term
and 1.1 for the second order. That rounding is monotone, so the output lies
between the roundings of ref - err and ref + err.

Where scores are huge that says nothing, but weights relative to the largest
one, W_r = 2^(s_r - s_top), still do: they move by factors of 2^(d_r + d_top) at
most, and W_top not at all. The smaller of both is taken."""

from __future__ import annotations

import numpy as np
import pytest

from test_tree import random_tree

torch = pytest.importorskip("torch")


def cache(kb, vb, groups, n_kv, page, lens, norm_frac=9, **fmt):
    from insitu_b200 import FixedFormat, Geometry, PagedCache, QuantConfig
    return PagedCache(QuantConfig(key_bits=kb, value_bits=vb, norm_frac=norm_frac), FixedFormat(**fmt),
                      Geometry(n_kv, groups, 64), max_seqs=len(lens), capacity=max(16, *lens), page_tokens=page)


def packed(rng, pc, norms):
    """Random codes under these norms (n, n_kv, 2)."""
    n = len(norms)
    rows = rng.integers(0, 256, (n, pc.geo.n_kv_heads, pc.row_bytes), dtype=np.uint8)
    rows[..., -4:] = np.ascontiguousarray(norms.astype("<i2")).view(np.uint8).reshape(n, pc.geo.n_kv_heads, 4)
    return rows


def half(x):
    return np.asarray(x, np.float64).astype(np.float16).astype(np.float64)


def reference(pc, q, rows, see):
    """q (n, heads, 64) int32, see (n, T) -> out and err, (n, heads, 64)."""
    from insitu_b200 import KVQuantizer
    g, nf, T = pc.geo, pc.quant.norm_frac, len(rows)
    n = len(q)
    shift = 25 - pc.fmt.qk_frac - nf
    many = n * g.kv_groups > 64 and (pc.quant.key_bits, pc.quant.value_bits) in ((4, 2), (3, 3)) and shift <= 5
    kv = KVQuantizer(64, pc.quant, pc.fmt).unpack(rows)
    unit = np.float32(np.float32(1.4426950408889634) / np.float32(65536) * np.float32(2.0 ** min(shift, 0) if many else 1))
    qh = (q.astype(np.float32) * unit).astype(np.float16).astype(np.float64).reshape(n, g.n_kv_heads, g.kv_groups, 64)
    score_unit, out_unit = 1.0 if many else 2.0 ** shift, 2.0 ** (9 - nf)

    def side(cent, idx, norm, factor):
        c = half(cent / 2.0 ** pc.fmt.centroid_frac)[idx]
        x = norm.astype(np.float64)[..., None] / 512 * factor
        if not many:
            return c, x
        hi = half(x)
        return half(c * hi + half(c * half(x - hi))), np.ones_like(x)

    dev = "cuda"
    kc, kn = (torch.from_numpy(x).to(dev) for x in side(pc.tables.k_centroids, kv.k_idx, kv.k_norm,
                                                     2.0 ** max(shift, 0) if many else 1))
    vc, vn = (torch.from_numpy(x).to(dev) for x in side(pc.tables.v_centroids, kv.v_idx, kv.v_norm, 1))
    qh, see = torch.from_numpy(qh).to(dev), torch.from_numpy(see).to(dev)
    out, bound = [], []
    for i in range(n):                      # a node at a time: (n_kv, groups, T)
        dot = torch.einsum("hgd,thd->hgt", qh[i], kc)
        size = torch.einsum("hgd,thd->hgt", qh[i].abs(), kc.abs())
        scale = kn[..., 0].T[:, None] * score_unit
        s = torch.where(see[i], dot * scale, -torch.inf)
        some = bool(see[i].any())
        m = s.amax(-1, keepdim=True) if some else torch.zeros_like(s[..., :1])
        a = torch.exp2(s - m)
        a = a / a.sum(-1, keepdim=True).clamp(min=1e-300)
        d = 2.0 ** -16 * size * scale.abs()
        rest = 2.0 ** -21 + (T / 16 + 64) * 2.0 ** -23
        err = (torch.exp2(d) - 1).clamp(max=1e300) + rest
        v = vc * vn * out_unit
        o = torch.einsum("hgt,thd->hgd", a, v)
        reach = torch.einsum("hgt,thd->hgd", a, v.abs())
        wrong = torch.where(see[i], a * err, 0.0)
        top = s.argmax(-1, keepdim=True)
        d = torch.where(see[i], d + d.gather(-1, top), 0.0)
        moved = (torch.exp2((s - m + d).clamp(max=900)) - torch.exp2(s - m)).scatter(-1, top, 0.0)
        least = torch.exp2(s - m - d).scatter(-1, top, 1.0).sum(-1, keepdim=True)
        near = 1.1 * (torch.einsum("hgt,thd->hgd", wrong, v.abs()) + o.abs() * wrong.sum(-1, keepdim=True))
        far = (torch.einsum("hgt,thd->hgd", moved, v.abs()) + o.abs() * moved.sum(-1, keepdim=True)) / least
        floor = T * 2.0 ** (-32 if many else -25) * float(vc.abs().max()) * out_unit
        out.append(o)
        bound.append(2.0 ** -11 * reach + floor + torch.fmin(near, far + 1.1 * rest * (reach + o.abs())))
    shape = (n, g.num_heads, 64)
    return torch.stack(out).reshape(shape), torch.stack(bound).reshape(shape)


def run(kb, vb, groups, context, nodes, norms, q_std, seed, page=64, **formats):
    """norms: (rng, shape) -> integers; q_std: of the queries, in their integer units."""
    from insitu_b200 import DraftTree
    rng = np.random.default_rng(seed)
    pc = cache(kb, vb, groups, 2, page, [context + nodes], **formats)
    rows = packed(rng, pc, norms(rng, (context + nodes, 2, 2)))
    pc.put_rows([0], [len(rows)], torch.from_numpy(rows).to(pc.device))
    tree = DraftTree([random_tree(rng, nodes)])
    bits = tree.mask("cpu").numpy().view(np.uint64)[:, 0, None] >> np.arange(nodes, dtype=np.uint64) & np.uint64(1)
    see = np.concatenate([np.ones((nodes, context), bool), bits.astype(bool)], 1)
    q = np.clip(np.rint(rng.standard_normal((nodes, pc.geo.num_heads, 64)) * q_std), -2 ** 31 + 1, 2 ** 31 - 1)
    q = q.astype(np.int32)
    got = pc.tree_scan([0], torch.from_numpy(q).to(pc.device), tree)
    pc.status()
    want, err = reference(pc, q, rows, see)
    pc.close()
    assert torch.isfinite(got).all()
    low, high = ((want + x).float().to(torch.bfloat16) for x in (-err, err))
    assert bool(((low <= got) & (got <= high)).all()), \
        f"{int(((got < low) | (high < got)).sum())} outside, by {float(((got.double() - want).abs() / err).max())} of err"


WIDTHS = [(4, 2), (3, 3), (8, 5)]


def small(rng, shape):
    """Norms near 1 whatever the format: a few units at few fraction bits."""
    return np.clip(np.rint(12 + 4 * rng.standard_normal(shape)), 1, 32767)


def large(rng, shape):
    return rng.integers(-32768, 32768, shape)


@pytest.mark.gpu
@pytest.mark.parametrize("kb,vb", WIDTHS)
@pytest.mark.parametrize("nodes", [1, 3, 6, 24, 64])
@pytest.mark.parametrize("norm_frac,qk_frac,centroid_frac", [(0, 8, 15), (4, 16, 15), (6, 12, 12), (7, 16, 15),
                                                             (9, 20, 17), (12, 16, 15), (15, 24, 15)])
@pytest.mark.parametrize("norms", [small, large])
def test_fraction_bits(kb, vb, nodes, norm_frac, qk_frac, centroid_frac, norms):
    """Norms beyond 2^8 and queries beyond fp16 in real units; scores of a few
    units, so that many tokens keep weight."""
    size = 12 if norms is small else 18918
    q_std = 2.0 / (8 * 0.9 * size / 2 ** norm_frac) * 2 ** qk_frac
    run(kb, vb, 4, 700, nodes, norms, q_std, seed=norm_frac + nodes, norm_frac=norm_frac, qk_frac=qk_frac,
        centroid_frac=centroid_frac)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 6, 24, 64])
@pytest.mark.parametrize("norm_frac,qk_frac", [(0, 0), (0, 15), (3, 4), (15, 28)])
def test_queries_of_all_32_bits(nodes, norm_frac, qk_frac):
    """One token takes the weight, at any format."""
    run(4, 2, 4, 300, nodes, large, 2.0 ** 29, seed=nodes, norm_frac=norm_frac, qk_frac=qk_frac)


def near_one(rng, shape):
    return np.clip(np.rint(512 + 60 * rng.standard_normal(shape)), 1, 32767)


@pytest.mark.gpu
@pytest.mark.parametrize("kb,vb", [(4, 2), (3, 3), (3, 2)])
@pytest.mark.parametrize("nodes", [1, 3, 6, 12, 24, 64])
@pytest.mark.parametrize("scale", [0.0, 0.25, 4.0, 60.0])
def test_scores_of_every_size(kb, vb, nodes, scale):
    """From the plain mean to one token that takes all the weight, maxima
    rising late and often; the widths that a cache has by default among them."""
    run(kb, vb, 4, 3000, nodes, near_one, scale * 65536, seed=nodes)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 3, 6, 12, 24, 64])
@pytest.mark.parametrize("groups", [1, 8])
def test_norms_of_either_sign_and_every_size(nodes, groups):
    run(4, 2, groups, 700, nodes, large, 0.01 * 65536, seed=nodes)


@pytest.mark.gpu
def test_formats_that_the_products_do_not_cover_are_refused():
    from insitu_b200 import DraftTree
    pc = cache(4, 2, 4, 1, 16, [16], qk_frac=-1)
    pc.put_rows([0], [3], torch.zeros((3, 1, 52), dtype=torch.uint8, device=pc.device))
    with pytest.raises(ValueError):
        pc.tree_scan([0], torch.zeros((1, 4, 64), dtype=torch.int32, device=pc.device), DraftTree([[-1]]))
    pc.close()
