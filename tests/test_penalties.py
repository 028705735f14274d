"""Penalties, biases and masks on logits against the definition in float64.

The kernel computes in fp32: the quotient or product, the product of frequency
and count, two differences and the bias's sum, half a unit of fp32 (2^-24) each
of the values' sizes; then one rounding to the logits' type."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")

TYPES = [torch.float32, torch.float16, torch.bfloat16]


def expected(x, settings, tokens=None, lengths=None, prompts=None, of=None, drafted=None, bias=None, mask=None):
    """The definition, row by row: y and the sum of the magnitudes behind it."""
    x = x.double().cpu().numpy()
    rows, vocab = x.shape
    get = lambda t: None if t is None else t.cpu().numpy()
    tokens, lengths, prompts, of, drafted, bias, mask = map(get, (tokens, lengths, prompts, of, drafted, bias, mask))
    y, size = x.copy(), np.abs(x)
    for i in range(rows):
        asked, said = np.zeros(vocab, bool), np.zeros(vocab)
        h = i if of is None else int(of[i])
        if tokens is not None and 0 <= h < len(tokens):
            n = tokens.shape[1] if lengths is None else min(max(int(lengths[h]), 0), tokens.shape[1])
            m = 0 if prompts is None else int(prompts[h])
            for j in range(n):
                t = int(tokens[h, j])
                if 0 <= t < vocab:
                    if j < m:
                        asked[t] = True
                    else:
                        said[t] += 1
        for t in (drafted[i] if drafted is not None else ()):
            if 0 <= t < vocab:
                said[t] += 1
        r, p, f = (np.float64(np.float32(settings[k][i] if np.ndim(settings[k]) else settings[k]))
                   for k in ("repetition", "presence", "frequency"))
        seen = asked | (said > 0)
        with np.errstate(invalid="ignore"):
            y[i] = np.where(seen, np.where(x[i] > 0, x[i] / r, x[i] * r), x[i])
            size[i] = np.abs(y[i]) + np.abs(f) * said + np.abs(p) * (said > 0)
            y[i] = np.where(said > 0, y[i] - f * said - p, y[i])
            if bias is not None:
                b = bias[i % len(bias)].astype(np.float64)
                y[i] += b
                size[i] += np.abs(b)
        if mask is not None:
            w = mask[i % len(mask)].view(np.uint32)
            allowed = (w[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            y[i, allowed.reshape(-1)[:vocab] == 0] = -np.inf
    return y, size


def check(got, logits, settings, **kw):
    want, size = expected(logits, settings, **kw)
    assert got.dtype == logits.dtype and got.shape == logits.shape
    have = got.double().cpu().numpy()
    info = torch.finfo(logits.dtype)
    err = 4 * 2.0 ** -24 * size
    with np.errstate(invalid="ignore", over="ignore"):
        limit = err + info.eps / 2 * (np.abs(want) + err) + info.smallest_normal * info.eps / 2
        big = np.abs(want) >= info.max                       # beyond the type: its infinity, or its largest number
        ok = (np.abs(have - want) <= limit) | (have == want) | (np.isnan(have) & np.isnan(want))
        ok |= big & (np.sign(have) == np.sign(want)) & (np.abs(have) >= info.max)
    assert ok.all(), np.argwhere(~ok)[:5]


def setup(rng, rows, vocab, dtype, history, pad=0, per_row=True):
    x = torch.from_numpy(rng.standard_normal((rows, vocab + pad)).astype(np.float32) * 3).cuda().to(dtype)[:, :vocab]
    tokens = torch.from_numpy((vocab * rng.random((rows, history)) ** 3).astype(np.int64)).cuda()
    pick = lambda *v: [float(rng.choice(v)) for _ in range(rows)]
    settings = {"repetition": pick(1.0, 1.2, 0.7), "presence": pick(0.0, 0.5, -1.0), "frequency": pick(0.0, 0.3, -0.1)}
    if not per_row:
        settings = {"repetition": 1.3, "presence": 0.25, "frequency": 0.125}
    return x, tokens, settings


def ints(*values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def some_mask(rng, rows, vocab):
    words = -(-vocab // 32)
    m = rng.integers(0, 2 ** 32, (rows, words), dtype=np.uint32)
    m[rng.random((rows, words)) < 0.3] = 0
    m[rng.random((rows, words)) < 0.3] = 2 ** 32 - 1
    return torch.from_numpy(m.view(np.int32)).cuda()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 32, 33, 257, 1000, 4097, 40_009])
@pytest.mark.parametrize("pad", [0, 1, 3, 8])
def test_sizes_types_and_strides(dtype, vocab, pad):
    from insitu_b200 import Penalties
    rng = np.random.default_rng(vocab + pad)
    x, tokens, settings = setup(rng, 3, vocab, dtype, 50, pad)
    kw = dict(tokens=tokens, lengths=ints(50, 0, 31), prompts=ints(10, 5, 31))
    check(Penalties(**settings)(x, **kw), x, settings, **kw)
    kw.update(bias=torch.from_numpy(rng.standard_normal((3, vocab)).astype(np.float32)).cuda(),
              mask=some_mask(rng, 3, vocab))
    check(Penalties(**settings)(x, **kw), x, settings, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [1, 2, 40, 300])
@pytest.mark.parametrize("per_row", [True, False])
def test_batches(rows, per_row):
    from insitu_b200 import Penalties
    rng = np.random.default_rng(rows)
    x, tokens, settings = setup(rng, rows, 5000, torch.bfloat16, 300, per_row=per_row)
    kw = dict(tokens=tokens, prompts=torch.arange(rows, device="cuda", dtype=torch.int32))
    p = Penalties(**settings)
    check(p(x, **kw), x, settings, **kw)
    shared = dict(bias=torch.from_numpy(rng.standard_normal((1, 5000)).astype(np.float32)).cuda(),
                  mask=some_mask(rng, 1, 5000))
    check(p(x, **kw, **shared), x, settings, **kw, **shared)
    flat = {k: v[0] for k, v in shared.items()}
    assert torch.equal(p(x, **kw, **flat), p(x, **kw, **shared))


@pytest.mark.gpu
@pytest.mark.parametrize("history", [0, 1, 255, 256, 257, 20_000])
@pytest.mark.parametrize("vocab", [5, 128_256, 262_144])
def test_long_histories_and_wide_vocabularies(history, vocab):
    from insitu_b200 import Penalties
    rng = np.random.default_rng(history)
    x, tokens, settings = setup(rng, 2, vocab, torch.float32, history)
    tokens[0, history // 2:] = min(3, vocab - 1)              # one token, very often
    kw = dict(tokens=tokens, prompts=ints(0, history // 3))
    check(Penalties(**settings)(x, **kw), x, settings, **kw)


@pytest.mark.gpu
def test_nodes_of_trees_add_their_paths():
    from insitu_b200 import DraftTree, Penalties
    rng = np.random.default_rng(1)
    tree = DraftTree([[-1, 0, 0, 1, -1], [], [-1, 0, 1]])
    drafted = rng.integers(0, 20, len(tree)).tolist()
    paths, of = tree.paths(drafted, "cuda"), tree.sequences("cuda")
    assert of.tolist() == [0] * 5 + [2] * 3 and paths.shape == (8, 3)
    d = drafted
    assert paths[:5].tolist() == [[d[0], -1, -1], [d[0], d[1], -1], [d[0], d[2], -1], [d[0], d[1], d[3]], [d[4], -1, -1]]
    x, _, settings = setup(rng, 8, 700, torch.float16, 1)
    tokens = torch.from_numpy(rng.integers(0, 20, (3, 30))).cuda()
    kw = dict(tokens=tokens, lengths=ints(30, 4, 9), prompts=ints(3, 0, 9), of=of, drafted=paths)
    check(Penalties(**settings)(x, **kw), x, settings, **kw)
    check(Penalties(**settings)(x, drafted=paths), x, settings, drafted=paths)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("history", [1400, 12_289])
def test_many_rows_of_shared_sequences(dtype, history):
    """Sequences' own tokens, drafted ones among them and beside them, repeated;
    sequences that no row names; rows aligned and not; more tokens of a slice
    than its list holds."""
    from insitu_b200 import Penalties
    rng = np.random.default_rng(history)
    for rows, vocab, pad, m in ((48, 30_001, 0, 5), (50, 9000, 3, 0), (64, 40_960, 0, 256)):
        x, _, settings = setup(rng, rows, vocab, dtype, 1, pad)
        tokens = torch.from_numpy((vocab * rng.random((5, history)) ** 3).astype(np.int64)).cuda()
        tokens[1] = 7
        tokens[2, ::2] = -1
        kw = dict(tokens=tokens, lengths=ints(history, history, history - 1, 0, history), prompts=ints(0, 9, history, 4, -2),
                  of=torch.from_numpy(rng.integers(0, 4, rows).astype(np.int32)).cuda())
        if m:
            drafted = torch.from_numpy((vocab * rng.random((rows, m)) ** 6).astype(np.int64)).cuda()
            drafted[:, m // 2] = drafted[:, 0]
            drafted[::3, 1:] = -1
            kw["drafted"] = drafted
        p = Penalties(**settings)
        want = p(x, **kw)
        check(want, x, settings, **kw)
        more = dict(bias=torch.from_numpy(rng.standard_normal((1, vocab)).astype(np.float32)).cuda(),
                    mask=some_mask(rng, rows, vocab))
        check(p(x, **kw, **more), x, settings, **kw, **more)
        y = x.contiguous()
        assert torch.equal(p(y, **kw, out=y), want)


@pytest.mark.gpu
def test_ids_that_are_no_tokens_and_rows_that_are_no_sequences():
    from insitu_b200 import Penalties
    rng = np.random.default_rng(2)
    x, tokens, settings = setup(rng, 4, 100, torch.float32, 40)
    tokens[:, ::3] = -1
    tokens[:, 1::5] = 100
    tokens[0, 2], tokens[1, 2], tokens[2, 2] = 2 ** 62, -2 ** 63, 2 ** 32 + 5
    kw = dict(tokens=tokens[:2], lengths=ints(1000, -4), prompts=ints(-3, 2000), of=ints(1, -1, 2, 0), drafted=tokens)
    check(Penalties(**settings)(x, **kw), x, settings, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_infinite_and_nan_logits(dtype):
    from insitu_b200 import Penalties
    rng = np.random.default_rng(3)
    x, tokens, settings = setup(rng, 3, 200, dtype, 60)
    x = x.contiguous()
    x[:, ::7], x[:, 1::7], x[:, 2::7], x[:, 3::7] = -np.inf, np.inf, np.nan, torch.finfo(dtype).min
    x[:, 4::7] = 0.0
    bias = torch.zeros((1, 200), device="cuda")
    bias[:, 5::9], bias[:, 4::9] = -np.inf, torch.finfo(torch.float32).min
    mask = some_mask(rng, 3, 200)
    mask[1] = 0                                                # nothing is allowed
    kw = dict(tokens=tokens, bias=bias, mask=mask)
    got = Penalties(**settings)(x, **kw)
    check(got, x, settings, **kw)
    assert torch.isinf(got[1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [0, 5])
def test_in_place_into_views_and_without_settings(pad):
    from insitu_b200 import Penalties
    rng = np.random.default_rng(4)
    x, tokens, settings = setup(rng, 5, 3001, torch.bfloat16, 80, pad)
    before, mask = x.clone(), some_mask(rng, 5, 3001)
    want = Penalties(**settings)(x, tokens, mask=mask)
    assert torch.equal(x, before)
    for width, first in ((3001, 0), (3010, 0), (3010, 3), (3009, 8)):
        wide = torch.full((5, width), 7.0, dtype=x.dtype, device="cuda")
        out = wide[:, first:first + 3001]
        assert Penalties(**settings)(x, tokens, mask=mask, out=out) is out
        assert torch.equal(out, want)
        assert (wide[:, :first] == 7).all() and (wide[:, first + 3001:] == 7).all()
    assert torch.equal(Penalties()(x, tokens), x)              # neutral settings: a copy
    assert torch.equal(Penalties(**settings)(x), x)            # no tokens
    assert Penalties(**settings)(x, tokens, mask=mask, out=x) is x
    assert torch.equal(x, want)
    again = x[:1].expand(4, -1)                                # one row for all
    assert torch.equal(Penalties()(again), again)


@pytest.mark.gpu
def test_another_stream_and_a_graph():
    from insitu_b200 import Penalties
    rng = np.random.default_rng(5)
    x, tokens, settings = setup(rng, 6, 9000, torch.float16, 500)
    p = Penalties(**settings)
    first = p(x, tokens)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = [p(x, tokens) for _ in range(3)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = p(x, tokens)
    held.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for y in again + [held]:
        assert torch.equal(first, y)
    # new inputs in the captured buffers give their own results
    tokens.random_(0, 9000)
    graph.replay()
    torch.cuda.synchronize()
    check(held, x, settings, tokens=tokens)


@pytest.mark.gpu
def test_a_draw_under_a_grammar_stays_in_it():
    """Penalties, then the sampler: only allowed tokens are drawn, and a row
    that allows nothing draws none."""
    from insitu_b200 import Penalties, Sampler
    rng = np.random.default_rng(6)
    x, tokens, settings = setup(rng, 64, 12_000, torch.bfloat16, 100)
    mask = some_mask(rng, 64, 12_000)
    mask[5] = 0
    y = Penalties(**settings)(x, tokens, mask=mask)
    token, logp = Sampler(temperature=0.9, top_k=40)(y, torch.rand((64, 12_000), device="cuda"))
    word = mask.gather(1, (token.clamp(min=0) // 32)[:, None])[:, 0]
    allowed = (word >> (token.clamp(min=0) % 32).int()) & 1
    assert token[5] == -1 and torch.isinf(logp[5])
    assert (allowed[torch.arange(64, device="cuda") != 5] == 1).all()


@pytest.mark.gpu
def test_refusals():
    from insitu_b200 import Penalties
    x = torch.zeros((3, 100), device="cuda")
    tokens = torch.zeros((3, 4), dtype=torch.int64, device="cuda")
    p = Penalties(repetition=1.2)
    bad = [dict(tokens=tokens[:2]), dict(tokens=tokens.int()), dict(tokens=tokens.cpu()), dict(tokens=tokens[0]),
           dict(tokens=tokens.T), dict(lengths=ints(1, 1, 1)), dict(tokens=tokens, lengths=ints(1, 1)),
           dict(tokens=tokens, lengths=ints(1, 1, 1).long()), dict(tokens=tokens, prompts=ints(1)),
           dict(tokens=tokens, of=ints(0, 0)), dict(of=ints(0, 0, 0)), dict(drafted=tokens[:2]),
           dict(bias=torch.zeros(99, device="cuda")), dict(bias=torch.zeros((2, 100), device="cuda")),
           dict(bias=torch.zeros(100, device="cuda").half()), dict(bias=torch.zeros(100)),
           dict(mask=torch.zeros(100, dtype=torch.int32, device="cuda")),
           dict(mask=torch.zeros((2, 4), dtype=torch.int32, device="cuda")),
           dict(mask=torch.zeros(4, dtype=torch.int64, device="cuda")),
           dict(out=torch.zeros((3, 100), device="cuda").half()), dict(out=torch.zeros((2, 100), device="cuda")),
           dict(out=torch.zeros((1, 100), device="cuda").expand(3, -1)), dict(out=torch.zeros((3, 100)))]
    for kw in bad:
        with pytest.raises(ValueError):
            p(x, **kw)
    wide = torch.zeros((4, 100), device="cuda")
    with pytest.raises(ValueError):
        p(wide[:3], out=wide[1:])                              # overlaps the logits
    for logits in (x.double(), x[0], x.cpu(), x.T, torch.zeros((1, (1 << 18) + 1), device="cuda"), x[:, :0]):
        with pytest.raises(ValueError):
            p(logits)
    with pytest.raises(ValueError):
        Penalties(presence=[0.0, 1.0])(x)                      # settings of two rows
    assert p(x[:0]).shape == (0, 100)


def test_settings_are_checked():
    from insitu_b200 import Penalties
    for kw in (dict(repetition=0.0), dict(repetition=-1.0), dict(repetition=float("nan")), dict(presence=float("inf")),
               dict(frequency=[0.0, float("nan")]), dict(presence=[[0.0]]), dict(presence=[0.0], frequency=[0.0, 1.0])):
        with pytest.raises(ValueError):
            Penalties(**kw)


def test_paths_are_checked():
    from insitu_b200.tree import DraftTree
    t = DraftTree([[-1, 0], [-1]])
    assert t.paths([7, 8, 9]).tolist() == [[7, -1], [7, 8], [9, -1]]
    assert t.paths(torch.tensor([7, 8, 9])).tolist() == [[7, -1], [7, 8], [9, -1]]
    assert t.sequences().tolist() == [0, 0, 1]
    assert DraftTree([]).paths([]).shape == (0, 0)
    with pytest.raises(ValueError):
        t.paths([1, 2])
    with pytest.raises(ValueError):
        DraftTree.from_mask([np.eye(2, dtype=bool)]).paths([1, 2])


def test_the_c_entry_checks_its_arguments():
    import ctypes as C
    from insitu_b200 import _lib
    L, p = _lib.lib(), _lib.PenaltiesArgs()
    for args in ((-1, 5, None, 0, 5, None, 5), (1, 0, None, 0, 5, None, 5), (1, 5, None, 9, 5, None, 5),
                 (1, 5, None, 0, 5, None, 5), (1, (1 << 18) + 1, None, 0, 5, None, 5)):
        assert L.ins_penalize(*args, C.byref(p), None) == _lib.INS_EINVAL
    assert L.ins_penalize(0, 5, None, 0, 5, None, 5, None, None) == _lib.INS_OK


def test_histories_whose_indexes_would_wrap_are_refused():
    import ctypes as C
    from insitu_b200 import _lib
    L, x = _lib.lib(), C.create_string_buffer(64)              # refused before any of it is read
    at = C.cast(x, C.c_void_p)
    for sizes in (dict(history=(1 << 30) + 1, histories=1), dict(n_drafted=(1 << 30) + 1), dict(history=2 ** 31 - 1)):
        p = _lib.PenaltiesArgs(**sizes)
        assert L.ins_penalize(1, 5, at, 0, 5, at, 5, C.byref(p), None) == _lib.INS_EBADLEN
