"""Sampling against its definition in float64 on the CPU, row by row.

Tokens are compared exactly: inputs are seeded, and no row's decision lies
within float32 rounding of a tie (equal logits are exact ties in both, broken
by the index). Log-probabilities: z = x/t - max carries a relative error of
2^-24 from each of the two quotients and the difference, the mass a few 1e-7
(float32 exponentials), so the bound is 2^-22 of the largest |x/t| plus 1e-6."""

from __future__ import annotations

import numpy as np
import pytest

torch = pytest.importorskip("torch")


def reference(x, u, t=1.0, k=0, p=1.0, m=0.0):
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if not (x > -np.inf).any():
        return -1, -np.inf
    top = x.max()
    if t == 0:
        return int(np.argmax(x)), 0.0
    with np.errstate(invalid="ignore", divide="ignore"):
        z = np.where(x == top, 0.0, x / t - top / t)
        order = np.argsort(-x, kind="stable")
        order = order[x[order] > -np.inf]
        if k > 0:
            order = order[:k]
        w = np.exp(z[order])
        if p < 1:
            before = np.cumsum(w) - w
            on = before < p * w.sum()
            order, w = order[on], w[on]
        on = w >= m
        order, w = order[on], w[on]
        key = z[order] - np.log(-np.log(u[order].astype(np.float64)))
    best = order[key == key.max()].min()
    return int(best), float(z[best] - np.log(w.sum()))


def compare(logits, u, settings):
    from insitu_b200.sampling import Sampler
    tokens, logp = Sampler(**settings)(logits, u)
    assert tokens.dtype == torch.int64 and logp.dtype == torch.float32
    tokens, logp = tokens.cpu().numpy(), logp.cpu().numpy()
    x, un = logits.float().cpu().numpy(), u.cpu().numpy()
    pick = lambda name, r: float(np.broadcast_to(np.asarray(settings[name]), len(x))[r]) if name in settings else None
    for r in range(len(x)):
        kw = {short: pick(name, r) for short, name in (("t", "temperature"), ("k", "top_k"), ("p", "top_p"), ("m", "min_p"))
              if name in settings}
        if "k" in kw:
            kw["k"] = int(kw["k"])
        if "p" in kw:
            kw["p"] = float(np.float32(kw["p"]))
        if "m" in kw:
            kw["m"] = float(np.float32(kw["m"]))
        if "t" in kw:
            kw["t"] = float(np.float32(kw["t"]))
        token, lp = reference(x[r], un[r], **kw)
        assert tokens[r] == token, f"row {r}: token {tokens[r]} for {token} ({kw})"
        if np.isfinite(lp):
            finite = x[r][np.isfinite(x[r])]
            scale = np.abs(finite).max() / (kw.get("t") or 1.0)
            assert abs(logp[r] - lp) <= 2.0 ** -22 * scale + 1e-6, f"row {r}: {logp[r]} for {lp}"
        else:
            assert logp[r] == lp


def inputs(rows, vocab, dtype=torch.float32, seed=0, scale=2.5, pad=0):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn((rows, vocab + pad), generator=g, device="cuda") * scale).to(dtype)[:, :vocab]
    return x, torch.rand((rows, vocab), generator=g, device="cuda")


FILTERS = [dict(), dict(top_k=1), dict(top_k=7), dict(top_p=0.9), dict(min_p=0.05), dict(top_p=0.3, temperature=0.5),
           dict(top_k=50, top_p=0.8, min_p=0.02, temperature=0.7), dict(temperature=0), dict(top_p=1e-6),
           dict(min_p=1.0), dict(temperature=30.0, top_p=0.999), dict(top_k=400, top_p=0.99, temperature=2.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 2049, 32003])
def test_every_filter(dtype, vocab):
    x, u = inputs(3, vocab, dtype, seed=vocab)
    for f in FILTERS:
        compare(x, u, f)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,vocab,pad,dtype", [(1, 262144, 0, torch.float32), (5, 128000, 3, torch.bfloat16),
                                                  (300, 5001, 1, torch.float16), (17, 50003, 61, torch.float32)])
def test_settings_of_each_row(rows, vocab, pad, dtype):
    x, u = inputs(rows, vocab, dtype, seed=rows, pad=pad)
    rng = np.random.default_rng(rows)
    compare(x, u, dict(temperature=torch.tensor(rng.choice([0.0, 0.6, 1.0, 1.7], rows).astype(np.float32)),
                       top_k=torch.tensor(rng.choice([0, 1, 40, 3000, 10 ** 6], rows).astype(np.int32)),
                       top_p=torch.tensor(rng.choice([1.0, 0.95, 0.5], rows).astype(np.float32)),
                       min_p=torch.tensor(rng.choice([0.0, 0.0, 0.03], rows).astype(np.float32))))


@pytest.mark.gpu
@pytest.mark.parametrize("settings", [dict(top_k=5), dict(top_k=700), dict(top_p=0.5), dict(top_k=900, top_p=0.25),
                                      dict(temperature=0), dict()])
def test_equal_logits_split_by_index(settings):
    vocab = 5000
    _, u = inputs(4, vocab, seed=9)
    x = torch.zeros((4, vocab), device="cuda")
    x[1] = torch.arange(vocab, device="cuda") % 3            # three values, each often
    x[2] = torch.where(torch.arange(vocab, device="cuda") % 2 == 0, 0.0, -0.0)
    x[3, 100:] = -1e30
    compare(x, u, settings)


@pytest.mark.gpu
@pytest.mark.parametrize("settings", [dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.1), dict(temperature=0),
                                      dict(top_k=40, top_p=0.9, temperature=0.8)])
def test_masked_infinite_and_nan_logits(settings):
    vocab = 3001
    x, u = inputs(7, vocab, seed=4)
    inf = float("inf")
    x[0] = -inf                                             # nothing left
    x[1, :] = -inf
    x[1, 2500] = -3.0                                       # one token left
    x[2, ::2] = float("nan")
    x[3, 17] = inf                                          # a certain token
    x[4, [5, 2900]] = inf                                   # two of them
    x[5] = float("nan")
    x[6, 1:] = -inf
    x[6, 0] = torch.finfo(torch.float32).min                # a mask of the type's lowest value, on the only token
    compare(x, u, settings)


@pytest.mark.gpu
def test_random_numbers_at_the_ends_of_their_range():
    x, u = inputs(3, 500, seed=2)
    u[0] = 0.0                                              # every key is -inf: the lowest kept index
    u[1, 250:] = 0.0
    u[2] = 1.0 - 2.0 ** -24
    compare(x, u, dict(top_k=20))
    compare(x, u, dict())


@pytest.mark.gpu
def test_frequencies_follow_the_kept_probabilities():
    """40,000 draws of one row: each token's count within 5 standard deviations."""
    n, vocab = 40000, 64
    g = torch.Generator("cuda").manual_seed(8)
    row = torch.randn(vocab, generator=g, device="cuda") * 2
    u = torch.rand((n, vocab), generator=g, device="cuda")
    from insitu_b200.sampling import Sampler
    tokens, logp = Sampler(temperature=0.9, top_k=12)(row.expand(n, -1), u)
    p = torch.softmax(torch.where(row >= row.topk(12).values[-1], row.double() / 0.9, -np.inf), 0)
    counts = torch.bincount(tokens, minlength=vocab).double()
    assert bool(((counts - n * p).abs() <= 5 * torch.sqrt(n * p * (1 - p)) + 1e-9).all())
    assert torch.allclose(logp.double(), torch.log(p)[tokens], atol=1e-5)


@pytest.mark.gpu
def test_the_stream_of_the_call_is_used_and_runs_repeat():
    from insitu_b200.sampling import Sampler
    x, u = inputs(64, 30011, torch.bfloat16, seed=6)
    s = Sampler(top_p=0.9, top_k=100)
    first = s(x, u)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        again = s(x, u)
    torch.cuda.synchronize()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    empty = s(x[:0], u[:0])
    assert empty[0].shape == (0,) and empty[1].shape == (0,)


def test_settings_are_checked():
    from insitu_b200.sampling import Sampler
    for bad in (dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")),
                dict(top_p=0.0), dict(top_p=1.5), dict(min_p=-0.1), dict(min_p=1.1), dict(top_k=-1),
                dict(top_p=torch.tensor([0.5, 2.0])), dict(top_k=torch.tensor([[1]])),
                dict(top_k=torch.tensor([1, 2]), top_p=torch.tensor([0.5]))):
        with pytest.raises(ValueError):
            Sampler(**bad)
    with pytest.raises(TypeError):
        Sampler(top_k=2.5)
    with pytest.raises(ValueError):
        Sampler()(torch.zeros(2, 8), torch.zeros(2, 8))     # not on the GPU


def test_the_c_entry_checks_its_arguments():
    from insitu_b200 import _lib
    L = _lib.lib()
    call = lambda rows, vocab, dtype: L.ins_sample(rows, vocab, None, dtype, vocab, None, vocab, None, None, None, None,
                                                   None, None, None)
    assert call(-1, 8, 0) == _lib.INS_EINVAL
    assert call(1, 0, 0) == _lib.INS_EINVAL
    assert call(1, (1 << 18) + 1, 0) == _lib.INS_EINVAL
    assert call(1, 8, 9) == _lib.INS_EINVAL
    assert call(1, 8, 0) == _lib.INS_EINVAL                 # NULL buffers
    assert call(0, 8, 0) == _lib.INS_OK


@pytest.mark.gpu
def test_tensors_are_checked():
    from insitu_b200.sampling import Sampler
    x, u = inputs(4, 100)
    for logits, uniform, sampler in ((x.double(), u, Sampler()), (x, u.double(), Sampler()), (x, u[:, :50], Sampler()),
                                     (x.t(), u.t(), Sampler()), (x[0], u[0], Sampler()), (x, u.cpu(), Sampler()),
                                     (x, u, Sampler(top_k=torch.tensor([1, 2, 3]))),
                                     (torch.zeros((1, (1 << 18) + 1), device="cuda"),
                                      torch.zeros((1, (1 << 18) + 1), device="cuda"), Sampler())):
        with pytest.raises(ValueError):
            sampler(logits, uniform)
