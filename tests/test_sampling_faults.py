"""Rows of logits whose sampling once went wrong, against the definition in
float64 (and its tolerances) of test_sampling.py."""

from __future__ import annotations

import numpy as np
import pytest

from test_sampling import inputs, reference

torch = pytest.importorskip("torch")


def compare(logits, u, t=1.0, k=0, p=1.0, m=0.0):
    """One setting for all rows; a row may hold no finite logit."""
    from insitu_b200.sampling import Sampler
    tokens, logp = (y.cpu().numpy() for y in Sampler(temperature=t, top_k=k, top_p=p, min_p=m)(logits, u))
    x, un = logits.float().cpu().numpy(), u.cpu().numpy()
    t, p, m = (float(np.float32(v)) for v in (t, p, m))
    for r in range(len(x)):
        token, lp = reference(x[r], un[r], t, k, p, m)
        assert tokens[r] == token, f"row {r}: token {tokens[r]} for {token}"
        scale = np.abs(x[r][np.isfinite(x[r])]).max(initial=0.0) / t
        if np.isfinite(lp):
            assert abs(logp[r] - lp) <= 2.0 ** -22 * scale + 1e-6, f"row {r}: {logp[r]} for {lp}"
        else:
            assert logp[r] == lp


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("vocab", [40, 3001, 40000])
@pytest.mark.parametrize("settings", [dict(k=1), dict(k=2), dict(k=5), dict(p=0.4), dict(p=0.6), dict(k=2, p=0.5),
                                      dict(k=3, p=0.34, t=0.5), dict(m=0.5), dict(k=30, t=3.0), dict()])
def test_several_infinite_logits_are_cut_by_their_index(settings, vocab, dtype):
    """Logits of +inf (an overflow of fp16 is enough) share all of the mass
    evenly; the cuts keep the lowest indexes."""
    x, u = inputs(5, vocab, dtype, seed=vocab)
    inf = float("inf")
    x[0, [3, vocab - 1]] = inf
    x[1, [7, 20, vocab - 2]] = inf
    x[2, vocab // 2:] = inf                     # more than a list holds
    x[3] = inf
    x[4, [0, 1, 2]] = torch.tensor([inf, -inf, float("nan")], dtype=dtype, device="cuda")
    x[4, vocab - 1] = inf
    u[:, :10] = 0.25                            # a lower index does not win by its number
    u[:, -1] = 0.99
    compare(x, u, **settings)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 40, 5001, 40000])
@pytest.mark.parametrize("k,p", [(0, 1.0), (7, 1.0), (0, 0.8), (7, 0.8)])
def test_a_min_p_that_keeps_nothing_writes_its_outputs(vocab, k, p):
    """The C entry takes any min_p: rows above 1, infinite or NaN have no token
    left, the rows beside them are drawn as always."""
    from insitu_b200 import _lib
    x, u = inputs(5, vocab, seed=vocab)
    x[4] = -float("inf")
    column = lambda v, dtype: torch.tensor(v, dtype=dtype, device="cuda")
    m = column([1.5, float("nan"), 0.02, float("inf"), 0.0], torch.float32)
    top_k, top_p = column([k] * 5, torch.int32), column([p] * 5, torch.float32)
    tokens = torch.full((5,), 777, dtype=torch.int64, device="cuda")
    logp = torch.full((5,), 777.0, device="cuda")
    at = lambda t: t.data_ptr()
    _lib.check(_lib.lib().ins_sample(5, vocab, at(x), 0, x.stride(0), at(u), u.stride(0), None, at(top_k), at(top_p),
                                     at(m), at(tokens), at(logp), torch.cuda.current_stream().cuda_stream))
    token, lp = reference(x[2].cpu().numpy(), u[2].cpu().numpy(), 1.0, k, float(np.float32(p)), float(np.float32(0.02)))
    assert tokens.tolist() == [-1, -1, token, -1, -1]
    assert torch.isinf(logp[[0, 1, 3, 4]]).all() and abs(float(logp[2]) - lp) <= 2.0 ** -22 * 20 + 1e-6
    op = _lib.ops().sample(x, u, None, top_k, top_p, m)
    assert torch.equal(op[0], tokens) and torch.equal(op[1], logp)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [128000, 262144])
@pytest.mark.parametrize("settings", [dict(), dict(k=120000), dict(m=1e-10), dict(k=120000, t=2.0)])
def test_a_flat_tail_far_below_the_peak_counts_in_the_log_probability(vocab, settings):
    """Tokens 22.2 to 23 nats under the maximum weigh less than 2^-32 each, and
    together 3e-5: summed to 2^-31 they were nothing."""
    x, u = inputs(3, vocab, seed=vocab)
    t = settings.get("t", 1.0)
    x = (-22.6 + 0.15 * x) * t                  # 2.5 * 0.15 nats wide
    x[:, 777] = 0.0
    x[1] = x[1].clamp(min=-22.9 * t)
    x[2, ::3] = -22.3 * t
    compare(x, u, **settings)


def _sleep():
    torch.cuda._sleep(200_000_000)              # about a tenth of a second of this stream


def _drawn(settings, x, u):
    from insitu_b200.sampling import Sampler
    out = Sampler(**settings)(x, u)
    torch.cuda.synchronize()
    return out


SETTINGS = dict(temperature=1.7, top_k=40, top_p=0.9, min_p=0.01)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [9, 700])
def test_a_sampler_fills_its_settings_before_another_stream_reads_them(rows):
    """A second stream's call, not ordered after the first stream's: the first
    stream has still a tenth of a second of other work to do."""
    from insitu_b200.sampling import Sampler
    x, u = inputs(rows, 500, seed=1)
    want = _drawn(SETTINGS, x, u)
    sampler, other = Sampler(**SETTINGS), torch.cuda.Stream()
    sampler(x[:3], u[:3])
    zeros = [torch.zeros(n, device="cuda") for n in (9, 256, 700, 1024) for _ in range(20)]
    torch.cuda.synchronize()
    del zeros                                   # memory that a fill would find holds zeros
    _sleep()
    sampler(x, u)
    with torch.cuda.stream(other):
        got = sampler(x, u)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_settings_that_a_sampler_replaces_stay_while_another_stream_reads_them():
    from insitu_b200.sampling import Sampler
    x, u = inputs(700, 500, seed=2)
    want = _drawn(SETTINGS, x[:9], u[:9])
    sampler, other = Sampler(**SETTINGS), torch.cuda.Stream()
    sampler(x[:9], u[:9])
    torch.cuda.synchronize()
    with torch.cuda.stream(other):
        _sleep()
        got = sampler(x[:9], u[:9])
    sampler(x, u)                               # more rows than any call before: new tensors
    for n in (9, 256):
        zeros = [torch.zeros(n, device="cuda") for _ in range(200)]
        zeros += [torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(200)]
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_settings_given_on_the_device_are_ready_on_every_stream():
    from insitu_b200.sampling import Sampler
    x, u = inputs(700, 500, seed=3)
    want = _drawn(SETTINGS, x, u)
    columns = {k: torch.full((700,), v, dtype=torch.float64 if isinstance(v, float) else torch.int64, device="cuda")
               for k, v in SETTINGS.items()}
    torch.cuda.synchronize()
    _sleep()
    sampler, other = Sampler(**columns), torch.cuda.Stream()
    with torch.cuda.stream(other):
        got = sampler(x, u)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
