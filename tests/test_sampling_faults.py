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
