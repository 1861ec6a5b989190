"""How near l2b_sample_device is to its definition where it is not equal to it: masses are whole multiples of 2^-44 of the largest weight."""
import numpy as np
import pytest

from test_gpu_sampling import L, sample  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("vocab", [5000, 393216])
@pytest.mark.parametrize("units", [0.3, 0.49, 0.51, 1.4, 20.3])
@pytest.mark.parametrize("cuts", [dict(), dict(top_p=1 - 2.0 ** -24), dict(top_k=4000)])
def test_a_flat_tail_around_the_unit(L, vocab, units, cuts):  # noqa: F811
    """One likely token among others of `units` units each.  A weight is off by half a unit at most, so a mass by vocab * 2^-45 of the largest: the token is one that
    the definition gives for a random number no further off than twice that (the mass before it and the whole); weights below half a unit are never drawn."""
    import torch
    at = vocab // 3
    x = torch.full((1, vocab), float(np.float32(np.log(units * 2.0 ** -44))), device="cuda")
    x[0, at] = 0.0
    w = np.exp(x[0].double().cpu().numpy())
    slack = 2 * vocab * 2.0 ** -45
    order = np.argsort(-w, kind="stable")
    if "top_k" in cuts:
        order = order[:cuts["top_k"]]
    if "top_p" in cuts:  # (the border, too, may be off by what masses are off)
        before = np.concatenate(([0.0], np.cumsum(w[order])[:-1]))
        order = order[before < cuts["top_p"] * w.sum()]
        slack *= 2
    keep = np.sort(order)
    run = np.cumsum(w[keep])
    tail = run[-1] - 1.0
    for u in [0.0, 0.25, 0.999] + [tail / run[-1] * f for f in (0.1, 0.3)] + [1 - tail / run[-1] * f for f in (0.1, 0.4, 0.6)] + [1 - 2.0 ** -53]:
        (token,), (prob,) = sample(L, x, temperature=1.0, uniform=u, **cuts)
        i = min(int(np.searchsorted(keep, token)), len(keep) - 1)
        assert keep[i] == token or "top_p" in cuts and (token - keep[i]) * w[token] <= slack
        before = run[i] - w[token]
        assert before - slack <= u * run[-1] <= run[i] + slack, (u, token, before, run[i])
        assert units >= 0.5 or token == at
        assert abs(prob - w[token] / run[-1]) <= 2.0 ** -24 * prob + slack
