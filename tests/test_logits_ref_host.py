"""The 64-bit restatement's distillation gradient (tests/logits_ref.py) against central differences of its own
loss, where the teacher's entries are not a whole distribution and no other outcome makes up for it.  A difference's
own error is h^2 / 6 of a third derivative of at most 1 / T^3, plus 2^-52 / h of the loss (about 10)."""
import numpy as np
import pytest

import logits_ref as ref

H = 1e-4
INF = float("inf")


def differences(z, ids, t, lse, T):
    d = np.zeros(len(z))
    for j in np.flatnonzero(np.isfinite(z)):
        up, dn = z.copy(), z.copy()
        up[j] += H
        dn[j] -= H
        d[j] = (ref.distill(up, ids, t, lse, T)[0] - ref.distill(dn, ids, t, lse, T)[0]) / (2 * H)
    return d


def cases():
    rng = np.random.default_rng(0)
    z = rng.normal(size=23)
    ids = np.arange(0, 23, 3)
    t = rng.normal(size=len(ids))
    masked = np.full(23, -INF)
    masked[ids] = z[ids]
    every = np.arange(23)
    te = rng.normal(size=23)
    for T in (1.0, 1.7):
        full = ref.logsumexp(t / T)
        yield "closed", z, ids, t, None, T
        yield "tail", z, ids, t, full - np.log(0.7), T
        yield "no entries", z, np.full(4, -1), np.zeros(4), None, T
        yield "no entries with a tail", z, np.full(4, -1), np.zeros(4), 0.3, T
        yield "entries of -inf", z, ids, np.full(len(ids), -INF), None, T
        yield "nothing outside", masked, ids, t, full - np.log(0.7), T
        yield "whole vocabulary", z, every, te, ref.logsumexp(te / T) - np.log(0.7), T
        yield "far outside", np.where(np.isfinite(masked), z, z - 200.0), ids, t, full - np.log(0.8), T


@pytest.mark.parametrize("case", list(cases()), ids=lambda c: f"{c[0]} T={c[-1]}")
def test_gradient_is_the_loss_s(case):
    _, z, ids, t, lse, T = case
    loss, _, g, mag = ref.distill(z, ids, t, lse, T)
    assert np.isfinite(loss)
    assert np.abs(g - differences(z, ids, t, lse, T)).max() <= H * H / 6 / T ** 3 + 2.0 ** -52 / H * (10 + mag)
    assert abs(g.sum()) <= 1e-12 * len(z)  # a loss does not change with a constant added to a row
