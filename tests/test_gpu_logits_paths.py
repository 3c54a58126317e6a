"""Operators on rows of logits where their kernels take paths that small tables do not reach: many equal
logits in one CTA's slice, long rows on one CTA, rows past a cluster's first, records and outcomes at the
edges of their definitions.  Tolerances are those of test_gpu_logits.py unless a test derives its own."""
import numpy as np
import pytest

import logits_ref as ref
from test_gpu_logits import DT, check_sample, host, table, tdt

pytestmark = pytest.mark.gpu


def uniform(rows, seed):
    import torch

    return torch.rand(rows, generator=torch.Generator().manual_seed(seed)).cuda()


# ---- sampling ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("rows,vocab", [(100, 262144), (150, 131072), (150, 131073), (40, 524288), (20, 1 << 20)])
def test_top_p_of_a_row_half_of_which_is_tied_at_the_maximum(ctx, rows, vocab):
    """The tied tokens of one CTA's slice weigh 2^47 units and more: no counter of theirs may wrap, and the
    first tenth of the whole is made of the lowest ids alone."""
    import torch

    z = torch.cat([torch.full((vocab // 2,), 1.5), torch.linspace(1.28, 1.48, vocab - vocab // 2)]).cuda()
    u = uniform(rows, vocab)
    out = ctx.sample_tokens(z.expand(rows, vocab), u, top_p=0.1)
    kept = ref.sample_weights(host(z), 1.0, 0, 0.1, 0.0)
    n = int((kept > 0).sum())
    assert (kept[:n] > 0).all() and n < vocab // 8
    assert np.array_equal(host(out["tokens"]), np.floor(host(u) * (n * ref.GRID)) // ref.GRID)
    assert np.abs(host(out["logprobs"]) + np.log(n)).max() <= 2e-6 * (1 + np.log(n))


@pytest.mark.parametrize("rows,vocab", [(150, 131072), (100, 262144)])
def test_top_p_of_a_row_of_equal_logits(ctx, rows, vocab):
    import torch

    z = torch.full((1, vocab), -2.0, device="cuda").bfloat16()
    u = uniform(rows, 1)
    got = host(ctx.sample_tokens(z.expand(rows, vocab), u, top_p=0.5)["tokens"])
    assert np.array_equal(got, np.floor(host(u) * (vocab // 2 * ref.GRID)) // ref.GRID)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab", [(300, 151936), (150, 262147)])
def test_top_p_of_long_rows_with_many_rows(ctx, rows, vocab, dtype):
    """One CTA a row, at vocabularies past 131072: a few distinct rows, each many times."""
    z = table(3, vocab, dtype, 31, spread=2.0)
    many = z.repeat(rows // 3, 1)
    u = uniform(rows, 3)
    out = ctx.sample_tokens(many, u, top_p=0.9)
    check_sample(ctx, many[:3], u[:3].contiguous(), p=0.9)
    kept = [ref.sample_weights(host(z)[r], 1.0, 0, 0.9, 0.0) for r in range(3)]
    tok, lp = host(out["tokens"]), host(out["logprobs"])
    for r in range(rows):
        w = kept[r % 3]
        W, c = w.sum(), np.cumsum(w)
        # (a token at the cut may be kept or not: moved limits as in check_sample)
        goal, slack, j = np.floor(host(u)[r] * W), 3e-6 * W + len(w), tok[r]
        assert c[j] - w[j] <= goal + slack and goal - slack < c[j], r
        zr = host(z)[r % 3]
        want = zr[j] - zr.max() - np.log(W / ref.GRID)
        assert abs(lp[r] - want) <= 4e-6 * (1 + abs(want)), r
