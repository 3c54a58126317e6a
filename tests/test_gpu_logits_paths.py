"""Operators on rows of logits where their kernels take paths that small tables do not reach: many equal
logits in one CTA's slice, long rows on one CTA, rows past a cluster's first, records and outcomes at the
edges of their definitions.  Tolerances are those of test_gpu_logits.py unless a test derives its own."""
import numpy as np
import pytest

import logits_ref as ref
from test_gpu_logits import DT, EPS, TINY, check_sample, host, record, table, tdt

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


# ---- distillation ---------------------------------------------------------------------------------


def check_rows(ctx, z, ids, t, lse, T, dtype, weight=None, rows=None):
    """Loss, gradient from the stats, and step.  An element's gradient w / T (P q - p) carries 4e-6 of q and p as in
    test_gpu_logits.py and the error of P, 2^-24 times 4 units of a power and the additions of a tree: 5e-6 in all."""
    import torch

    if weight is None:
        weight = torch.linspace(0.5, 1.5, z.shape[0], device="cuda")
    a = ctx.distill_loss(z, ids, t, teacher_lse=lse, temperature=T)
    g = ctx.distill_grad(z, ids, t, a["stats"], weight, teacher_lse=lse, temperature=T)
    b = ctx.distill_step(z, ids, t, weight, teacher_lse=lse, temperature=T)
    for r in range(z.shape[0]) if rows is None else rows:
        zh, ih, w = host(z[r]), host(ids[r]), float(weight[r])
        loss, _, grad, mag = ref.distill(zh, ih, host(t[r]), None if lse is None else float(lse[r]), T, w)
        q = np.exp(zh / T - ref.logsumexp(zh / T))
        tol = w / T * 5e-6 * q + 5e-6 * np.abs(grad) + EPS[dtype] * np.abs(grad) + TINY[dtype]
        have = ih[ih >= 0]
        tol[have] += 5e-6 * np.abs(w / T * q[have] - grad[have])  # of p
        for got, what in ((g, "grad"), (b["grad"], "step")):
            d = np.abs(host(got[r]) - grad)
            assert (d <= tol).all(), (what, r, int(np.argmax(d - tol)), float((d - tol).max()))
        if w != 0:
            for got, what in ((a, "loss"), (b, "step")):
                assert abs(float(got["loss"][r]) - loss) <= 4e-6 * mag + 1e-6, (what, r, float(got["loss"][r]), loss)
        else:
            assert float(b["loss"][r]) == 0.0 and (host(b["grad"][r]) == 0).all()
    return a, g, b


WIDE = {"f32": 240000, "f16": 470000, "bf16": 470001}  # longer than a cluster's stages


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("size", ["small", "wide"])
@pytest.mark.parametrize("k", [9, 200])
def test_distill_rows_whose_entries_are_no_distribution(ctx, size, dtype, k):
    """Closed rows without an entry (or none above -inf) have neither loss nor gradient; where the outcome outside
    the record is missing the gradient is P q - p."""
    import torch

    V = 1003 if size == "small" else WIDE[dtype]
    T = 1.25
    z = table(4, V, dtype, 41, spread=1.5)
    ids, t, lse = record(z, k, T, 3, dtype, True)
    ids[1] = -1
    t[2] = -float("inf")
    a, g, b = check_rows(ctx, z, ids, t, None, T, dtype)
    for r in (1, 2):
        assert float(a["loss"][r]) == 0.0 and (host(g[r]) == 0).all() and (host(b["grad"][r]) == 0).all()
    # a masked vocabulary: nothing outside the entries; the recorded p sum to 0.7
    ids, t, _ = record(z, k, T, 3, dtype, False)
    lse = (torch.logsumexp(t.double() / T, 1) - np.log(0.7)).float()
    out = torch.ones(4, V, dtype=torch.bool, device="cuda")
    out.scatter_(1, ids.long(), False)
    z = z.masked_fill(out, -float("inf"))
    a, g, b = check_rows(ctx, z, ids, t, lse, T, dtype)
    assert (a["stats"][:, 1] == 1).all() and (b["stats"][:, 1] == 1).all()
    w = host(torch.linspace(0.5, 1.5, 4))
    for got in (g, b["grad"]):
        assert np.abs(host(got).sum(1)).max() <= (w / T * (5e-6 + 2 * EPS[dtype])).max() + V * TINY[dtype]


@pytest.mark.parametrize("dtype", DT)
def test_distill_whole_vocabulary_of_a_part_of_the_teacher(ctx, dtype):
    import torch

    T = 0.8
    z = table(3, 301, dtype, 2)
    ids, t, _ = record(z, 301, T, 2, dtype, False)
    lse = (torch.logsumexp(t.double() / T, 1) - np.log(0.4)).float()
    check_rows(ctx, z, ids, t, lse, T, dtype)


def far_outside(dtype, V, T, gap, spread=1.0):
    """Rows whose logits outside the record lie `gap` (in units of T) below those in it, with a teacher that leaves 0.2
    outside."""
    import torch

    z = table(3, V, dtype, 51, spread=spread)
    ids, t, _ = record(z, 12, T, 3, dtype, False)
    lse = (torch.logsumexp(t.double() / T, 1) - np.log(0.8)).float()
    out = torch.ones_like(z, dtype=torch.bool)
    out.scatter_(1, ids.long(), False)
    z = torch.where(out, (z.float() - gap * T).to(z.dtype), z)
    return z, ids, t, lse, out


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T,gap", [(1.0, 70.0), (0.1, 75.0), (1.0, 120.0), (0.1, 120.0), (2.0, 3000.0), (1.0, 40000.0)])
@pytest.mark.parametrize("size", ["small", "wide"])
def test_distill_other_tokens_far_below_the_entries(ctx, dtype, T, gap, size):
    """The other-token outcome counts however small the student's probability of it is: the loss has p_r log q_r.
    z / T of the outside logits is a rounded number of the size of the gap: 2^-23 of it in the exponent's argument."""
    import torch

    V = 1003 if size == "small" else WIDE[dtype]
    z, ids, t, lse, out = far_outside(dtype, V, T, gap)
    w = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    a = ctx.distill_loss(z, ids, t, teacher_lse=lse, temperature=T)
    b = ctx.distill_step(z, ids, t, w, teacher_lse=lse, temperature=T)
    g = ctx.distill_grad(z, ids, t, a["stats"], w, teacher_lse=lse, temperature=T)
    for r in range(3):
        zh, ih = host(z[r]), host(ids[r])
        # (the restatement's q_r underflows too at a gap of thousands: the loss by its logarithm); the temperature is the
        # 32-bit number that the call takes
        x = zh / float(np.float32(T))
        L, o = ref.logsumexp(x), host(out[r])
        logp = host(t[r]) / float(np.float32(T)) - float(lse[r])
        p, lq_r = np.exp(logp), ref.logsumexp(x[o]) - L
        p_r = 1.0 - p.sum()
        terms = np.append(p * (logp - x[ih] + L), p_r * (np.log(p_r) - lq_r))
        loss, mag = terms.sum(), np.abs(terms).sum()
        wr = float(w[r])
        q = np.exp(x - L)
        # q_j / q_r (p(S) - q(S)), with powers of two below 2^-126 of the largest there 0
        e = np.where(o & ((x - x[o].max()) / np.log(2.0) >= -126), np.exp(np.where(o, x, -np.inf) - ref.logsumexp(x[o])), 0.0)
        grad = e * (p.sum() - q[ih].sum()) * wr / T
        grad[ih] = (q[ih] - p) * wr / T
        tol = 1e-5 * np.abs(grad) + EPS[dtype] * np.abs(grad) + TINY[dtype] + 1e-38
        tol[ih] += 5e-6 * wr / T * (q[ih] + p)
        for got in (a, b):
            assert abs(float(got["loss"][r]) - loss) <= 4e-6 * mag + 1e-6, (r, float(got["loss"][r]), loss)
        d = np.abs(host(b["grad"][r]) - grad)
        assert (d <= tol).all(), (r, int(np.argmax(d - tol)), float(d.max()))
        if lq_r > -86:  # the factor of q_j and its stats are within the type's range
            # (there it is the product q_j factor whose power of two is 0 below 2^-126)
            rel = 2e-5 + 3 * 2.0 ** -23 * abs(lq_r)
            want = np.where(o & (np.abs(grad) < 2.0 ** -126 * wr / T), 0.0, grad)
            d = np.abs(host(g[r]) - want)
            assert (d <= tol + rel * np.abs(want)).all(), (r, float(d.max()))
        assert np.isfinite(host(g[r])).all()


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("T", [1.0, 0.0625, 4.0])
@pytest.mark.parametrize("offset", [0.0, 1e3, -1e3, 1e4, -1e4, 3e6])
def test_gradient_from_saved_stats_at_any_size_of_the_logits(ctx, offset, T, tail):
    """The gradient from six stats is the step's.  An exponent e = (z - m) log2(e) / T carries three roundings, 3 * 2^-24 of
    its size (times ln 2) in the power; with 4e-6 of q and p as elsewhere, and 0 for a power below 2^-126."""
    import torch

    V = 2003
    z = (table(4, V, "f32", 61, spread=1.0).double() + offset).float()
    ids, t, lse = record(z - offset, 17, T, 3, "f32", tail)
    w = torch.tensor([1.0, 0.5, 0.0, 2.0], device="cuda")
    a = ctx.distill_loss(z, ids, t, teacher_lse=lse, temperature=T, full_stats=True)
    two = ctx.distill_loss(z, ids, t, teacher_lse=lse, temperature=T)
    assert a["stats"].shape == (4, 6) and torch.equal(a["stats"][:, :2], two["stats"]) and torch.equal(a["loss"], two["loss"])
    g = ctx.distill_grad(z, ids, t, a["stats"], w, teacher_lse=lse, temperature=T)
    b = ctx.distill_step(z, ids, t, w, teacher_lse=lse, temperature=T)
    for r in range(4):
        zh, ih, wr = host(z[r]), host(ids[r]), float(w[r])
        _, (L, off), grad, _ = ref.distill(zh, ih, host(t[r]), None if lse is None else float(lse[r]), T, wr)
        q = np.exp(zh / T - L)
        q_out = 1.0 - q[ih].sum()
        tol = (wr / T * q + np.abs(grad)) * (5e-6 + 3 * 2.0 ** -24 * (zh.max() - zh) / T) + 2.0 ** -125 * wr / T
        tol += wr / T * q * (2e-6 / q_out if tail else 0.0)
        tol[ih] += 5e-6 * np.abs(wr / T * q[ih] - grad[ih])
        for got, what in ((g, "grad"), (b["grad"], "step")):
            d = np.abs(host(got[r]) - grad)
            assert (d <= tol).all(), (what, r, int(np.argmax(d - tol)), float((d - tol).max()))


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("T", [1.0, 0.5, 2.0])
def test_gradient_of_a_row_of_the_lowest_value(ctx, dtype, T):
    """Masks of the type's lowest value that leave nothing: a uniform student."""
    import torch

    V = 1000
    z = torch.full((2, V), torch.finfo(tdt(dtype)).min, device="cuda", dtype=tdt(dtype))
    ids, t, lse = record(table(2, V, dtype, 5), 10, T, 3, dtype, False)
    w = torch.ones(2, device="cuda")
    a = ctx.distill_loss(z, ids, t, temperature=T, full_stats=True)
    g = ctx.distill_grad(z, ids, t, a["stats"], w, temperature=T)
    b = ctx.distill_step(z, ids, t, w, temperature=T)
    for r in range(2):
        th = host(t[r]) / T
        want = np.full(V, 1.0 / V / T)
        want[host(ids[r])] -= np.exp(th - ref.logsumexp(th)) / T
        tol = 5e-6 / T * (1.0 / V + np.abs(want)) + EPS[dtype] * np.abs(want) + TINY[dtype]
        for got in (g, b["grad"]):
            assert (np.abs(host(got[r]) - want) <= tol).all()


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("gap", [70.0, 120.0, 3000.0])
@pytest.mark.parametrize("size", ["small", "wide"])
def test_gradient_from_saved_stats_far_outside(ctx, dtype, gap, size):
    """The student's probability outside the record is past the type's range, the gradient there is not."""
    import torch

    z, ids, t, lse, out = far_outside(dtype, 1003 if size == "small" else WIDE[dtype], 1.0, gap)
    w = torch.tensor([1.0, 0.5, 2.0], device="cuda")
    a = ctx.distill_loss(z, ids, t, teacher_lse=lse, full_stats=True)
    g = host(ctx.distill_grad(z, ids, t, a["stats"], w, teacher_lse=lse))
    b = host(ctx.distill_step(z, ids, t, w, teacher_lse=lse)["grad"])
    assert np.isfinite(g).all() and np.abs(b).max() > 0.01
    assert (np.abs(g - b) <= 1e-6 * np.abs(b) + 2 * EPS[dtype] * np.abs(b) + TINY[dtype] + 2.0 ** -120).all()


def test_autograd_at_large_logits(ctx):
    """wb.distill_loss's gradient is the step's, whatever constant the rows carry."""
    import torch

    import winrapids_b200 as wb

    z = table(4, 999, "f32", 2)
    rec = wb.top_logits(table(4, 999, "f32", 1), 25)
    w = torch.linspace(0.5, 2.0, 4, device="cuda")
    for c in (0.0, 8192.0):
        x = (z + c).requires_grad_(True)
        (wb.distill_loss(x, rec) * w).sum().backward()
        step = ctx.distill_step(x.detach(), rec.ids, rec.values, w, teacher_lse=rec.lse)["grad"]
        scale = float(step.abs().max())
        assert float((x.grad - step).abs().max()) <= 2e-6 * scale
        assert float(x.grad.sum(1).abs().max()) <= 2e-5 * scale


def test_stats_columns_are_two_or_six(ctx):
    import torch

    import winrapids_b200 as wb

    z = table(2, 100, "f32", 1)
    ids, t, lse = record(z, 3, 1.0, 1, "f32", False)
    w = torch.ones(2, device="cuda")
    for cols in (1, 3, 4, 5, 7):
        with pytest.raises(wb.InvalidArgument):
            ctx.distill_grad(z, ids, t, torch.zeros(2, cols, device="cuda"), w)
    with pytest.raises(wb.InvalidArgument):
        ctx.distill_loss(z, ids, t, full_stats=True, out={"stats": torch.zeros(2, 2, device="cuda")})
    x, teacher = ctx._logits(z), ctx._teacher(ctx._logits(z), ids, t, None, 1.0, 4)
    loss = torch.zeros(2, device="cuda")
    assert ctx._L.tbgb_distill_loss(ctx._h, x, teacher, loss.data_ptr(), loss.data_ptr(), None) == 7


# ---- host threads ---------------------------------------------------------------------------------


def test_threads_with_tables_of_different_sizes():
    """Contexts are independent: two host threads launch the same kernels with different amounts of shared memory."""
    import threading

    import torch

    import winrapids_b200 as wb

    R = 300
    failed = []

    def work(vocab, k):
        c = wb.Context(0)
        try:
            z = torch.zeros(R, vocab, device="cuda")
            ids = torch.arange(8, dtype=torch.int32, device="cuda").repeat(R, 1)
            t, w, u = torch.zeros(R, 8, device="cuda"), torch.ones(R, device="cuda"), torch.zeros(R, device="cuda")
            out = {"loss": torch.empty(R, device="cuda"), "stats": torch.empty(R, 2, device="cuda")}
            grad = torch.empty_like(z)
            for i in range(400):
                c.distill_step(z, ids, t, w, grad=grad, out=out, sync=i % 100 == 99)
                c.sample_tokens(z, u, top_k=k, sync=False)
                c.top_logits(z, k, sync=False)
            c.sync()
        except Exception as e:  # noqa: BLE001
            failed.append(repr(e))
        finally:
            c.close()

    threads = [threading.Thread(target=work, args=a) for a in ((7000, 900), (8600, 600), (7800, 1000))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


# ---- many rows, long rows --------------------------------------------------------------------------


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("rows,vocab,dtype,k", [(2000, 4099, "f32", 20), (2000, 4099, "bf16", 20), (600, 50001, "f16", 64),
                                                (600, 50001, "f32", 100), (700, 4099, "bf16", 200)])
def test_distill_more_rows_than_clusters(ctx, rows, vocab, dtype, k, tail):
    """Each cluster takes several rows: every stage, barrier phase and part is used again, padding rows (which are
    not counted there) lie between others."""
    import torch

    z = table(rows, vocab, dtype, rows, spread=1.5)
    ids, t, lse = record(z, k, 1.0, 3, dtype, tail)
    weight = torch.rand(rows, generator=torch.Generator().manual_seed(5)) + 0.5
    weight[torch.rand(rows, generator=torch.Generator().manual_seed(6)) < 0.2] = 0.0
    weight[-1] = 0.0
    weight = weight.cuda()
    a, g, b = check_rows(ctx, z, ids, t, lse, 1.0, dtype, weight=weight)
    in_place = z.clone()
    c = ctx.distill_step(in_place, ids, t, weight, teacher_lse=lse, grad=in_place)
    assert torch.equal(in_place, b["grad"]) and torch.equal(c["loss"], b["loss"])


@pytest.mark.parametrize("dtype", DT)
def test_top_logits_of_long_rows_on_one_cta(ctx, dtype):
    from test_gpu_logits import check_top

    import torch

    z = table(80, 50001, dtype, 71)
    for k in (1, 64, 1000):
        check_top(ctx, z, k)
    bits = np.random.default_rng(0).random((80, 50001)) < 0.3
    words = torch.from_numpy(np.stack([ref.pack_mask(b) for b in bits])).cuda()
    check_top(ctx, z, 20, T=0.7, mask=words, bits=bits)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("setting", [dict(), dict(mp=0.05), dict(p=0.9), dict(k=40), dict(k=1000, p=0.95), dict(T=0.0)],
                         ids=str)
def test_sampling_of_long_rows_on_one_cta(ctx, dtype, setting):
    z = table(150, 50001, dtype, 81, spread=2.0)
    check_sample(ctx, z, uniform(150, 4), **setting)


@pytest.mark.parametrize("dtype", DT)
def test_sampling_of_long_masked_rows_on_one_cta(ctx, dtype):
    import torch

    z = table(150, 20001, dtype, 82, spread=2.0)
    bits = np.random.default_rng(1).random((150, 20001)) < 0.1
    words = torch.from_numpy(np.stack([ref.pack_mask(b) for b in bits])).cuda()
    for s in (dict(), dict(p=0.9), dict(k=50)):
        check_sample(ctx, z, uniform(150, 5), mask=words, bits=bits, **s)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab", [(4, 70001), (150, 9001)])
def test_k_past_the_lists_with_top_p(ctx, rows, vocab, dtype):
    z = table(rows, vocab, dtype, 83)
    for s in (dict(k=3000, p=0.8), dict(k=1025, p=0.3), dict(k=vocab, p=0.7), dict(k=vocab - 1, mp=0.01)):
        check_sample(ctx, z, uniform(rows, 6), **s)


@pytest.mark.parametrize("rows", [2, 150])
def test_top_p_whose_end_lies_among_thousands_of_equal_logits(ctx, rows):
    """More equal logits at the end of the prefix than the quick way lists."""
    import torch

    z = (table(1, 60000, "f32", 84, spread=2.0) * 2).round().div(2).bfloat16()
    for p in (0.5, 0.9, 0.99):
        check_sample(ctx, z.expand(rows, 60000), uniform(rows, 7), p=p)


@pytest.mark.parametrize("dtype", DT)
def test_few_rows_with_a_k_of_their_own(ctx, dtype):
    """Lists of up to 1024 on several CTAs a row, as many as the lists hold."""
    import torch

    z = table(6, 70001, dtype, 85)
    k = torch.tensor([1024, 1000, 700, 300, 1, 0], dtype=torch.int32, device="cuda")
    p = torch.tensor([1.0, 0.5, 0.9, 1.0, 0.3, 0.9], device="cuda")
    check_sample(ctx, z, uniform(6, 8), k=k, p=p)
