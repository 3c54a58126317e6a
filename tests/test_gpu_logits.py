"""The operators on rows of logits (tbgb_top_logits, tbgb_distill_*, tbgb_sample_tokens) against a
64-bit restatement (tests/logits_ref.py).

Tolerances.  Values, ids and tokens are exact.  A log-sum-exp in 32 bits: the exponent's rounding
(2^-24 of |d| log2 e, weighted by e^d, at most about 2^-24), 2 units of the power of two and the
additions (64 in a thread, then a tree) stay under 16 * 2^-24 ~ 1e-6, and the result is rounded at its
own size: 1e-6 + 2^-23 |lse|, doubled.  The loss is a sum of terms p (log p - log q) whose logarithms
carry that error and p 4 units: 4e-6 of the terms' magnitude, plus 1e-6.  A gradient element is
w / T (q - p): 4e-6 of q + p (12 units of the power of two's argument at |d| <= 16, then a few
products), then rounded to its type (2^-8 bf16, 2^-11 f16 of its size, and f16's smallest step);
the factor outside the entries, a quotient of differences, carries 1e-6 / q_out absolutely.
A token is the one whose running sum covers floor(u W); the kernel's and the restatement's powers of
two may differ by 2 units each, so running sums by 3e-7 W + 1 unit per token at most: a token
has to cover the goal within that, for the cuts' limits (top-p, min-p) as they are or moved by 2e-6 of
themselves either way."""
import numpy as np
import pytest

import logits_ref as ref

pytestmark = pytest.mark.gpu

DT = ["f32", "f16", "bf16"]
EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}
TINY = {"f32": 0.0, "f16": 2.0 ** -24, "bf16": 0.0}


def tdt(name):
    import torch

    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[name]


def table(rows, vocab, dtype, seed, spread=3.0, stride=None, offset=0):
    """Logits [rows, vocab] on the device inside a larger buffer (row stride, first element)."""
    import torch

    g = torch.Generator().manual_seed(seed)
    z = torch.randn(rows, vocab, generator=g) * spread
    stride = stride or vocab
    buf = torch.full((offset + max(rows, 1) * stride + 16,), 77.0).to(tdt(dtype))
    v = buf[offset:offset + rows * stride].view(rows, stride)[:, :vocab]
    v.copy_(z.to(tdt(dtype)))
    d = buf.cuda()
    return d[offset:offset + rows * stride].view(rows, stride)[:, :vocab]


def host(t):
    return t.detach().double().cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


# sizes around the vectors' (4 or 8 elements), the warps' and the CTAs' edges; rows that start
# anywhere; one row per cluster and many
SHAPES = [(1, 1, 1, 0), (3, 2, 5, 1), (2, 7, 7, 0), (2, 8, 9, 3), (5, 31, 31, 0), (3, 257, 260, 2), (2, 1000, 1001, 1),
          (4, 4099, 4099, 0), (2, 32768, 32768, 0), (1, 50001, 50001, 5), (3, 65537, 65537, 0), (2, 150001, 150001, 0)]
BIG = [(1, 1 << 19), (2, (1 << 21) + 3)]  # past what a cluster holds in registers for some or all types


# ---- top_logits ---------------------------------------------------------------------------------


def check_top(ctx, z, k, T=1.0, mask=None, bits=None, **kw):
    out = ctx.top_logits(z, k, temperature=T, mask=mask, **kw)
    zh, v, i, l = host(z), host(out["values"]), host(out["ids"]), host(out["lse"])
    for r in range(zh.shape[0]):
        b = None if bits is None else bits[r if bits.ndim == 2 else slice(None)]
        wv, wi, wl = ref.top(zh[r], k, T, b)
        assert np.array_equal(i[r], wi), r
        assert np.array_equal(v[r], wv), r
        if np.isfinite(wl):
            assert abs(l[r] - wl) <= 2 * (1e-6 + 2.0 ** -23 * abs(wl)), (r, l[r], wl)
        else:
            assert l[r] == wl, r


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab,stride,offset", SHAPES)
def test_top_shapes(ctx, rows, vocab, stride, offset, dtype):
    z = table(rows, vocab, dtype, vocab + rows, stride=stride, offset=offset)
    for k in (1, 5, 64, 1000):
        check_top(ctx, z, k, T=2.0 if k == 5 else 1.0)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab", BIG)
def test_top_big(ctx, rows, vocab, dtype):
    check_top(ctx, table(rows, vocab, dtype, 5), 100)


@pytest.mark.parametrize("dtype", DT)
def test_top_ties_take_the_lowest_id(ctx, dtype):
    import torch

    z = torch.zeros(4, 40000, device="cuda").to(tdt(dtype))
    z[1, 100:39000] = 2.0
    z[2, ::3] = -0.0
    z[3] = (torch.arange(40000, device="cuda") % 7).to(tdt(dtype))
    for k in (1, 3, 1024):
        check_top(ctx, z, k)


@pytest.mark.parametrize("dtype", DT)
def test_top_special_values(ctx, dtype):
    import torch

    inf, nan = float("inf"), float("nan")
    low = torch.finfo(tdt(dtype)).min
    z = table(8, 5000, dtype, 3)
    z[0] = -inf
    z[1] = nan
    z[2, 5:] = -inf
    z[3, 7] = inf
    z[4, ::2] = nan
    z[5] = low
    z[6] = low
    z[6, 4321] = 1.0
    z[7, :4000] = -inf
    check_top(ctx, z, 16)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("vocab", [1, 63, 64, 65, 1000, 70001])
def test_top_masks(ctx, vocab, dtype):
    import torch

    rng = np.random.default_rng(vocab)
    z = table(6, vocab, dtype, 11, stride=vocab + 3, offset=1)
    bits = rng.random((6, vocab)) < np.array([0.5, 0.01, 1.0, 0.0, 0.5, 0.5])[:, None]
    bits[4, vocab // 2:] = False
    bits[5, :vocab // 2] = False
    words = torch.from_numpy(np.stack([ref.pack_mask(b) for b in bits])).cuda()
    check_top(ctx, z, 20, mask=words, bits=bits)
    check_top(ctx, z, 20, mask=words[0].contiguous(), bits=bits[0])


def test_top_into_given_outputs_and_without_lse(ctx):
    import torch

    z = table(3, 3001, "bf16", 1)
    out = {"values": torch.empty(3, 9, dtype=torch.bfloat16, device="cuda"),
           "ids": torch.empty(3, 9, dtype=torch.int32, device="cuda")}
    got = ctx.top_logits(z, 9, lse=False, out=out)
    assert got["ids"] is out["ids"] and "lse" not in got
    assert np.array_equal(host(got["ids"][2]), ref.top(host(z[2]), 9, 1.0)[1])


# ---- distillation ---------------------------------------------------------------------------------


def record(z, k, T, seed, dtype, tail, unused=0):
    """A teacher near the student: ids, its logits there, its log-sum-exp (or None)."""
    import torch

    g = torch.Generator().manual_seed(seed)
    rows, vocab = z.shape
    t = (z.float().cpu() + torch.randn(rows, vocab, generator=g)).to(tdt(dtype)).float()
    top, ids = torch.topk(t, min(k, vocab), dim=1)
    lse = torch.logsumexp(t.double() / T, 1).float() if tail else None
    mix = torch.randperm(ids.shape[1], generator=g)  # the order of the entries is free
    top, ids = top[:, mix].contiguous(), ids[:, mix].int().contiguous()
    if unused:
        ids[:, :unused] = -1
    return ids.cuda(), top.to(tdt(dtype)).cuda(), None if lse is None else lse.cuda()


def check_distill(ctx, z, ids, t, lse, T, dtype, weight=None, **kw):
    import torch

    rows, vocab = z.shape
    if weight is None:
        weight = torch.linspace(0.5, 1.5, rows, device="cuda")
    zh, ih, th, wh = host(z), host(ids), host(t), host(weight)
    lh = [None] * rows if lse is None else host(lse)
    a = ctx.distill_loss(z, ids, t, teacher_lse=lse, temperature=T)
    g = ctx.distill_grad(z, ids, t, a["stats"], weight, teacher_lse=lse, temperature=T)
    b = ctx.distill_step(z, ids, t, weight, teacher_lse=lse, temperature=T, **kw)
    for r in range(rows):
        loss, (L, off), grad, mag = ref.distill(zh[r], ih[r], th[r], lh[r], T, wh[r])
        q = np.exp(zh[r] / T - L)
        have = ih[r][ih[r] >= 0]
        p_at = np.abs(grad)
        q_out = max(1.0 - q[have].sum(), 1e-30)
        out_err = 2e-6 / q_out if lse is not None else 0.0
        assert abs(host(a["loss"])[r] - loss) <= 4e-6 * mag + 1e-6, (r, host(a["loss"])[r], loss)
        s = host(a["stats"])[r]
        assert abs(s[0] - L) <= 2 * (1e-6 + 2.0 ** -23 * abs(L))
        assert abs(s[1] - off) <= 4e-6 * abs(off) + out_err
        tol = wh[r] / T * (4e-6 * q + q * out_err) + 4e-6 * p_at + EPS[dtype] * np.abs(grad) + TINY[dtype] + 1e-30
        if have.size:
            tol[have] += 4e-6 * wh[r] / T * q[have]
        for got in (g, b["grad"]):
            d = np.abs(host(got)[r] - grad)
            assert (d <= tol).all(), (r, np.argmax(d - tol), d.max())
        if wh[r] != 0:
            assert host(b["loss"])[r] == host(a["loss"])[r]


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab,stride,offset", SHAPES)
def test_distill_shapes(ctx, rows, vocab, stride, offset, dtype, tail):
    z = table(rows, vocab, dtype, vocab, stride=stride, offset=offset, spread=1.5)
    for k, T in ((1, 1.0), (min(vocab, 20), 2.0), (min(vocab, 300), 0.7)):
        if tail and k == vocab:
            continue  # no token is left: test_distill_whole_vocabulary
        ids, t, lse = record(z, k, T, k, dtype, tail)
        check_distill(ctx, z, ids, t, lse, T, dtype)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab", BIG)
def test_distill_big(ctx, rows, vocab, dtype):
    z = table(rows, vocab, dtype, 9, spread=1.0)
    ids, t, lse = record(z, 64, 1.0, 3, dtype, True)
    check_distill(ctx, z, ids, t, lse, 1.0, dtype)


def test_distill_whole_vocabulary(ctx):
    """Every token is an entry: with a tail nothing is left outside, the same as closed."""
    z = table(3, 40, "f32", 2)
    ids, t, lse = record(z, 40, 1.0, 2, "f32", True)
    a = ctx.distill_loss(z, ids, t, teacher_lse=lse)
    b = ctx.distill_loss(z, ids, t)
    assert np.allclose(host(a["loss"]), host(b["loss"]), rtol=0, atol=4e-6)
    assert np.array_equal(host(a["stats"])[:, 1], np.ones(3))


@pytest.mark.parametrize("tail", [False, True])
def test_distill_unused_entries_and_padding(ctx, tail):
    import torch

    z = table(4, 3000, "bf16", 4, spread=1.5)
    ids, t, lse = record(z, 30, 1.0, 7, "bf16", tail, unused=7)
    ids[2] = -1
    t[:, 3] = float("nan")  # an unused entry's logit means nothing
    weight = torch.tensor([1.0, 0.0, 2.0, 0.5], device="cuda")
    check_distill(ctx, z, ids, t, lse, 1.0, "bf16", weight=weight)
    z2 = z.clone()
    z2[1] = float("nan")  # a padding row is not read
    b = ctx.distill_step(z2, ids, t, weight, teacher_lse=lse)
    assert host(b["loss"])[1] == 0 and (host(b["grad"])[1] == 0).all()
    assert host(b["loss"])[2] == 0


def test_distill_padding_of_rows_past_the_registers(ctx):
    import torch

    z = table(2, 1 << 20, "f32", 4, spread=1.0)
    ids, t, lse = record(z, 8, 1.0, 7, "f32", True)
    z[1] = float("nan")
    b = ctx.distill_step(z, ids, t, torch.tensor([1.0, 0.0], device="cuda"), teacher_lse=lse)
    assert host(b["loss"])[1] == 0 and (host(b["grad"])[1] == 0).all() and np.isfinite(host(b["grad"])[0]).all()
    assert np.array_equal(host(b["stats"])[1], [0.0, 1.0])


@pytest.mark.parametrize("dtype", DT)
def test_distill_special_values(ctx, dtype):
    import torch

    inf = float("inf")
    low = torch.finfo(tdt(dtype)).min
    z = table(6, 3000, dtype, 8, spread=1.0)
    ids, t, lse = record(z, 10, 1.0, 1, dtype, False)
    outside = [j for j in range(40) if j not in set(host(ids)[:, :].reshape(-1).tolist())]
    z[0, outside] = -inf           # a masked vocabulary
    z[1, outside] = low
    t[2, 0] = -inf                 # the teacher never says it
    t[3] = -inf                    # a teacher without any entry above -inf
    check_distill(ctx, z[:3], ids[:3], t[:3], None, 1.0, dtype)
    w = torch.ones(6, device="cuda")
    z[4, int(ids[4, 3])] = -inf    # the student never says what the teacher says
    z[5, 17] = float("nan")
    out = ctx.distill_step(z, ids, t, w)
    assert host(out["loss"])[3] == 0
    assert host(out["loss"])[4] == inf
    g4 = host(out["grad"])[4]
    assert np.isfinite(g4).all() and g4[int(ids[4, 3])] < 0
    assert np.isnan(host(out["loss"])[5]) and np.isnan(host(out["grad"])[5]).any()
    z[0] = -inf
    out = ctx.distill_step(z, ids, t, w)
    assert np.isnan(host(out["loss"])[0])
    z[0] = low  # uniform: nothing overflows
    out = ctx.distill_loss(z, ids, t)
    p = np.exp(host(t)[0] - ref.logsumexp(host(t)[0]))
    want = (p * np.log(p)).sum() + np.log(3000)
    assert abs(host(out["loss"])[0] - want) <= 1e-5


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("stride", [3000, 3001, 3008])
def test_distill_in_place_and_strided_gradient(ctx, dtype, stride):
    import torch

    z = table(5, 2999, dtype, 8, stride=stride, offset=3, spread=1.5)
    ids, t, lse = record(z, 33, 1.0, 1, dtype, True)
    w = torch.linspace(1, 2, 5, device="cuda")
    want = ctx.distill_step(z, ids, t, w, teacher_lse=lse)
    buf = torch.full((5, stride + 5), 3.0, device="cuda").to(tdt(dtype))
    got = ctx.distill_step(z, ids, t, w, teacher_lse=lse, grad=buf[:, 2:2 + 2999])
    assert torch.equal(got["grad"], want["grad"])
    assert (buf[:, :2] == 3).all() and (buf[:, 2 + 2999:] == 3).all()
    # a call's bits depend on where the rows start (it sets which thread adds what): the same layout again
    z2 = table(5, 2999, dtype, 8, stride=stride, offset=3, spread=1.5)
    got = ctx.distill_step(z2, ids, t, w, teacher_lse=lse, grad=z2)
    assert got["grad"] is z2 and torch.equal(z2, want["grad"])
    z3 = table(5, 2999, dtype, 8, stride=stride, offset=3, spread=1.5)
    g1 = ctx.distill_grad(z, ids, t, want["stats"], w, teacher_lse=lse)
    ctx.distill_grad(z3, ids, t, want["stats"], w, teacher_lse=lse, grad=z3)
    assert torch.equal(z3, g1)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_against_differences(ctx, tail):
    """Central differences of the 64-bit loss: their own error is h^2 / 6 times a third derivative of
    at most 1 / T^3, plus 2^-52 / h of the loss's terms (about 10)."""
    import torch

    T, h = 1.5, 1e-4
    z = table(2, 37, "f32", 21, spread=1.0)
    ids, t, lse = record(z, 6, T, 5, "f32", tail)
    g = host(ctx.distill_step(z, ids, t, torch.ones(2, device="cuda"), teacher_lse=lse, temperature=T)["grad"])
    for r in range(2):
        zh = host(z)[r]
        l = None if lse is None else float(host(lse)[r])
        for j in range(37):
            up, dn = zh.copy(), zh.copy()
            up[j] += h
            dn[j] -= h
            d = (ref.distill(up, host(ids)[r], host(t)[r], l, T)[0] - ref.distill(dn, host(ids)[r], host(t)[r], l, T)[0]) / (2 * h)
            assert abs(g[r, j] - d) <= 1e-8 + 1e-10 + 1e-5 * (abs(d) + 0.01), (r, j)


def test_distill_autograd(ctx):
    import torch

    import winrapids_b200 as wb

    teacher = table(6, 999, "bf16", 1)
    student = table(6, 999, "bf16", 2).contiguous().view(2, 3, 999).requires_grad_(True)
    rec = wb.top_logits(teacher.contiguous().view(2, 3, 999), 25, temperature=2.0)
    assert rec.ids.shape == (2, 3, 25) and rec.lse.shape == (2, 3)
    for r in (rec, rec.closed()):
        loss = wb.distill_loss(student, r)
        assert loss.shape == (2, 3)
        student.grad = None
        (loss * torch.arange(6, device="cuda").view(2, 3)).sum().backward()
        zh = host(student).reshape(6, 999)
        for i in range(6):
            l = None if r.lse is None else float(host(r.lse).reshape(-1)[i])
            want = ref.distill(zh[i], host(r.ids).reshape(6, -1)[i], host(r.values).reshape(6, -1)[i], l, 2.0, float(i))
            assert abs(host(loss).reshape(-1)[i] - want[0]) <= 4e-6 * want[3] + 1e-6
            got = host(student.grad).reshape(6, 999)[i]
            assert (np.abs(got - want[2]) <= 2.0 ** -8 * np.abs(want[2]) + 1e-5 * (np.abs(want[2]) + 1e-3)).all()


def test_distill_broadcast_student_row(ctx):
    """One row of logits read by every row: the rows' gradients are their own, autograd adds them."""
    import torch

    import winrapids_b200 as wb

    one = table(1, 515, "f32", 3).contiguous().requires_grad_(True)
    teacher = table(4, 515, "f32", 4)
    rec = wb.top_logits(teacher, 12)
    loss = wb.distill_loss(one.expand(4, 515), rec)
    loss.sum().backward()
    want = sum(ref.distill(host(one)[0], host(rec.ids)[i], host(rec.values)[i], float(host(rec.lse)[i]), 1.0)[2]
               for i in range(4))
    assert np.abs(host(one.grad)[0] - want).max() <= 4e-5


def test_distill_reports_bad_ids(ctx):
    import torch

    import winrapids_b200 as wb

    z = table(2, 100, "f32", 1)
    ids = torch.tensor([[1, 2], [3, 100]], dtype=torch.int32, device="cuda")
    t = torch.zeros(2, 2, device="cuda")
    with pytest.raises(wb.KeyOutOfRange):
        ctx.distill_loss(z, ids, t)
    ids[1, 1] = -2
    with pytest.raises(wb.KeyOutOfRange):
        ctx.distill_step(z, ids, t, torch.ones(2, device="cuda"))
    ids[1, 1] = 3
    with pytest.raises(wb.InvalidArgument):
        ctx.distill_loss(z, ids, t)
    ids[1, 1] = 4
    ctx.distill_loss(z, ids, t)


# ---- sampling ---------------------------------------------------------------------------------------


def check_sample(ctx, z, u, T=1.0, k=0, p=1.0, mp=0.0, mask=None, bits=None, **kw):
    import torch

    out = ctx.sample_tokens(z, u, temperature=T, top_k=k, top_p=p, min_p=mp, mask=mask, **kw)
    zh, uh = host(z), host(u)
    tok, lp = host(out["tokens"]), host(out["logprobs"])
    at = lambda v, r: float(host(v)[r]) if isinstance(v, torch.Tensor) else v  # noqa: E731
    for r in range(zh.shape[0]):
        b = None if bits is None else bits[r if bits.ndim == 2 else slice(None)]
        good = []
        for nudge in (0.0, -2e-6, 2e-6):
            kept = ref.sample_weights(zh[r], at(T, r), int(at(k, r)), at(p, r), at(mp, r), b, nudge)
            W, j = kept.sum(), tok[r]
            if W == 0:
                good.append(j == -1 and lp[r] == -np.inf)
                continue
            if not (0 <= j < len(kept) and kept[j] > 0):
                good.append(False)
                continue
            c = np.cumsum(kept)
            goal = min(np.floor(uh[r] * W), W - 1)
            slack = 3e-7 * W + len(kept)
            covers = c[j] - kept[j] <= goal + slack and goal - slack < c[j]
            if not at(T, r) > 0:
                want = 0.0
            else:
                m = ref.allowed_logits(zh[r], b).max()
                x = 0.0 if zh[r][j] == m else (zh[r][j] - m) / at(T, r)
                want = x - np.log(W / ref.GRID)
            good.append(covers and abs(lp[r] - want) <= 2e-6 * (1 + abs(want)))
            if good[-1]:
                break
        assert any(good), (r, tok[r], lp[r], good)


SETTINGS = [dict(), dict(T=0.7), dict(k=1), dict(k=40), dict(k=3000), dict(p=0.9), dict(p=0.5, T=1.5), dict(p=0.0),
            dict(mp=0.1), dict(k=50, p=0.9), dict(k=50, p=0.8, mp=0.02, T=0.6), dict(T=0.0), dict(mp=1.0)]


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab,stride,offset", SHAPES)
def test_sample_shapes(ctx, rows, vocab, stride, offset, dtype):
    import torch

    z = table(rows, vocab, dtype, vocab + 1, stride=stride, offset=offset)
    u = torch.rand(rows, generator=torch.Generator().manual_seed(vocab)).cuda()
    for s in SETTINGS:
        check_sample(ctx, z, u, **s)


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("rows,vocab", BIG)
def test_sample_big(ctx, rows, vocab, dtype):
    import torch

    z = table(rows, vocab, dtype, 2, spread=2.0)
    u = torch.tensor([0.3, 0.95], device="cuda")[:rows].contiguous()
    for s in (dict(), dict(k=50, p=0.9), dict(p=0.95), dict(k=100000), dict(mp=0.05)):
        check_sample(ctx, z, u, **s)


@pytest.mark.parametrize("dtype", DT)
def test_sample_many_rows_per_row_settings(ctx, dtype):
    import torch

    g = torch.Generator().manual_seed(6)
    R, V = 700, 2003
    z = table(R, V, dtype, 12)
    u = torch.rand(R, generator=g).cuda()
    T = (torch.rand(R, generator=g) * 2).cuda()
    T[::50] = 0.0
    k = torch.randint(0, 60, (R,), generator=g, dtype=torch.int32).cuda()
    p = (torch.rand(R, generator=g) * 1.2).cuda()
    mp = (torch.rand(R, generator=g) * 0.2 - 0.1).cuda()
    check_sample(ctx, z, u, T=T, k=k, p=p, mp=mp)


@pytest.mark.parametrize("dtype", DT)
def test_sample_ties_and_ends(ctx, dtype):
    """Equal logits: token floor(u n) of the first n kept; u = 0 the first, u -> 1 the last."""
    import torch

    V = 40000
    z = torch.full((5, V), 1.5, device="cuda").to(tdt(dtype))
    u = torch.tensor([0.0, 0.25, 0.5, 1 - 2.0 ** -24, 0.999], device="cuda")
    for s, n in ((dict(), V), (dict(k=1000), 1000), (dict(p=0.25), 10000), (dict(k=1000, p=0.5), 500), (dict(k=7), 7)):
        got = host(ctx.sample_tokens(z, u, top_k=s.get("k", 0), top_p=s.get("p", 1.0))["tokens"])
        want = np.floor(host(u) * n * ref.GRID) // ref.GRID
        assert np.array_equal(got, want), s
    z[:, 100:] = -0.0
    z[:, :100] = 0.0
    got = host(ctx.sample_tokens(z, u, top_k=200)["tokens"])
    assert np.array_equal(got, np.floor(host(u) * 200))


@pytest.mark.parametrize("dtype", DT)
def test_sample_special_values(ctx, dtype):
    import torch

    inf, nan = float("inf"), float("nan")
    low = torch.finfo(tdt(dtype)).min
    z = table(9, 5000, dtype, 5)
    u = torch.full((9,), 0.6, device="cuda")
    z[0] = -inf
    z[1] = nan
    z[2] = -inf
    z[2, 4999] = -3.0
    z[3, 7] = inf
    z[3, 4000] = inf
    z[4, ::2] = nan
    z[5] = low
    z[6] = low
    z[6, 4321] = 1.0
    z[7, :4000] = -inf
    for s in SETTINGS + [dict(T=inf), dict(T=1e-30), dict(T=nan), dict(T=-1.0)]:
        check_sample(ctx, z, u, **s)
    assert host(ctx.sample_tokens(z, u)["tokens"])[3] == 4000


@pytest.mark.parametrize("dtype", DT)
@pytest.mark.parametrize("vocab", [1, 64, 65, 1000, 70001])
def test_sample_masks(ctx, vocab, dtype):
    import torch

    rng = np.random.default_rng(vocab)
    z = table(6, vocab, dtype, 13, stride=vocab + 1, offset=1)
    u = torch.rand(6, generator=torch.Generator().manual_seed(1)).cuda()
    bits = rng.random((6, vocab)) < np.array([0.5, 0.01, 1.0, 0.0, 0.5, 0.5])[:, None]
    bits[4, vocab // 2:] = False
    bits[5, :vocab // 2] = False
    words = torch.from_numpy(np.stack([ref.pack_mask(b) for b in bits])).cuda()
    for s in (dict(), dict(k=20), dict(p=0.9), dict(mp=0.05), dict(T=0.0)):
        check_sample(ctx, z, u, mask=words, bits=bits, **s)
        check_sample(ctx, z, u, mask=words[0].contiguous(), bits=bits[0], **s)


def test_sample_frequencies_follow_the_softmax(ctx):
    """50,000 draws from one row of 20 logits: every frequency within 5 standard deviations."""
    import torch

    n = 50000
    z = table(1, 20, "bf16", 3, spread=1.5).expand(n, 20)
    u = torch.rand(n, generator=torch.Generator().manual_seed(4)).cuda()
    tok = host(ctx.sample_tokens(z, u)["tokens"])
    zh = host(z[0])
    p = np.exp(zh - zh.max())
    p /= p.sum()
    f = np.bincount(tok, minlength=20) / n
    assert (np.abs(f - p) <= 5 * np.sqrt(p * (1 - p) / n) + 1e-4).all()


def test_sampled_tokens_are_groupby_keys(ctx):
    """Tokens are the dense codes that the grouped statistics take: per-token counts and log-probabilities."""
    import torch

    V, R = 300, 4000
    z = table(1, V, "f16", 3, spread=2.0).expand(R, V).contiguous()
    u = torch.rand(R, generator=torch.Generator().manual_seed(8)).cuda()
    out = ctx.sample_tokens(z, u)
    got = ctx.groupby_dense(out["tokens"], out["logprobs"].double(), V)
    tok = host(out["tokens"])
    assert np.array_equal(host(got["count"]), np.bincount(tok, minlength=V))
    some = np.bincount(tok, minlength=V) > 0
    assert (host(got["min"])[some] == host(got["max"])[some]).all()


# ---- streams, empty tables, refusals -----------------------------------------------------------------


def test_other_stream(ctx):
    import torch

    z = table(64, 32001, "bf16", 3)
    u = torch.full((64,), 0.5, device="cuda")
    want = ctx.sample_tokens(z, u)["tokens"]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a = ctx.sample_tokens(z, u, stream=s, sync=False)
    b = ctx.top_logits(z, 4, stream=s, sync=False)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(a["tokens"], want)
    assert torch.equal(b["ids"], ctx.top_logits(z, 4, stream=s.cuda_stream)["ids"])


def test_graph_capture(ctx):
    """A captured call replays on new contents of the same tensors."""
    import torch

    z = table(8, 5001, "bf16", 3)
    u = torch.full((8,), 0.5, device="cuda")
    out = {"tokens": torch.empty(8, dtype=torch.int32, device="cuda"), "logprobs": torch.empty(8, device="cuda")}
    ctx.sample_tokens(z, u, top_k=20, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ctx.sample_tokens(z, u, top_k=20, out=out, sync=False)
    z.copy_(table(8, 5001, "bf16", 4))
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out["tokens"], ctx.sample_tokens(z, u, top_k=20)["tokens"])


def test_no_rows(ctx):
    import torch

    z = torch.empty(0, 100, device="cuda")
    none = torch.empty(0, device="cuda")
    assert ctx.sample_tokens(z, none)["tokens"].shape == (0,)
    assert ctx.top_logits(z, 3)["ids"].shape == (0, 3)
    ids = torch.empty(0, 4, dtype=torch.int32, device="cuda")
    assert ctx.distill_step(z, ids, torch.empty(0, 4, device="cuda"), none)["grad"].shape == (0, 100)


def test_refusals(ctx):
    import torch

    import winrapids_b200 as wb

    z = table(2, 100, "f32", 1)
    u = torch.zeros(2, device="cuda")
    ids = torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    t, w = torch.zeros(2, 3, device="cuda"), torch.ones(2, device="cuda")
    bad = [
        lambda: ctx.top_logits(z.double(), 3),
        lambda: ctx.top_logits(z.cpu(), 3),
        lambda: ctx.top_logits(z[0], 3),
        lambda: ctx.top_logits(z.t(), 3),
        lambda: ctx.top_logits(z[:, ::2], 3),
        lambda: ctx.top_logits(z, 0),
        lambda: ctx.top_logits(z, 1025),
        lambda: ctx.top_logits(z, 3, temperature=0.0),
        lambda: ctx.top_logits(z, 3, temperature=float("nan")),
        lambda: ctx.top_logits(z, 3, temperature=float("inf")),
        lambda: ctx.top_logits(z[:, :0], 3),
        lambda: ctx.top_logits(z, 3, mask=torch.zeros(1, dtype=torch.int64, device="cuda")),
        lambda: ctx.top_logits(z, 3, mask=torch.zeros(2, 2, device="cuda")),
        lambda: ctx.top_logits(z, 3, mask=torch.zeros(3, 2, dtype=torch.int64, device="cuda")),
        lambda: ctx.top_logits(z, 3, out={"ids": torch.empty(2, 3, device="cuda")}),
        lambda: ctx.sample_tokens(z, u[:1]),
        lambda: ctx.sample_tokens(z, u.double()),
        lambda: ctx.sample_tokens(z, u, top_k=torch.zeros(2, device="cuda")),
        lambda: ctx.sample_tokens(z, u, temperature=torch.ones(3, device="cuda")),
        lambda: ctx.sample_tokens(z, u, temperature=torch.ones(4, device="cuda")[::2]),
        lambda: ctx.distill_loss(z, ids.long(), t),
        lambda: ctx.distill_loss(z, ids[:1], t),
        lambda: ctx.distill_loss(z, ids, t[:, :2]),
        lambda: ctx.distill_loss(z, ids, t.double()),
        lambda: ctx.distill_loss(z, ids, t, temperature=-1.0),
        lambda: ctx.distill_loss(z, ids, t, teacher_lse=w.double()),
        lambda: ctx.distill_loss(z, ids[:, :0], t[:, :0]),
        lambda: ctx.distill_step(z, ids, t, w[:1]),
        lambda: ctx.distill_step(z, ids, t, w, grad=torch.empty(2, 100, device="cuda", dtype=torch.float16)),
        lambda: ctx.distill_step(z, ids, t, w, grad=torch.empty(1, 100, device="cuda").expand(2, 100)),
        lambda: ctx.distill_grad(z, ids, t, torch.zeros(2, device="cuda"), w),
        lambda: wb.distill_loss(z.t(), wb.TopLogits(t, ids, None, 1.0)),
    ]
    for f in bad:
        with pytest.raises(wb.InvalidArgument):
            f()
    ctx.sync()


def test_example_runs(ctx):
    """examples/distill_and_sample.py: the loss falls, the answers come from the record, every row is counted."""
    import importlib.util
    from pathlib import Path

    path = Path(__file__).resolve().parents[1] / "examples" / "distill_and_sample.py"
    spec = importlib.util.spec_from_file_location("distill_and_sample", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    got = m.main(["--rows", "256", "--vocab", "1000", "--k", "16", "--steps", "20"])
    assert got["after"] < 0.7 * got["before"]
    assert got["agree"] > 0.5 and got["count"] == 256
