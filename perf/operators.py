"""What is measured of the operators on rows of logits: recording a teacher's top logits, the
distillation loss with its gradient, and sampling of tokens.

A case names the operator, the rows R, the vocabulary V, the element type and what the operator
needs besides.  `run` with `own` false is the plain form (elementary torch operations in 32 bits);
with `own` true it makes the calls of winrapids_b200.Context.  `exact` is the definition in 64 bits.

Sampling weights are whole numbers: 2^((z - zmax) * log2(e) / T) in 32 bits, rounded to multiples of
2^-30, so that every sum is exact and a token does not depend on the order of summation.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
LOG2E = 1.4426950408889634
GRID = float(2 ** 30)
NEG_INF = float("-inf")


def listed():
    return [
        # the top five of each token that a server has just produced, asked for beside the text
        dict(name="top_served", op="top", R=8, V=32000, dtype="bf16", K=5, T=1.0),
        # a record of a teacher in 32 bits over a vocabulary of odd size (rows start anywhere)
        dict(name="top_odd", op="top", R=509, V=50001, dtype="f32", K=20, T=1.0),
        # a training batch of teacher logits recorded for later
        dict(name="top_record", op="top", R=2048, V=131072, dtype="bf16", K=64, T=2.0),
        # a byte-sized experiment: few tokens, small vocabulary, the teacher's entries closed among themselves
        dict(name="distill_small", op="step", R=16, V=4099, dtype="f32", K=8, T=1.0, tail=False),
        # validation loss of a student
        dict(name="distill_eval", op="loss", R=2048, V=100003, dtype="f16", K=32, T=1.0, tail=True),
        # the backward pass alone, for a loss whose weights are known only after the forward pass
        dict(name="distill_backward", op="grad", R=1024, V=50001, dtype="f32", K=100, T=2.0, tail=True),
        # a training step: loss and gradient of a batch
        dict(name="distill_train", op="step", R=4096, V=131072, dtype="bf16", K=64, T=1.0, tail=True),
        # one conversation
        dict(name="sample_one", op="sample", R=1, V=131072, dtype="bf16", params="top_k+top_p", mask=0.0),
        # a server's batch, each row with settings of its own
        dict(name="sample_served", op="sample", R=256, V=131072, dtype="bf16", params="mixed", mask=0.0),
        # rollouts for training: the model's own distribution, nothing cut off
        dict(name="sample_rollout", op="sample", R=1024, V=100000, dtype="bf16", params="free", mask=0.0),
        # nucleus sampling alone, from logits in 32 bits
        dict(name="sample_nucleus", op="sample", R=64, V=150001, dtype="f32", params="top_p", mask=0.0),
        # constrained output: one token in fifty is allowed
        dict(name="sample_grammar", op="sample", R=32, V=50001, dtype="f16", params="min_p", mask=0.02),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["top", "loss", "grad", "step", "sample", "sample"])
    most = {"top": 2048 * 131072, "loss": 4096 * 131072, "grad": 2048 * 131072, "step": 4096 * 131072,
            "sample": 1024 * 100000}[op]
    V = _log_int(rng, 1000, 150001)
    dtype = rng.choice(["f32", "f16", "bf16"])
    if dtype == "f32":
        most //= 2
    R = _log_int(rng, 1, max(1, min(4096, most // V)))
    if op == "sample":
        return dict(op=op, R=R, V=V, dtype=dtype, params=rng.choice(["top_k+top_p", "mixed", "free", "top_p", "min_p"]),
                    mask=rng.choice([0.0, 0.0, 0.02, 0.5]))
    case = dict(op=op, R=R, V=V, dtype=dtype, K=_log_int(rng, 1, 128), T=rng.choice([0.7, 1.0, 2.0]))
    if op != "top":
        case.update(K=max(8, case["K"]), tail=rng.choice([False, True]))
    return case


def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _logits(case, g):
    """Logits as a language model gives them: common tokens ahead of rare ones, a spread of two around
    that, and a few tokens per row that stand out."""
    R, V = case["R"], case["V"]
    prior = -0.7 * torch.log1p(torch.randperm(V, generator=g, device="cuda").float())
    z = torch.randn(R, V, generator=g, device="cuda").mul_(2.0).add_(prior)
    at = torch.randint(0, V, (R, 6), generator=g, device="cuda")
    high = 3.0 + 5.0 * torch.rand(R, 6, generator=g, device="cuda")
    for j in range(6):  # one at a time: where a row draws a position twice, the later value stays, in every process
        z.scatter_(1, at[:, j:j + 1], high[:, j:j + 1])
    return z


def prepare(case, seed):
    g = _gen(seed)
    R, V, dt = case["R"], case["V"], DTYPES[case["dtype"]]
    z = _logits(case, g)
    if case["op"] == "top":
        return dict(case=case, logits=z.to(dt))
    if case["op"] == "sample":
        s = dict(case=case, logits=z.to(dt), u=torch.rand(R, generator=g, device="cuda"),
                 temperature=0.8, top_k=0, top_p=1.0, min_p=0.0, allowed=None)
        kind = case["params"]
        if kind == "top_k+top_p":
            s.update(top_k=50, top_p=0.9)
        elif kind == "top_p":
            s.update(top_p=0.95)
        elif kind == "min_p":
            s.update(min_p=0.05)
        elif kind == "free":
            s.update(temperature=1.0)
        else:  # every row its own
            pick = torch.randint(0, 4, (R,), generator=g, device="cuda")
            s["temperature"] = torch.rand(R, generator=g, device="cuda") + 0.5
            s["top_k"] = torch.where((pick == 0) | (pick == 1), torch.randint(1, 200, (R,), generator=g, device="cuda"),
                                     0).int()
            s["top_p"] = torch.where((pick == 1) | (pick == 2), 0.8 + 0.19 * torch.rand(R, generator=g, device="cuda"), 1.0)
            s["min_p"] = torch.where(pick == 3, 0.02 + 0.1 * torch.rand(R, generator=g, device="cuda"), 0.0)
        if case["mask"]:
            words = (V + 63) // 64
            bit = torch.rand(R, words * 64, generator=g, device="cuda") < case["mask"]
            bit[:, 0] = True
            place = torch.ones(64, dtype=torch.int64, device="cuda") << torch.arange(64, device="cuda")
            s["allowed"] = (bit.view(R, words, 64) * place).sum(2)
        return s
    # distillation: a teacher near the student, its K largest logits in the order of their size
    K, T = min(case["K"], V), case["T"]
    teacher = torch.randn(R, V, generator=g, device="cuda").mul_(1.5).add_(z).to(dt).float()
    lse = torch.logsumexp(teacher / T, 1) if case["tail"] else None
    top, ids = torch.topk(teacher, K, dim=1)
    del teacher
    weight = (0.5 + torch.rand(R, generator=g, device="cuda")) / R
    s = dict(case=case, logits=z.to(dt), ids=ids.int(), teacher=top.to(dt), lse=lse, weight=weight)
    if case["op"] == "grad":
        s["stats"] = _distill(s, with_grad=False)["stats"]
    return s


# ---- the plain forms ---------------------------------------------------------------------------------


def _top(s):
    case = s["case"]
    K = min(case["K"], case["V"])
    z = s["logits"].float()
    top, ids = torch.sort(z, dim=1, descending=True, stable=True)
    x = z / case["T"]
    m = x.max(1).values
    lse = m + torch.log(torch.exp(x - m[:, None]).sum(1))
    return dict(values=top[:, :K].to(s["logits"].dtype), ids=ids[:, :K].int(), lse=lse)


def _distill(s, with_grad=True, stats=None):
    T, ids = s["case"]["T"], s["ids"].long()
    x, t = s["logits"].float() / T, s["teacher"].float() / T
    if s["lse"] is not None:
        logp = t - s["lse"][:, None]
    else:
        tm = t.max(1, keepdim=True).values
        logp = t - tm - torch.log(torch.exp(t - tm).sum(1, keepdim=True))
    p = torch.exp(logp)
    out = {}
    if stats is None:
        m = x.max(1, keepdim=True).values
        lse = m + torch.log(torch.exp(x - m).sum(1, keepdim=True))
        logq = x.gather(1, ids) - lse
        loss = (p * (logp - logq)).sum(1)
        off = torch.ones_like(loss)
        if s["lse"] is not None:  # one more outcome: any token outside the record
            p_in, q_in = p.sum(1), torch.exp(logq).sum(1)
            e = torch.exp(x - m)
            q_out = e.scatter(1, ids, 0.0).sum(1) / e.sum(1)
            there = (p_in < 1) & (q_out > 0)
            log_q_out = torch.where(q_in < 0.5, torch.log1p(-q_in), torch.log(q_out))
            loss = loss + torch.where(there, (1 - p_in) * (torch.log1p(-p_in) - log_q_out), 0.0)
            off = torch.where(there, (p_in - q_in) / q_out, 1.0)
        stats = torch.stack([lse[:, 0], off], 1)
        out.update(loss=loss, stats=stats)
    if with_grad:
        q = torch.exp(x - stats[:, :1])
        g = (q * stats[:, 1:]).scatter(1, ids, q.gather(1, ids) - p)
        out["grad"] = (g * (s["weight"] / T)[:, None]).to(s["logits"].dtype)
    return out


def _bits(words, V):
    i = torch.arange(V, device=words.device)
    return ((words[:, i >> 6] >> (i & 63)) & 1).bool()


def _column(v, R):
    return v[:, None] if isinstance(v, torch.Tensor) else torch.full((R, 1), v, device="cuda")


def _sample(s):
    R, V = s["case"]["R"], s["case"]["V"]
    z = s["logits"].float()
    if s["allowed"] is not None:
        z = torch.where(_bits(s["allowed"], V), z, NEG_INF)
    T, min_p = _column(s["temperature"], R).float(), _column(s["min_p"], R)
    zmax = z.max(1, keepdim=True).values
    e = torch.exp2((z - zmax) * (torch.full_like(T, LOG2E) / T))
    w = torch.round(e * GRID).to(torch.int64)
    if isinstance(s["top_k"], torch.Tensor) or s["top_k"] > 0 or s["top_p"] < 1.0:
        k, top_p = _column(s["top_k"], R), _column(s["top_p"], R)
        order = torch.sort(z, dim=1, descending=True, stable=True).indices
        at = torch.arange(V, device="cuda")[None]
        ws = torch.where((at < k) | (k <= 0), w.gather(1, order), 0)
        need = torch.ceil(top_p.double() * ws.sum(1, keepdim=True).double()).clamp(min=1.0)
        before = torch.cumsum(ws, 1) - ws
        ws = torch.where((before.double() < need) | (top_p >= 1.0), ws, 0)
        w = torch.zeros_like(w).scatter(1, order, ws)
    w = torch.where(e >= min_p, w, 0)
    total = torch.cumsum(w, 1)
    W = total[:, -1:]
    target = torch.floor(s["u"].double()[:, None] * W.double()).to(torch.int64)
    token = (total <= torch.minimum(target, W - 1)).sum(1)
    logprob = (z.gather(1, token[:, None]) - zmax) / T - torch.log((W.double() / GRID).float())
    return dict(tokens=token.int(), logprobs=logprob[:, 0])


# ---- the framework's calls ----------------------------------------------------------------------------

_ctx = None


def _context():
    global _ctx
    if _ctx is None:
        import winrapids_b200 as wb

        _ctx = wb.Context(0)
    return _ctx


def _run_own(s):
    ctx, case, op = _context(), s["case"], s["case"]["op"]
    if op == "top":
        return ctx.top_logits(s["logits"], min(case["K"], case["V"]), temperature=case["T"], sync=False)
    if op == "sample":
        return ctx.sample_tokens(s["logits"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                 min_p=s["min_p"], mask=s["allowed"], sync=False)
    teach = dict(teacher_lse=s["lse"], temperature=case["T"], sync=False)
    if op == "loss":
        return ctx.distill_loss(s["logits"], s["ids"], s["teacher"], **teach)
    if op == "grad":
        return dict(grad=ctx.distill_grad(s["logits"], s["ids"], s["teacher"], s["stats"], s["weight"], **teach))
    return ctx.distill_step(s["logits"], s["ids"], s["teacher"], s["weight"], **teach)


def run(state):
    if own:
        return _run_own(state)
    op = state["case"]["op"]
    if op == "top":
        return _top(state)
    if op == "sample":
        return _sample(state)
    if op == "loss":
        return _distill(state, with_grad=False)
    if op == "grad":
        return _distill(state, stats=state["stats"])
    return _distill(state)


def work(case):
    R, V, b = case["R"], case["V"], 4 if case["dtype"] == "f32" else 2
    rows = R * V * b
    if case["op"] == "top":
        K = min(case["K"], V)
        return {"bytes": rows + R * (K * (b + 4) + 4), "flops": 3 * R * V}
    if case["op"] == "sample":
        return {"bytes": rows + (R * ((V + 63) // 64) * 8 if case["mask"] else 0) + R * 12, "flops": 4 * R * V}
    record = R * (min(case["K"], V) * (4 + b) + (4 if case["tail"] else 0))
    if case["op"] == "loss":
        return {"bytes": rows + record + 12 * R, "flops": 3 * R * V}
    if case["op"] == "grad":
        return {"bytes": 2 * rows + record + 12 * R, "flops": 4 * R * V}
    return {"bytes": 2 * rows + record + 16 * R, "flops": 7 * R * V}


# ---- the definition in 64 bits ---------------------------------------------------------------------------


def _exact_sample(s):
    """The definition with the power of two and the comparisons in 64 bits; the exponent is the one that the
    definition rounds to 32 bits.  Rows are cut by thresholds in the order of their sorted logits."""
    z, u = s["logits"].double(), s["u"].double()
    R, V = z.shape
    if s["allowed"] is not None:
        bit = torch.stack([(s["allowed"] >> j) & 1 for j in range(64)], 2).reshape(R, -1)[:, :V]
        z = z.masked_fill(bit == 0, NEG_INF)
    tensor = lambda v: v.double() if isinstance(v, torch.Tensor) else torch.full((R,), float(v), dtype=torch.float64,  # noqa: E731
                                                                                   device=z.device)
    T, k, top_p, min_p = (tensor(s[n]) for n in ("temperature", "top_k", "top_p", "min_p"))
    top_p = top_p if isinstance(s["top_p"], torch.Tensor) else top_p.float().double()
    zs, order = torch.sort(z, dim=1, descending=True, stable=True)
    scale = torch.full_like(u, LOG2E).float() / T.float()
    d = ((zs.float() - zs[:, :1].float()) * scale[:, None]).double()
    e = torch.pow(2.0, d)
    unit = torch.floor(e * GRID + 0.5)
    place = torch.arange(V, device=z.device, dtype=torch.float64).expand(R, V)
    unit[(place >= k[:, None]) & (k[:, None] > 0)] = 0.0
    sums = unit.cumsum(1)
    need = torch.ceil(top_p * sums[:, -1]).clamp(min=1.0)[:, None]
    last = torch.searchsorted(sums, need)  # the entry whose sum reaches what is needed
    unit[(place > last) & (top_p < 1.0)[:, None]] = 0.0
    unit[e < min_p.float().double()[:, None]] = 0.0
    sums = torch.zeros_like(unit).scatter_(1, order, unit).cumsum(1)
    goal = torch.floor(u * sums[:, -1])[:, None]
    token = torch.searchsorted(sums, goal, right=True).clamp(max=V - 1)
    x = (z.gather(1, token)[:, 0] - zs[:, 0]) / T
    return dict(tokens=token[:, 0].int(), logprobs=x - torch.log(sums[:, -1] / GRID))


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    T, z = case["T"], s["logits"].double()
    if case["op"] == "top":
        values = torch.topk(z, min(case["K"], case["V"]), dim=1).values
        return dict(values=values, ids=None, lse=torch.logsumexp(z / T, 1))
    ids = s["ids"].long()
    logq = torch.log_softmax(z / T, 1)
    if s["lse"] is None:
        logp, p_rest = torch.log_softmax(s["teacher"].double() / T, 1), None
    else:
        logp = s["teacher"].double() / T - s["lse"].double()[:, None]
        p_rest = (1.0 - logp.exp().sum(1)).clamp(min=0.0)
    if case["op"] == "grad":
        q = torch.exp(z / T - s["stats"][:, :1].double())
        off = s["stats"][:, 1].double()
    else:
        loss = (logp.exp() * (logp - logq.gather(1, ids))).sum(1)
        q, off = logq.exp(), torch.ones_like(loss)
        if p_rest is not None:
            q_rest = q.scatter(1, ids, 0.0).sum(1)
            loss = loss + torch.xlogy(p_rest, p_rest) - p_rest * q_rest.log()
            off = 1.0 - p_rest / q_rest
    if case["op"] == "loss":
        return dict(loss=loss, stats=torch.stack([torch.logsumexp(z / T, 1), off], 1))
    slope = q * off[:, None]
    slope.scatter_(1, ids, q.gather(1, ids) - logp.exp())
    grad = slope * (s["weight"].double() / T)[:, None]
    if case["op"] == "grad":
        return dict(grad=grad)
    return dict(loss=loss, stats=torch.stack([torch.logsumexp(z / T, 1), off], 1), grad=grad)
