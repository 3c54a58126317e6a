"""The protocol of the distillation kernel's ring (winrapids_b200/csrc/distill.cu, distill_kernel) as a model:
a cluster of CTAs, in each a producer, an entries' warp and softmax warps, with the kernel's barriers, taken
in random orders.  Every bounded wait may give up at any moment.  Then:

* nothing waits without a limit for a warp that does not come (the softmax warps' barrier, the cluster's)
* no CTA is written to after it has left
* without a wait that gives up, every role sees the row that it works on in every buffer it reads
"""
import random

import pytest

NW = 4


class Barrier:
    def __init__(self, count):
        self.count, self.left, self.phase = count, count, 0

    def arrive(self):
        self.left -= 1
        assert self.left >= 0
        if self.left == 0:
            self.left, self.phase = self.count, self.phase + 1

    def passed(self, n):  # the kernel asks by the parity of phase n
        return (self.phase & 1) != (n & 1)


class Cta:
    def __init__(self, C):
        mk = lambda c: [Barrier(c), Barrier(c)]  # noqa: E731
        self.full, self.done, self.ready, self.counted, self.heard = mk(1), mk(NW), mk(1), mk(1), mk(C)
        self.stage, self.counted_row, self.parts = [None, None], [None, None], [[None] * C for _ in range(4)]
        self.met = 0        # warps at the softmax warps' barrier
        self.failed = []    # what each brought
        self.meetings = 0
        self.left = 0       # warps that have ended


class Model:
    """`closing`: the kernel as it is; otherwise roles end one by one where a wait gives up."""

    def __init__(self, C, rows, weights, gives_up, grad, closing, rng):
        self.ctas = [Cta(C) for _ in range(C)]
        self.C, self.rows, self.weights, self.gives_up, self.grad, self.closing, self.rng = (
            C, rows, weights, gives_up, grad, closing, rng)
        self.at_end, self.gave_up, self.wrote_to_left = 0, 0, 0

    # yields: ("wait", predicate) bounded, ("must", predicate) unbounded, None: another may go first.  wait() is the answer.
    def wait(self, pred):
        ok = yield ("wait", pred)
        return ok

    def end(self, cta):
        if self.closing:
            self.at_end += 1
            yield ("must", lambda: self.at_end == self.C * (NW + 2))
        cta.left += 1

    def live(self, r):
        return self.weights[r] != 0

    def producer(self, cta):
        n = 0
        for r in range(self.rows):
            if not self.live(r):
                continue
            s = n & 1
            if n >= 2 and not (yield from self.wait(lambda: cta.done[s].passed((n >> 1) - 1))):
                break
            cta.stage[s] = ("copy", r)
            yield None
            cta.full[s].arrive()
            n += 1
        yield from self.end(cta)

    def entries(self, cta):
        n, last = 0, None
        ok = True

        def finish():
            m, r = last
            if not (yield from self.wait(lambda: cta.heard[m & 1].passed(m >> 1))):
                return False
            yield None
            self.see(cta.parts[m & 3], [r] * self.C)
            if self.grad and not (yield from self.wait(lambda: cta.done[m & 1].passed(m >> 1))):
                return False
            return True

        for r in range(self.rows):
            if not self.live(r):
                continue
            s = n & 1
            ok = yield from self.wait(lambda: cta.full[s].passed(n >> 1))
            if not ok:
                break
            self.see(cta.stage[s], ("copy", r))
            cta.stage[s] = ("cut", r)
            yield None
            cta.ready[s].arrive()
            yield None
            cta.counted_row[s] = r
            cta.counted[s].arrive()
            if last is not None:
                ok = yield from finish()
                if not ok:
                    break
            last = (n, r)
            n += 1
        if last is not None and ok:
            yield from finish()
        yield from self.end(cta)

    def see(self, got, want):
        if not self.gave_up:
            assert got == want, (got, want)

    def softmax(self, cta, rank, warp):
        n, ok = 0, True
        for r in range(self.rows):
            if not self.live(r):
                continue
            s = n & 1
            ok = ok and (yield from self.wait(lambda: cta.full[s].passed(n >> 1)))
            ok = ok and (yield from self.wait(lambda: cta.ready[s].passed(n >> 1)))
            if not ok and not self.closing:
                break
            if ok:
                self.see(cta.stage[s], ("cut", r))
                yield None
                if not self.grad:
                    cta.done[s].arrive()
            # the barrier of these warps, with what each brings
            mine = cta.meetings
            cta.failed.append(not ok)
            if len(cta.failed) == NW:
                cta.verdict, cta.failed, cta.meetings = any(cta.failed), [], cta.meetings + 1
            yield ("must", lambda: cta.meetings > mine)
            if cta.verdict and self.closing:
                break
            if warp == 0:
                ok = yield from self.wait(lambda: cta.counted[s].passed(n >> 1))
                if not ok and not self.closing:
                    break
                self.see(cta.counted_row[s], r)
                for c in range(self.C if ok else 0):
                    yield None
                    peer = self.ctas[c]
                    self.wrote_to_left += peer.left == NW + 2
                    peer.parts[n & 3][rank] = r
                    peer.heard[s].arrive()
            ok = ok and (yield from self.wait(lambda: cta.heard[s].passed(n >> 1)))
            if not ok and not self.closing:
                break
            if ok:
                self.see(cta.parts[n & 3], [r] * self.C)
                yield None
                if self.grad:
                    self.see(cta.stage[s], ("cut", r))
                    cta.done[s].arrive()
            n += 1
        yield from self.end(cta)

    def run(self):
        tasks = []
        for rank, cta in enumerate(self.ctas):
            tasks += [self.producer(cta), self.entries(cta)] + [self.softmax(cta, rank, w) for w in range(NW)]
        state = {t: None for t in tasks}  # what each waits for
        answer = {t: None for t in tasks}
        while state:
            go = []
            for t, w in state.items():
                if w is None or w[1]():
                    go.append((t, True))
                elif w[0] == "wait" and (self.rng.random() < self.gives_up):
                    go.append((t, False))
            if not go:  # nothing moves: the limits run out
                go = [(t, False) for t, w in state.items() if w[0] == "wait"]
                if not go or self.gives_up == 0:
                    return False  # waits without a limit (or, without a delay, at all)
            t, ok = self.rng.choice(go)
            if not ok:
                self.gave_up += 1
            answer[t] = ok
            try:
                state[t] = t.send(ok if state[t] is not None and state[t][0] == "wait" else None)
            except StopIteration:
                del state[t]
        return True


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("C,rows", [(1, 9), (2, 7), (4, 6), (8, 5)])
def test_buffers_hold_the_row_that_is_worked_on(C, rows, grad):
    for seed in range(60):
        rng = random.Random(seed)
        weights = [rng.random() < 0.75 for _ in range(rows)]  # padding rows between the others
        m = Model(C, rows, weights, 0.0, grad, True, rng)
        assert m.run() and not m.gave_up and not m.wrote_to_left, seed


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("C,rows", [(1, 5), (2, 5), (4, 4)])
def test_a_wait_that_gives_up_ends_the_kernel(C, rows, grad):
    gave_up = 0
    for seed in range(400):
        m = Model(C, rows, [1] * rows, 10.0 ** -random.Random(seed).uniform(0.5, 4), grad, True, random.Random(seed))
        assert m.run(), seed
        assert not m.wrote_to_left, seed
        gave_up += m.gave_up > 0
    assert gave_up > 100


def test_the_model_sees_roles_that_leave_on_their_own():
    hangs = written = 0
    for seed in range(400):
        m = Model(2, 5, [1] * 5, 0.01, True, False, random.Random(seed))
        hangs += not m.run()
        written += m.wrote_to_left > 0
    assert hangs > 0


def test_the_kernel_leaves_by_one_way():
    """The roles end in one cluster barrier, and a softmax warp reaches its barrier before it may stop."""
    from test_logits_source_host import kernel

    body = kernel("distill.cu", "distill_kernel")
    roles = body[body.index("if (warp == NW)"):]
    outer = [line.strip() for line in roles.split("\n") if line.startswith("    return") or line.startswith("  return")]
    assert outer == []
    assert roles.rstrip().endswith("cl.sync();")
    soft = roles[roles.index("bool ok = true;"):]
    assert "return;" not in soft
    assert soft.count("break;") == 1 and "if (any_failed<NT>(!ok)) break;" in soft
