"""The functions of winrapids_b200/logits.py without a device: what they hand to a context, and when."""
import threading
import time

import pytest

torch = pytest.importorskip("torch")

import winrapids_b200 as wb  # noqa: E402
from winrapids_b200 import logits as module  # noqa: E402


class FakeContext:
    """Takes calls as a Context does; notes the ones that overlap."""

    made = 0

    def __init__(self, device):
        type(self).made += 1
        self.inside, self.overlaps, self.calls = 0, 0, []
        time.sleep(0.01)

    def _enter(self, name, args, kwargs):
        self.overlaps += self.inside > 0
        self.inside += 1
        time.sleep(0.001)
        self.inside -= 1
        self.calls.append((name, args, kwargs))

    def top_logits(self, z, k, **kw):
        self._enter("top_logits", (z, k), kw)
        rows = z.shape[0]
        return {"values": torch.zeros(rows, k), "ids": torch.zeros(rows, k, dtype=torch.int32), "lse": torch.zeros(rows)}

    def sample_tokens(self, z, u, **kw):
        self._enter("sample_tokens", (z, u), kw)
        rows = z.shape[0]
        return {"tokens": torch.zeros(rows, dtype=torch.int32), "logprobs": torch.zeros(rows)}


@pytest.fixture
def fake(monkeypatch):
    FakeContext.made = 0
    monkeypatch.setattr(module, "Context", FakeContext)
    monkeypatch.setattr(module, "_CTX", {})
    monkeypatch.setattr(module, "_device", lambda z: 0)
    return module._CTX


def test_one_call_at_a_time_on_the_shared_context(fake):
    def work():
        for _ in range(10):
            wb.top_logits(torch.zeros(2, 3, 5), 2)
            wb.sample_tokens(torch.zeros(2, 5), torch.zeros(2))

    threads = [threading.Thread(target=work) for _ in range(6)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert FakeContext.made == 1
    assert len(fake[0].calls) == 120 and fake[0].overlaps == 0


def test_logits_on_the_host_are_refused():
    for f in (lambda z: wb.top_logits(z, 2), lambda z: wb.sample_tokens(z, torch.zeros(2)),
              lambda z: wb.distill_loss(z, wb.TopLogits(z[:, :2], z[:, :2].int(), None, 1.0))):
        with pytest.raises(wb.InvalidArgument):
            f(torch.zeros(2, 5))


def test_masks_take_the_leading_shape(fake):
    z, u = torch.zeros(2, 3, 130), torch.zeros(2, 3)
    words = torch.arange(18).view(2, 3, 3)
    wb.top_logits(z, 2, mask=words)
    wb.sample_tokens(z, u, mask=words)
    wb.top_logits(z, 2, mask=words[0, 0])
    wb.sample_tokens(z[0], u[0], mask=words[0])
    wb.sample_tokens(z[0, 0], u[0, 0], mask=words[0, 0])
    wb.sample_tokens(z, u, mask=words.view(6, 3))
    got = [c[2]["mask"] for c in fake[0].calls]
    assert torch.equal(got[5], words.view(6, 3))
    assert torch.equal(got[0], words.view(6, 3)) and torch.equal(got[1], words.view(6, 3))
    assert torch.equal(got[2], words[0, 0]) and torch.equal(got[3], words[0]) and torch.equal(got[4], words[0, 0])
    with pytest.raises(wb.InvalidArgument):
        wb.top_logits(z, 2, mask=words[:, :2])
    with pytest.raises(wb.InvalidArgument):
        wb.sample_tokens(z, u, mask=words.view(3, 2, 3))


def test_k_past_32_bits_is_no_other_k(fake):
    z, u = torch.zeros(3, 130), torch.zeros(3)
    wb.sample_tokens(z, u, top_k=torch.tensor([7, 2 ** 32 + 5, -2 ** 32 + 3]))
    assert fake[0].calls[0][2]["top_k"].tolist() == [7, 2 ** 31 - 1, 0]


@pytest.mark.parametrize("k,want", [(5, 5), (2 ** 32 + 5, 2 ** 31 - 1), (-2 ** 32 + 3, 0), (2 ** 31, 2 ** 31 - 1)])
def test_a_number_k_past_32_bits_is_no_other_k(monkeypatch, k, want):
    seen = []

    class Library:
        def tbgb_sample_tokens(self, h, x, u, p, *rest):
            seen.append(p.top_k_all)
            return 0

    c = wb.Context.__new__(wb.Context)
    c._L, c._h, c.device, c._torch_dev = Library(), None, 0, torch.device("cpu")
    monkeypatch.setattr(wb.Context, "_check_tensor", lambda self, t, what, dtypes: None)
    monkeypatch.setattr(wb, "_current_stream", lambda device: 0)
    c.sample_tokens(torch.zeros(2, 9), torch.zeros(2), top_k=k, sync=False)
    assert seen == [want]


def test_a_context_does_not_need_torch():
    """Only the calls that make tensors do."""
    import subprocess
    import sys

    program = """
import sys
sys.modules["torch"] = None  # an import of it fails
import winrapids_b200 as wb

class Library:
    def tbgb_create(self, device, handle): return 0
    def tbgb_destroy(self, handle): return 0

wb.lib = Library
c = wb.Context(0)
c.close()
print("made")
"""
    got = subprocess.run([sys.executable, "-c", program], capture_output=True, text=True, timeout=120)
    assert got.stdout.strip() == "made", got.stderr
