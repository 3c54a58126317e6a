"""The cases of perf/operators.py: what a seed prepares is the same in every process, also where a row's
standing-out logits fall on one position more than once (4096 rows of 1000: about 60 rows do)."""
import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent

PROGRAM = """
import hashlib, importlib.util, torch
spec = importlib.util.spec_from_file_location("operators", "perf/operators.py")
m = importlib.util.module_from_spec(spec)
spec.loader.exec_module(m)
for seed in range(8):
    s = m.prepare(dict(op="step", R=4096, V=1000, dtype="f32", K=64, T=1.0, tail=True), seed)
    for k in sorted(s):
        if isinstance(s[k], torch.Tensor):
            print(seed, k, hashlib.md5(s[k].cpu().numpy().tobytes()).hexdigest())
"""


def test_a_seed_prepares_the_same_in_every_process():
    said = [subprocess.run([sys.executable, "-c", PROGRAM], cwd=ROOT, capture_output=True, text=True, timeout=300)
            for _ in range(3)]
    for s in said:
        assert s.returncode == 0, s.stderr
    assert len(said[0].stdout.split("\n")) > 40
    assert said[0].stdout == said[1].stdout == said[2].stdout


def test_the_later_value_stays():
    """What a row holds at a repeated position is the last of the values drawn for it."""
    import importlib.util

    import torch

    spec = importlib.util.spec_from_file_location("operators", ROOT / "perf" / "operators.py")
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    R, V = 4096, 1000
    z = m._logits(dict(R=R, V=V), m._gen(3)).cpu()
    g = m._gen(3)
    torch.randperm(V, generator=g, device="cuda")
    torch.randn(R, V, generator=g, device="cuda")
    at = torch.randint(0, V, (R, 6), generator=g, device="cuda").cpu()
    high = (3.0 + 5.0 * torch.rand(R, 6, generator=g, device="cuda")).cpu()
    last = [dict(zip(a, h)) for a, h in zip(at.tolist(), high.tolist())]
    assert sum(len(d) < 6 for d in last) > 20
    assert all(float(z[r, p]) == h for r, d in enumerate(last) for p, h in d.items())
