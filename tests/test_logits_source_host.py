"""Orders in the kernels on rows of logits that no run shows reliably, read from their source."""
import re
from pathlib import Path

CSRC = Path(__file__).resolve().parent.parent / "winrapids_b200" / "csrc"


def kernel(source: str, name: str) -> str:
    """The text of one function template, without comments."""
    s = re.sub(r"//[^\n]*", "", (CSRC / source).read_text())
    at = re.search(r"\b%s\(const \w+ a[^)]*\) \{" % name, s)
    assert at, name
    depth = 0
    for i in range(at.end() - 1, len(s)):
        depth += (s[i] == "{") - (s[i] == "}")
        if depth == 0:
            return s[at.end():i]
    raise AssertionError(name)


def test_wide_rows_reach_peers_after_a_cluster_barrier():
    """A CTA may touch another's shared memory only once that one is known to have started."""
    body = kernel("distill.cu", "distill_wide_kernel")
    assert body.index("cl.sync()") < body.index("map_shared_rank")
