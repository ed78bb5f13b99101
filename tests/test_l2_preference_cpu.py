"""No kernel leaves lines in L2 that it asked to be kept above all others: they would outlive the call."""
import os

from hdcmamba_b200.build import CSRC


def test_no_load_asks_to_be_kept():
    text = {f: open(os.path.join(CSRC, f)).read() for f in os.listdir(CSRC) if f.endswith((".cu", ".cuh"))}
    assert len(text) > 20
    for word in ("evict_last", "persisting", "AccessPolicyWindow"):
        assert not [f for f, t in text.items() if word in t], word
