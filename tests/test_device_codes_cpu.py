"""Codes of the device error word, by the sources: an id outside a table has one of its own, which no wait reports."""
import os
import re

from hdcmamba_b200.build import CSRC

REPORTS = (r"(?:mbar_wait(?:_warp)?|wait_flags?|cta_wait_flags)\(.*?, (k\w+|\d+)\)", r"atomicCAS\(&g_dev_error, 0, (k\w+|\d+)\)")


def codes(name):
    """The numbers that a source's waits and checks report (a name's by its constant)."""
    text = open(os.path.join(CSRC, name)).read()
    named = dict(re.findall(r"constexpr int (k\w+) = (\d+);", text))
    return {int(named.get(c, c)) for report in REPORTS for c in re.findall(report, text)}


def test_an_id_outside_the_table_has_a_code_of_its_own():
    found = {n: codes(n) for n in sorted(os.listdir(CSRC)) if n.endswith(".cu")}
    assert found["embedding.cu"] == {71}
    assert found["decay_attn_tc.cu"] == {81} and found["slot_tc.cu"] and found["slot_mc.cu"]
    assert [n for n, c in found.items() if 71 in c] == ["embedding.cu"]
