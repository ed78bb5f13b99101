"""Codes of the device error word: an id outside a table has one of its own, which no wait reports, and is told apart
from a wait that ran out."""
import ctypes
import os
import re

import pytest
import torch

from hdcmamba_b200 import _lib, ops, sp
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


@pytest.mark.parametrize("code,text", [(71, "outside its table"), (13, "wait"), (41, "wait"), (-1, "wait")])
def test_what_the_checks_say(code, text, monkeypatch):
    """A bad id is not told as a wait, nor the other way round."""
    class Fake:
        def hdc_device_error(self, reset):
            assert reset == 1
            return code

    monkeypatch.setattr(_lib, "load", Fake)
    monkeypatch.setattr(torch.cuda, "synchronize", lambda *a: None)
    with pytest.raises(_lib.HdcError, match=text):
        ops.check_device()
    runner = sp.SequenceParallel.__new__(sp.SequenceParallel)
    runner.k, runner.rank = sp.CudaKernels(), 3
    with pytest.raises(_lib.HdcError, match="rank 3.*" + text):
        runner.check()


@pytest.mark.gpu
def test_a_wait_is_not_hidden_by_a_bad_id():
    """A flag that nothing raises, waited for 20 ms, and an id outside a table: the wait is told first, the id by the
    next check."""
    ops.check_device()
    w = torch.zeros(10, 8, device="cuda")
    flags, gen = torch.zeros(32, dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
    for first in ("id", "wait"):
        def wait():
            rc = _lib.load().hdc_peer_wait_for(ctypes.c_void_p(flags.data_ptr()), 1, ctypes.c_void_p(gen.data_ptr()), 20_000_000,
                                               ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
            assert rc == 0

        if first == "wait":
            wait()
        ops.embedding(torch.tensor([1, 10], device="cuda"), w)
        if first == "id":
            wait()
        torch.cuda.synchronize()
        assert _lib.load().hdc_device_error(0) == 41  # looking at it takes nothing back
        with pytest.raises(_lib.HdcError, match="41"):
            ops.check_device()
        with pytest.raises(_lib.HdcError, match="71"):
            ops.check_device()
        ops.check_device()
