"""The host module belongs to the torch and the Python that it was compiled against: another one's is built again, and
refused where it would be loaded."""
import platform

import pytest
import torch

from hdcmamba_b200 import _lib, build


@pytest.mark.parametrize("what", ["torch", "python", "abi"])
def test_a_host_module_of_another_torch_or_python(what, monkeypatch):
    monkeypatch.setattr(build, "_deps", lambda: [])  # whatever the sources' times are
    assert build.up_to_date() and _lib.host() is not None
    monkeypatch.setattr(_lib, "_host", None)
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "0.9.1")
    elif what == "python":
        monkeypatch.setattr(platform, "python_version", lambda: "3.5.0")
    else:
        monkeypatch.setattr(torch._C, "_GLIBCXX_USE_CXX11_ABI", not torch._C._GLIBCXX_USE_CXX11_ABI)
    assert not build.up_to_date()
    with pytest.raises(OSError, match="build it with"):
        _lib.host()
