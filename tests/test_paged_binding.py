"""The C++ binding of the paged calls belongs to the torch it was built with (CPU)."""
import os
import sys

import pytest
import torch


@pytest.fixture
def P(monkeypatch):
    from bml_b200 import build
    build.build()
    import bml_b200.paged as P
    monkeypatch.setattr(P, "_fast", None)
    return P


def test_binding_of_this_torch_is_used(P):
    assert P._load().built_for == torch.__version__
    assert P._fast is not P._Wrappers


def test_binding_of_another_torch_is_not_used(P, monkeypatch):
    """Not one function of it is called, nor its addresses set."""
    from bml_b200 import _torch_calls
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    monkeypatch.setattr(_torch_calls, "set_calls", None)
    with pytest.warns(RuntimeWarning, match="0.0.1"):
        fast = P._load()
    assert fast is P._fast is P._Wrappers
    for call in (fast.plan, fast.append, fast.tree, fast.commit):
        assert call(1, 2, 3) is None
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="lens"):      # by the wrapper
        P.page_plan(i, i, i, i, i, i, 16, 4)


def test_missing_binding(P, monkeypatch):
    import bml_b200
    monkeypatch.delattr(bml_b200, "_torch_calls", raising=False)
    monkeypatch.setitem(sys.modules, "bml_b200._torch_calls", None)
    with pytest.warns(RuntimeWarning, match="ctypes"):
        assert P._load() is P._Wrappers


def test_build_sees_another_torch(P, monkeypatch):
    from bml_b200 import build
    assert not build.needs_build()
    with open(build.CALLS_FOR) as f:
        assert f.read() == torch.__version__
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    assert build.needs_build()


@pytest.mark.parametrize("why", ["torch", "compiler"])
def test_c_library_needs_neither_torch_nor_its_compiler(P, monkeypatch, tmp_path, why):
    """Then the binding is neither looked for nor built."""
    from bml_b200 import build
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "none.so"))
    monkeypatch.setattr(build, "_build_calls", lambda verbose: pytest.fail("built"))
    if why == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    else:
        monkeypatch.setenv("CXX", "no-such-compiler")
    assert not build.needs_build()
    # as after a change of a source: the C library alone
    newest = max(os.path.getmtime(f) for f in build.sources() + build.headers())
    monkeypatch.setattr(build, "needs_build", lambda: True)
    assert build.build() == build.LIB and os.path.getmtime(build.LIB) >= newest
