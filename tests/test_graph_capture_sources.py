"""Every graph capture goes with the garbage collector held off: the package's own through ``seal_amd.utils.captured``, the tests' through the class that
tests/conftest.py puts in the place of ``torch.cuda.graph``."""
import gc
import glob
import os

import pytest
import torch

import seal_amd

ROOT = os.path.dirname(os.path.abspath(seal_amd.__file__))


def test_the_package_captures_in_one_place():
    found = {}
    for path in glob.glob(os.path.join(ROOT, "**", "*.py"), recursive=True):
        with open(path) as f:
            src = f.read()
        n = src.count("torch.cuda.graph(") - src.count("``torch.cuda.graph(")
        if n or "capture_begin" in src or "make_graphed_callables" in src:
            found[os.path.relpath(path, ROOT)] = n
    assert found == {"utils.py": 1}


@pytest.mark.parametrize("fails", [False, True], ids=["captured", "refused"])
def test_a_tests_own_capture_is_held(monkeypatch, fails):
    """``torch.cuda.graph`` as a test finds it; the class below it is replaced by a stand-in"""
    cls = torch.cuda.graph
    base = cls.__mro__[1]
    log = []

    def enter(self):
        log.append(("begin", gc.isenabled()))
        if fails:
            raise RuntimeError("no capture")

    def leave(self, *exc):
        log.append(("end", gc.isenabled()))
    monkeypatch.setattr(base, "__init__", lambda self, graph, **kw: None)
    monkeypatch.setattr(base, "__enter__", enter)
    monkeypatch.setattr(base, "__exit__", leave)
    assert gc.isenabled()
    if fails:
        with pytest.raises(RuntimeError):
            with torch.cuda.graph(object()):
                pass
        assert log == [("begin", False)]
    else:
        with torch.cuda.graph(object()):
            log.append(("inside", gc.isenabled()))
        assert log == [("begin", False), ("inside", False), ("end", False)]
    assert gc.isenabled()
