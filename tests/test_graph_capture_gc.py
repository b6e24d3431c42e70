"""No garbage collection inside a graph capture (``seal_amd.utils.captured``): a dead step decoder's graphs are only freed by the cyclic collector, and
freeing a graph while another one is captured ends the process.  On the CPU: the capture itself is replaced by a stand-in."""
import contextlib
import gc

import pytest
import torch

from seal_amd import bart_decoder, utils


class _Finalized:
    def __init__(self, log):
        self.log, self.me = log, self              # (a cycle: only the collector frees it)

    def __del__(self):
        self.log.append("freed")


@contextlib.contextmanager
def _capture(log):
    log.append("begin")
    try:
        yield
    finally:
        log.append("end")


@pytest.fixture
def log(monkeypatch):
    out = []
    monkeypatch.setattr(torch.cuda, "graph", lambda graph, **kw: _capture(out))
    old = gc.get_threshold()
    gc.set_threshold(1, 1, 1)                      # (as unlucky as it gets: a collection after every allocation)
    yield out
    gc.set_threshold(*old)


def test_a_capture_is_free_of_collections(log):
    gc.disable()
    _Finalized(log)                                # dead before the capture: freed before it begins
    gc.enable()
    with utils.captured(object()):
        _Finalized(log)                            # dies inside: waits
        keep = [[i] for i in range(1000)]
        assert not gc.isenabled() and log == ["freed", "begin"]
    del keep
    assert gc.isenabled()
    gc.collect()
    assert log == ["freed", "begin", "end", "freed"]


def test_the_collector_is_left_as_it_was(log):
    with pytest.raises(RuntimeError):
        with utils.captured(object()):
            raise RuntimeError("capture failed")
    assert gc.isenabled()
    gc.disable()
    try:
        with utils.captured(object()):
            pass
        assert not gc.isenabled()
    finally:
        gc.enable()


def test_the_decoder_captures_through_it():
    import inspect
    src = inspect.getsource(bart_decoder)
    assert "torch.cuda.graph(" not in src and src.count("with captured(") == 2
