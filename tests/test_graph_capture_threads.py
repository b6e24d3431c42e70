"""Captures of two threads at once (``seal_amd.utils.captured``): the collector is one switch for the process, so the thread that ends first must not switch it on under
the other's capture.  On the CPU: the capture itself is replaced by a stand-in."""
import contextlib
import gc
import threading

import pytest
import torch

from seal_amd import utils


@contextlib.contextmanager
def _no_capture(graph, **kw):
    yield


@pytest.fixture(autouse=True)
def stand_in(monkeypatch):
    monkeypatch.setattr(torch.cuda, "graph", _no_capture)
    assert gc.isenabled()
    yield
    gc.enable()


def test_a_capture_that_ends_leaves_the_collector_off_under_another():
    seen, inside, go_on = [], threading.Event(), threading.Event()

    def first():
        with utils.captured(object()):
            inside.set()
            go_on.wait(10)

    def second():
        inside.wait(10)
        with utils.captured(object()):               # (begins while the first is captured, or after it)
            seen.append(gc.isenabled())
            threads[0].join(0.5)                     # the first ends, if it has not yet
            seen.append(gc.isenabled())
    threads = [threading.Thread(target=first), threading.Thread(target=second)]
    for t in threads:
        t.start()
    inside.wait(10)
    threads[1].join(0.2)                             # (the second is inside by now, or waits)
    go_on.set()
    for t in threads:
        t.join(20)
        assert not t.is_alive()
    assert seen == [False, False]
    assert gc.isenabled()


def test_a_capture_does_not_collect(monkeypatch):
    """neither under another thread's capture nor at all: a full collection is 50 ms and more in a process with many objects, and every new shape would pay it"""
    calls = []
    monkeypatch.setattr(gc, "collect", lambda *a: calls.append(a) or 0)
    with utils.captured(object()):
        pass
    assert not calls


def test_a_capture_inside_a_held_block_of_the_same_thread():
    with utils.collector_held():
        with utils.captured(object()):
            assert not gc.isenabled()
        assert not gc.isenabled()
    assert gc.isenabled()
