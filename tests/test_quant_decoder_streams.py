"""On which stream ``QuantStepDecoder`` captures its step.  No GPU: torch's streams and the capture are replaced by stand-ins."""
import contextlib

import torch

from seal_amd import quant_decoder
from seal_amd.quant_decoder import QuantStepDecoder


class _Stream:
    def __init__(self, device=None):
        self.device = torch.device(device) if device is not None else torch.device("cuda:0")

    def wait_stream(self, other):
        pass


def test_the_step_is_captured_on_a_stream_of_the_models_device(monkeypatch):
    """the model may be on another device than the current one (0): a capture on the current device's stream would not see the kernels, and its replays would do nothing"""
    made, seen, entered = [], [], []
    monkeypatch.setattr(torch.cuda, "Stream", lambda device=None: made.append(_Stream(device)) or made[-1])
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: _Stream(device))
    monkeypatch.setattr(torch.cuda, "CUDAGraph", object)

    @contextlib.contextmanager
    def stream(s):
        entered.append(s)
        yield

    @contextlib.contextmanager
    def captured(graph, stream=None, **kw):
        seen.append(stream)
        yield
    monkeypatch.setattr(torch.cuda, "stream", stream)
    monkeypatch.setattr(quant_decoder, "captured", captured)
    d = object.__new__(QuantStepDecoder)
    d._side = None
    d._forward = lambda st: st.t + 1
    for device in ("cuda:1", "cuda:1", "cuda:2"):
        st = QuantStepDecoder._State()
        st.t, st.lengths, st.graph = torch.zeros(1), torch.zeros(1), None
        d._capture(st, torch.device(device))
        assert st.graph is not None and seen[-1] is not None and seen[-1].device == torch.device(device) and entered[-1] is seen[-1]
    assert len(made) == 2                                  # (one stream for a device, not one for every shape)


def test_calls_on_another_stream_wait_for_the_one_before(monkeypatch):
    waits, now, capturing = [], [None], [False]

    class Stream:
        def __init__(self, name):
            self.name = name

        def wait_stream(self, other):
            waits.append((self.name, other.name))
    a, b = Stream("a"), Stream("b")
    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: now[0])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    d = object.__new__(QuantStepDecoder)
    d._last_stream = None
    for s in (a, a, b, b, a):
        now[0] = s
        d._in_order(torch.device("cuda:0"))
    assert waits == [("b", "a"), ("a", "b")]
    now[0], capturing[0] = b, True                         # (a wait for work outside a capture would end it)
    d._in_order(torch.device("cuda:0"))
    assert len(waits) == 2
