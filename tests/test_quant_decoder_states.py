"""What ``QuantStepDecoder`` keeps between decodes is bounded: the least recently used shapes go, the one that is about to run never does.  (CPU: the bookkeeping; the
decodes themselves are in tests/test_gpu_quant_ops_edges.py.)"""
from collections import OrderedDict

import torch

from seal_amd.quant_decoder import QuantStepDecoder


def _decoder(**limits):
    d = object.__new__(QuantStepDecoder)
    d.layers, d.h, d.dh, d.block, d.lm_w = [None] * 12, 16, 64, 16, torch.zeros(50265, 1)
    d._states = OrderedDict()
    for k, v in limits.items():
        setattr(d, k, v)
    return d


def _use(d, key, tails=()):
    d._make_room(key, torch.device("cpu"))
    st = d._states.get(key)
    if st is None:
        st = d._states[key] = QuantStepDecoder._State()
        st.tails = {}
    d._states.move_to_end(key)
    for t in tails:
        st.tails[t] = None


def test_bytes_of_a_shape_are_those_of_its_buffers():
    from seal_amd.kv8 import KV8Cache
    d = _decoder()
    B, K, S, T = 3, 5, 128, 64
    caches = [KV8Cache.empty(n, d.h, t, d.dh, block=d.block, device="cpu") for n, t in ((B * K, T), (B, S))]
    want = 12 * sum(t.numel() * t.element_size() for c in caches for t in (c.k, c.v, c.k_scale, c.v_scale))
    assert d._state_bytes((B, K, S, T), tails=(1, 2)) == want + 4 * 50265 * K * (3 + 2 + 1)


def test_the_shapes_that_are_kept_are_bounded_in_number():
    d = _decoder(MAX_STATES=4)
    for i in range(1, 20):
        _use(d, (i, 1, 64, 64))
        assert len(d._states) <= 4 and (i, 1, 64, 64) in d._states
    assert list(d._states) == [(i, 1, 64, 64) for i in (16, 17, 18, 19)]
    _use(d, (16, 1, 64, 64))                     # used again: the next to go is 17
    _use(d, (20, 1, 64, 64))
    assert list(d._states) == [(i, 1, 64, 64) for i in (18, 19, 16, 20)]


def test_the_shapes_that_are_kept_are_bounded_in_bytes():
    d = _decoder()
    long = (20, 15, 1024, 1024)                  # 300 rows of 1024 positions: 8 GB
    assert 7e9 < d._state_bytes(long) < 9e9
    _use(d, long, tails=(5, 10))
    for i in range(1, 21):
        _use(d, (i, 15, 1024, 1024))
        assert sum(d._state_bytes(k, st.tails) for k, st in d._states.items()) <= d.STATE_BYTES
    big = (60, 15, 1024, 1024)                   # more than the limit by itself: alone
    _use(d, big)
    assert list(d._states) == [big]
    _use(d, (1, 1, 64, 64))
    assert list(d._states) == [(1, 1, 64, 64)]
