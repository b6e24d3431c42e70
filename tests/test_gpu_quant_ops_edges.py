"""The quantised, sampled decode's operators at the edges of what their documentation allows, against the definitions in 64 bits (tests/quant_refs.py) or against the same
call made the ordinary way."""
import numpy as np
import pytest
import torch

from tests import quant_refs as ref
from tests import test_gpu_quant_ops as ops
from tests.helpers import tiny_bart

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


# ---------------------------------------------------------------------------
# what a decoder keeps
# ---------------------------------------------------------------------------
def test_a_decoder_that_forgets_shapes_decodes_the_same():
    """more shapes than are kept: each decode equals that of a decoder which has seen no other, also one whose shape went and came back"""
    from seal_amd.quant_decoder import QuantStepDecoder
    model = tiny_bart(130, d_model=128, heads=2, max_positions=160).to(DEV)
    g = torch.Generator().manual_seed(17)
    dec = QuantStepDecoder(model)
    dec.MAX_STATES = 2

    def decode(d, B, S, T, plan=()):
        ids, mask, toks = inputs[B, S, T]
        d.start(d.encode(ids, mask), mask, 2, T, narrow_plan=plan)
        return [d.step(t).clone() for t in toks]
    inputs = {}
    shapes = [(1, 10, 8), (2, 70, 8), (3, 10, 70), (2, 10, 8)]
    for B, S, T in shapes:
        ids = torch.randint(4, 122, (B, S), generator=g).to(DEV)
        inputs[B, S, T] = ids, torch.ones_like(ids), [torch.randint(4, 122, (2 * B,), generator=g).to(DEV) for _ in range(6)]
    first = [decode(QuantStepDecoder(model), *s) for s in shapes]
    for _ in range(2):
        for s, want in zip(shapes, first):
            got = decode(dec, *s, plan=(1,) if s[0] > 1 else ())
            assert len(dec._states) <= 2
            assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("T,beams", [(64, 1), (64, 3), (128, 2)])
def test_a_mask_that_starts_between_words(T, beams):
    """a contiguous view at any byte, and rows cut out of a wider mask"""
    g = torch.Generator().manual_seed(T)
    S, H, D = 3, 2, 64
    c = ops._filled(S, H, T, D, 16, g)
    q = torch.randn(S * beams, H, D, generator=g).to(DEV)
    ln = torch.tensor([T, T - 7, 5], dtype=torch.int32, device=DEV)
    keep = (torch.rand(S, T, generator=g) < 0.5).to(DEV)
    want = c.attend(q, ln, beams=beams, keep=keep)
    for off in (1, 2, 3, 4):
        flat = torch.zeros(S * T + 4, dtype=torch.bool, device=DEV)
        view = flat[off:off + S * T].view(S, T)
        view.copy_(keep)
        assert view.is_contiguous() and torch.equal(c.attend(q, ln, beams=beams, keep=view), want)
    wide = torch.zeros(S, T + 5, dtype=torch.bool, device=DEV)
    wide[:, 3:3 + T] = keep
    assert torch.equal(c.attend(q, ln, beams=beams, keep=wide[:, 3:3 + T]), want)


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("K,N", [(256, 40), (1300, 40), (1300, 9000)])
def test_a_row_that_is_not_finite(K, N):
    """NaN: the whole row; an infinity: NaN in fp32, what inf * w sums to in bf16; the other rows stay"""
    from seal_amd.w4 import quantize_w4, w4_linear
    g = torch.Generator().manual_seed(K)
    w = quantize_w4(torch.randn(N, K, generator=g).to(DEV), 32)
    W = w.dequantize()
    for dt in (F32, BF16):
        x = torch.randn(20, K, generator=g).to(dt).to(DEV)
        want = w4_linear(x, w)
        x[3, 17], x[18, K - 1], x[19, 0], x[19, 5] = float("nan"), float("inf"), float("inf"), -float("inf")
        got = w4_linear(x, w)
        assert torch.equal(torch.cat([got[:3], got[4:18]]), torch.cat([want[:3], want[4:18]]))
        assert torch.isnan(got[3]).all()
        if dt == F32:
            assert torch.isnan(got[18:]).all()
        else:
            col = W[:, K - 1]
            assert torch.equal(torch.isnan(got[18]), col == 0)
            assert torch.equal(got[18][col != 0].float(), torch.sign(col[col != 0]) * float("inf"))
            a, b = torch.sign(W[:, 0]), -torch.sign(W[:, 5])
            both = (a != 0) & (a == b)
            assert torch.equal(torch.isnan(got[19]), ~both) and torch.equal(got[19][both].float(), a[both] * float("inf"))
