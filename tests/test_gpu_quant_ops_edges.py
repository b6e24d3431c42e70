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


def _tokens(v):
    """the cache's V, token by token: [slots, heads, T, dh] (a copy)"""
    S, H, n, D, _ = v.shape
    return v.view(S, H, n, D, 4, 4, 4).permute(0, 1, 2, 5, 4, 6, 3).reshape(S, H, n * 64, D)


def _tiles(v):
    S, H, T, D = v.shape
    return v.view(S, H, T // 64, 4, 4, 4, D).permute(0, 1, 2, 6, 4, 3, 5).reshape(S, H, T // 64, D, 64)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T,share,beams", [(64, 1, 1), (64, 1, 15), (64, 4, 1), (64, 1, 17), (128, 1, 1), (128, 1, 15)])
@pytest.mark.parametrize("block", [16, 64])
def test_attend_among_garbage(T, share, beams, block, D, dt):
    """caches as a decode that is not the first finds them, for every kernel of the attention: any codes, NaN among them, behind the lengths and under the mask, and scales that are NaN or
    infinite where a block has no token that counts"""
    g = torch.Generator().manual_seed(T + beams + share + block)
    S, H = 6, 2
    c = ops._filled(S, H, T, D, block, g, garbage=True)
    lengths = [0, 1, 16, 17, T - 1, T]
    keep = torch.rand(S, T, generator=g) < 0.6
    keep[1, 0] = True
    keep[4] = False                                       # nothing left
    keep[5, 16:32] = False
    live = keep & (torch.arange(T) < torch.tensor(lengths)[:, None])
    at = live[:, None, :, None].to(DEV)
    tame = lambda t: torch.where(at & ((t & 127) == 127), t - 1, t)  # noqa: E731
    c.k.copy_(tame(c.k))
    c.v.copy_(_tiles(tame(_tokens(c.v))))
    dead = ~live.view(S, T // block, block).any(-1)[:, None].expand(S, H, T // block).to(DEV)
    for t, bad in ((c.k_scale, float("nan")), (c.v_scale, float("inf"))):
        t.masked_fill_(dead, bad)
    assert bool(dead.any()) and bool(((c.k & 127) == 127).any()) and bool(((c.v & 127) == 127).any())
    q = (torch.randn(S * beams, H * share, D, generator=g) * 0.3).to(dt)
    k, v = ops._refs(c)
    with np.errstate(invalid="ignore"):
        kv, vv = k.values(), v.values()
    want, mag, vmax = ref.attend(q.double().numpy(), kv, vv, lengths, beams, keep.numpy())
    got = c.attend(q.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), beams=beams, keep=keep.to(DEV)).double().cpu().numpy()
    assert (np.abs(got - want) <= ops._attend_bound(mag, T, want, D, vmax, dt)).all()
    assert not got[:beams].any() and not got[4 * beams:5 * beams].any()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D", [64, 128])
def test_a_nan_among_the_tokens_of_one_tile_shows(D, dt):
    g = torch.Generator().manual_seed(5)
    for beams in (1, 3):
        c = ops._filled(3, 1, 64, D, 16, g)
        q, ln = torch.randn(3 * beams, 1, D, generator=g).to(dt).to(DEV), torch.tensor([40, 40, 40], dtype=torch.int32, device=DEV)
        want = c.attend(q, ln, beams=beams)
        c.k[1, 0, 20, D - 1] = 0x7f
        c.v[2, 0, 0, D - 1, ref.place(39)] = 0xff
        got = c.attend(q, ln, beams=beams)
        assert torch.equal(got[:beams], want[:beams]) and torch.isnan(got[beams:2 * beams]).all()
        assert torch.isnan(got[2 * beams:, :, D - 1]).all() and torch.equal(got[2 * beams:, :, :D - 1], want[2 * beams:, :, :D - 1])


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("D,block", [(64, 16), (128, 16), (64, 64), (128, 32)])
def test_append_of_one_token_with_counts_and_odd_values(D, block, dt):
    """the single-token kernel: slots that bring none, values that are not finite, zeros, scales that grow, lengths outside the cache; step by step, all buffers compared each time"""
    g = torch.Generator().manual_seed(D + block)
    S, H, T = 6, 3, 64
    c = ops._filled(S, H, T, D, block, g)
    k, v = ops._refs(c)
    lengths = torch.tensor([0, 14, 15, 30, 63, 7], dtype=torch.int32)
    odd = [0.0, float("inf"), -float("inf"), float("nan"), 448.0, 449.0, 1e-30, 1e30]
    for step in range(12):
        x = (torch.randn(S, 1, 2, H, D, generator=g) * 2.0 ** (2 * step - 8))
        counts = torch.randint(0, 2, (S,), generator=g).to(torch.int32)
        for s in range(S):
            for o in odd[step % 8:step % 8 + 3]:
                x[s, 0, int(torch.randint(0, 2, (1,), generator=g)), int(torch.randint(0, H, (1,), generator=g)), int(torch.randint(0, D, (1,), generator=g))] = o
        if step % 5 == 4:
            x[:] = 0
        if step == 6:
            x[2] = float("nan")
            x[3] = float("inf")
            counts[2:4] = 1
        if step == 9:
            counts = torch.tensor([7, -1, 1, 0, 1, 2], dtype=torch.int32)     # (never more than the token that is there)
        x = x.to(dt)
        c.append(x.to(DEV)[:, :, 0], x.to(DEV)[:, :, 1], lengths.to(DEV), None if step == 3 else counts.to(DEV))
        brought = torch.ones_like(counts) if step == 3 else counts.clamp(0, 1)
        k.append(x[:, :, 0].double().numpy(), lengths.tolist(), brought.tolist())
        v.append(x[:, :, 1].double().numpy(), lengths.tolist(), brought.tolist())
        ops._assert_same(c, k, v)
        lengths += brought
        lengths[4] = 63 if step % 2 else 64                # (full: dropped)
        if step == 7:
            lengths[0] = -1


@pytest.mark.parametrize("size", [1.0, 1e-36, 1e-38, 3e-39, 1e-40])
def test_weights_are_quantised_alike_on_the_gpu_and_multiply_with_tiny_scales(size):
    """scales below the smallest normal number: the same codes as on the CPU, and the product still applies them (fp32 has them as subnormals; x large enough that y is normal)"""
    from seal_amd.w4 import quantize_w4, w4_linear
    g = torch.Generator().manual_seed(8)
    w = (torch.rand(33, 300, generator=g) * 2 - 1) * size
    a, b = quantize_w4(w, 32), quantize_w4(w.to(DEV), 32)
    assert torch.equal(a.codes, b.codes.cpu()) and torch.equal(a.scales, b.scales.cpu())
    x = torch.randn(3, 300, generator=g) * (1 / size if size > 1e-38 else 1e36)
    W, X = a.dequantize().double().numpy(), x.double().numpy()
    want = X @ W.T
    got = w4_linear(x.to(DEV), b).double().cpu().numpy()
    assert (np.abs(got - want) <= ops._product_bound(X, W, want, 300, F32)).all()


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("V,rows", [(50, 1), (40000, 1), (40000, 70)])
def test_weights_below_the_unit_are_not_drawn(V, rows):
    """weights are multiples of 2^-44 of the largest: exp(-30.8) is one of them, exp(-31.3) is none, so that u = 0 falls on the first token of at least 2^-45; in each of the ways that a
    row is gone through (a list that one wave finishes, the whole row, rows spread over the card)"""
    from seal_amd.sampling import sample_tokens
    x = torch.full((rows, V), -200.0)
    x[:, V - 1] = 0.0
    x[:, 3], x[:, 7] = -31.3, -30.8
    u = torch.zeros(rows, 1)
    for kw in (dict(), dict(top_k=10), dict(top_k=600), dict(top_p=1 - 2.0 ** -24), dict(min_p=2.0 ** -46)):
        tok, lp = sample_tokens(x.to(DEV), u.to(DEV), **kw)
        want = V - 1 if "top_p" in kw else 7               # (the nucleus is the largest alone: it holds 1 - 2^-44 of the weight)
        assert (tok == want).all(), kw
        assert torch.allclose(lp.cpu(), x[:, want:want + 1], atol=1e-5)
    x[:, 7] = -31.3
    assert (sample_tokens(x.to(DEV), u.to(DEV))[0] == V - 1).all()


def test_decodes_of_one_decoder_on_several_streams():
    """a decode right behind another of the same shape (the same buffers and graph) on another stream, and one that changes streams on its way, without a wait between them: each is what
    it is alone"""
    from seal_amd.quant_decoder import QuantStepDecoder
    model = tiny_bart(130, d_model=128, heads=2, max_positions=160).to(DEV)
    g = torch.Generator().manual_seed(23)
    B, S, T = 2, 90, 12
    work = []
    for _ in range(4):
        ids = torch.randint(4, 122, (B, S), generator=g).to(DEV)
        work.append((ids, torch.ones_like(ids), [torch.randint(4, 122, (2 * B,), generator=g).to(DEV) for _ in range(T)]))
    order = torch.tensor([1, 0, 3, 3], device=DEV)
    for graph in (True, False):
        dec = QuantStepDecoder(model)
        dec.use_graph = graph
        enc = [dec.encode(ids, mask) for ids, mask, _ in work]

        def decode(i, streams):
            ids, mask, toks = work[i]
            out = []
            with torch.cuda.stream(streams[0]):
                dec.start(enc[i], mask, 2, T)
            for t in range(T):
                with torch.cuda.stream(streams[t % len(streams)]):
                    out.append(dec.step(toks[t]).clone())
                if t == 5:
                    with torch.cuda.stream(streams[-1]):
                        dec.reorder(order)
            return out
        here = torch.cuda.current_stream()
        want = [decode(i, [here]) for i in range(4)]
        torch.cuda.synchronize()
        a, b, c = (torch.cuda.Stream() for _ in range(3))
        for _ in range(3):
            with torch.cuda.stream(a):
                torch.cuda._sleep(20_000_000)              # (the first decode is still to come when the others are given out)
            got = [decode(0, [a]), decode(1, [b]), decode(2, [a, b, c]), decode(3, [c])]
            torch.cuda.synchronize()
            for x, y in zip(got, want):
                assert all(torch.equal(p, q) for p, q in zip(x, y))
