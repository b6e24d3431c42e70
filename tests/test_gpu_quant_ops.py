"""The quantised, sampled decode's kernels (sealnn_w4_linear, sealnn_kv8_append, sealnn_kv8_attend, sealnn_sample_tokens) against their definitions
in 64 bits (tests/quant_refs.py), where they can go wrong: sizes around the tiles, strides and alignment, empty rows, masks, values that are not
finite, ties, ragged and dropped tokens, graphs, other streams."""
import numpy as np
import pytest
import torch

from seal_amd.kv8 import KV8Cache
from seal_amd.sampling import sample_tokens
from seal_amd.w4 import quantize_w4, w4_linear
from tests import quant_refs as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16
U32 = 2.0 ** -24                                    # half a step of fp32, relative
U16 = 2.0 ** -8                                     # ... of bf16


def _half_step(dt):
    return U32 if dt == F32 else U16


def _replayed(call, change, times=3):
    """``call()`` captured once and replayed with other inputs (``change(i)``), eager work in between: [(replay's outputs, eager outputs)]"""
    change(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = call()
    got = []
    for i in range(times):
        change(i)
        g.replay()
        torch.cuda.synchronize()
        a = [t.clone() for t in out]
        torch.randn(1000, device=DEV).sum().item()
        change(i)
        got.append((a, [t.clone() for t in call()]))
        torch.cuda.synchronize()
    return got


# ---------------------------------------------------------------------------
# products
# ---------------------------------------------------------------------------
def _product_bound(x, w, y, K, dt):
    """Every term is exact (bf16 x e2m1 in the matrix unit); an output is a sum of at most 3 K of them (three planes) and of K / 32 scaled partial sums,
    each addition and scaling off by half a step of a partial sum that is at most sum |x w|; then the bias and the store."""
    return (3 * K + K / 32 + 64) * U32 * (np.abs(x) @ np.abs(w).T) + 4 * U32 * np.abs(y) + _half_step(dt) * np.abs(y) + 1e-30


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("M,N,K,group", [(1, 16, 128, 32), (1, 1, 1, 32), (1, 50, 7, 64), (2, 33, 129, 128), (3, 64, 256, 64), (15, 100, 1000, 32), (16, 48, 1024, 128),
                                         (17, 1000, 384, 32), (33, 17, 640, 64), (60, 96, 1030, 32), (64, 31, 128, 128), (65, 40, 260, 64), (130, 16, 512, 32),
                                         (1, 20000, 96, 64), (5, 300, 4096, 32), (2, 50265, 640, 64), (40, 50000, 500, 32), (17, 9000, 130, 128), (70, 8200, 65, 32),
                                         (3, 17000, 1100, 64), (40, 8200, 1500, 128)])
def test_product(M, N, K, group, dt):
    g = torch.Generator().manual_seed(M * 7 + N * 3 + K)
    w = quantize_w4(torch.randn(N, K, generator=g), group)
    x = (torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-6, 6, (M, K), generator=g).float())).to(dt)
    b = torch.randn(N, generator=g).to(dt)
    W = w.dequantize().double().numpy()
    if N * K <= 20000:
        assert np.array_equal(W, ref.w4_values(w.codes.numpy(), w.scales.float().numpy(), N, K))
    xd = x.double().numpy()
    wd = type(w)(w.codes.to(DEV), w.scales.to(DEV), N, K)
    for bias in (None, b):
        want = xd @ W.T + (0 if bias is None else bias.double().numpy())
        tol = _product_bound(xd, W, np.abs(want) + (0 if bias is None else np.abs(bias.double().numpy())), K, dt)
        got = w4_linear(x.to(DEV), wd, None if bias is None else bias.to(DEV))
        assert got.dtype == dt and got.shape == (M, N)
        assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
    # gelu'(y) <= 1.13; erff is good to 4 steps of 1 + erf <= 2, and the two products of the formula round once each
    from math import erfc
    act = np.vectorize(lambda t: 0.5 * t * erfc(-t / 2 ** 0.5))(want)
    got = w4_linear(x.to(DEV), wd, b.to(DEV), gelu=True).double().cpu().numpy()
    assert (np.abs(got - act) <= 1.13 * tol + 16 * U32 * np.abs(want) + _half_step(dt) * np.abs(act)).all()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_product_of_strided_and_misaligned_rows(dt):
    g = torch.Generator().manual_seed(3)
    M, N, K = 9, 70, 200
    w = quantize_w4(torch.randn(N, K, generator=g).to(DEV), 64)
    big = torch.randn(M, 3 * K + 5, generator=g).to(dt).to(DEV)
    for off in (0, 1, 3, 8):
        x = big[:, off:off + K]
        assert torch.equal(w4_linear(x, w), w4_linear(x.contiguous(), w))
    row = big[2:3, 1:1 + K]
    assert torch.equal(w4_linear(row, w), w4_linear(row.contiguous(), w))
    assert w4_linear(big[:0, :K], w).shape == (0, N)


def test_a_non_finite_row_stays_alone():
    g = torch.Generator().manual_seed(4)
    w = quantize_w4(torch.randn(40, 256, generator=g).to(DEV), 32)
    x = torch.randn(20, 256, generator=g).to(DEV)
    want = w4_linear(x, w)
    x[3, 17], x[18, 255] = float("nan"), float("inf")
    got = w4_linear(x, w)
    assert torch.isnan(got[[3, 18]]).all()
    rest = [i for i in range(20) if i not in (3, 18)]
    assert torch.equal(got[rest], want[rest])


# ---------------------------------------------------------------------------
# the cache
# ---------------------------------------------------------------------------
def _filled(S, H, T, D, block, g, garbage=False):
    """a cache of random codes (NaN codes too with ``garbage``) and scales, and its reference"""
    c = KV8Cache.empty(S, H, T, D, block=block, device=DEV)
    for t in (c.k, c.v):
        u = torch.randint(0, 256, t.shape, generator=g, dtype=torch.int64).to(torch.uint8)
        if not garbage:
            u = torch.where((u & 127) == 127, u - 1, u)
        t.copy_(u)
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp2(torch.randint(-12, -4, t.shape, generator=g).float()))
    return c


def _refs(c):
    S, H, T, D = c.k.shape
    v = c.v.cpu().view(torch.float8_e4m3fn).double().numpy()
    tok = np.array([ref.place(t) for t in range(64)])
    v = v[..., tok].transpose(0, 1, 2, 4, 3).reshape(S, H, T, D)
    return (ref.Cache(c.k.cpu().view(torch.float8_e4m3fn).double().numpy(), c.k_scale.cpu().numpy(), c.block), ref.Cache(v, c.v_scale.cpu().numpy(), c.block))


def _assert_same(c, k, v):
    gk, gv = _refs(c)
    for got, want in ((gk, k), (gv, v)):
        assert np.array_equal(got.scale, want.scale)
        assert np.array_equal(got.codes, want.codes, equal_nan=True)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("S,H,T,D,block,n,lengths", [(1, 1, 64, 64, 16, 1, [0]), (3, 2, 128, 64, 16, 1, [15, 16, 63]), (2, 3, 128, 128, 64, 1, [64, 100]), (4, 1, 64, 64, 32, 2, [0, 31, 32, 63]),
                                                     (2, 2, 192, 64, 16, 65, [0, 7]), (2, 2, 256, 128, 32, 130, [1, 63]), (3, 2, 128, 64, 64, 128, [0, 1, 127]), (2, 1, 64, 64, 16, 200, [0, 10]),
                                                     (3, 1, 64, 64, 16, 1, [64, -1, 70])])
def test_append(S, H, T, D, block, n, lengths, dt):
    g = torch.Generator().manual_seed(S * 100 + n + T)
    c = _filled(S, H, T, D, block, g)
    k, v = _refs(c)
    qkv = (torch.randn(S, n, 3, H, D, generator=g) * torch.exp2(torch.randint(-8, 9, (S, n, 1, H, 1), generator=g).float())).to(dt)
    ln = torch.tensor(lengths, dtype=torch.int32)
    c.append(qkv.to(DEV)[:, :, 1], qkv.to(DEV)[:, :, 2], ln.to(DEV))
    k.append(qkv[:, :, 1].double().numpy(), lengths)
    v.append(qkv[:, :, 2].double().numpy(), lengths)
    _assert_same(c, k, v)


def test_append_ragged_then_token_by_token():
    g = torch.Generator().manual_seed(11)
    S, H, T, D = 5, 2, 192, 64
    c = KV8Cache.empty(S, H, T, D, block=16, device=DEV)
    k, v = _refs(c)
    new = torch.randn(S, 70, H, D, generator=g)
    counts = [0, 1, 37, 70, 64]
    lengths = torch.zeros(S, dtype=torch.int32)
    c.append(new.to(DEV), (2 * new).to(DEV), lengths.to(DEV), torch.tensor(counts, dtype=torch.int32, device=DEV))
    k.append(new.double().numpy(), [0] * S, counts)
    v.append(2 * new.double().numpy(), [0] * S, counts)
    _assert_same(c, k, v)
    lengths = torch.tensor(counts, dtype=torch.int32)
    for step in range(20):
        x = torch.randn(S, 1, H, D, generator=g) * 2.0 ** (step % 7 - 3)
        c.append(x.to(DEV), (x * 3).to(DEV), lengths.to(DEV))
        k.append(x.double().numpy(), lengths.tolist())
        v.append(3 * x.double().numpy(), lengths.tolist())
        lengths += 1
    _assert_same(c, k, v)
    kv, vv = c.values()
    assert np.array_equal(kv.transpose(1, 2).double().cpu().numpy(), k.values()) and np.array_equal(vv.transpose(1, 2).double().cpu().numpy(), v.values())


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_append_of_odd_values_and_strides(dt):
    """zeros, values at the border of a scale, infinities and NaN, tiny and huge magnitudes; rows whose pointers are only element-aligned; both halves of a tile
    written in two calls"""
    g = torch.Generator().manual_seed(12)
    S, H, T, D = 2, 1, 64, 64
    c = KV8Cache.empty(S, H, T, D, block=16, device=DEV)
    k, v = _refs(c)
    wide = torch.randn(S, 48, H, D + 3, generator=g).to(dt)
    wide[0, 0:16] = 0
    wide[0, 16, 0, 5], wide[0, 17, 0, 6], wide[0, 18, 0, 7] = float("inf"), float("-inf"), float("nan")
    wide[0, 32:48] = 0
    wide[0, 33, 0, 9] = 448.0
    wide[1, 0:16] *= 1e-30
    wide[1, 16:32] *= 1e30
    wide[1, 32, 0, 1:] = 449.0 if dt == F32 else 450.0
    new = wide[..., 1:D + 1]
    dev = wide.to(DEV)[..., 1:D + 1]
    for a, b in ((0, 20), (20, 48)):
        at = torch.full((S,), a, dtype=torch.int32)
        c.append(dev[:, a:b], dev[:, a:b], at.to(DEV))
        k.append(new[:, a:b].double().numpy(), at.tolist())
        v.append(new[:, a:b].double().numpy(), at.tolist())
    _assert_same(c, k, v)


def _attend_bound(mag, n, out, dh, vmax, dt):
    """A score is a sum of 3 dh exact products (three planes), scaled twice: off by (3 dh + 4) half steps of sum |q k| scale; its exponent rounds once more, twice with
    the maximum's, and exp2 is good to two steps: the relative error of a weight is twice that (the maximum's score is off as well).  Numerator and
    denominator carry it once each; a sum of n weights of three (two) planes adds 3 n half steps of the largest value, the joining of parts and
    the division a few more.  bf16: the weights keep 16 bits, and the result is stored in bf16."""
    w = 2 * ((3 * dh + 8) * U32 * mag * 1.4427 + 8 * U32)
    return ((2 * w + (3 * n + 64) * U32 + (2.0 ** -15 if dt == BF16 else 0)) * vmax)[..., None] + _half_step(dt) * np.abs(out) + 1e-30


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("S,H,share,beams,T,D,block,lengths", [(1, 1, 1, 1, 64, 64, 16, [1]), (3, 2, 1, 1, 64, 64, 16, [0, 17, 64]), (4, 1, 1, 15, 64, 64, 32, [1, 12, 30, 0]), (2, 3, 1, 16, 128, 64, 64, [65, 128]),
                                                               (2, 2, 1, 17, 128, 64, 16, [63, 127]), (2, 2, 4, 1, 320, 128, 64, [319, 5]), (1, 2, 8, 3, 256, 64, 32, [200]), (1, 1, 1, 1, 4096, 64, 64, [4001]),
                                                               (2, 1, 2, 1, 2048, 128, 16, [2048, 0]), (1, 1, 1, 33, 512, 64, 16, [300]), (2, 1, 1, 1, 64, 64, 16, [-3, 200])])
@pytest.mark.parametrize("masked", [False, True], ids=["all", "masked"])
def test_attend(S, H, share, beams, T, D, block, lengths, dt, masked):
    g = torch.Generator().manual_seed(T + S * 10 + beams)
    c = _filled(S, H, T, D, block, g)
    q = (torch.randn(S * beams, H * share, D, generator=g) * 0.3).to(dt)
    keep = None
    if masked:
        keep = torch.rand(S, T, generator=g) < 0.6
        keep[0] = False                                   # a row with nothing left
    k, v = _refs(c)
    want, mag, vmax = ref.attend(q.double().numpy(), k.values(), v.values(), lengths, beams, None if keep is None else keep.numpy())
    got = c.attend(q.to(DEV), torch.tensor(lengths, dtype=torch.int32, device=DEV), beams=beams, keep=None if keep is None else keep.to(DEV))
    assert got.dtype == dt and got.shape == q.shape
    got = got.double().cpu().numpy()
    n = np.array([min(max(x, 0), T) for x in lengths]).max()
    assert (np.abs(got - want) <= _attend_bound(mag, n, want, D, vmax, dt)).all(), np.abs(got - want).max()
    if masked:
        assert not got[:beams].any()


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_attend_ignores_what_is_masked_or_behind(dt):
    """NaN codes and infinite or NaN scales in masked places and behind a slot's length change nothing"""
    g = torch.Generator().manual_seed(21)
    S, H, T, D, beams = 3, 2, 192, 64, 2
    c = _filled(S, H, T, D, 16, g)
    q = torch.randn(S * beams, H, D, generator=g).to(dt).to(DEV)
    ln = torch.tensor([1, 100, 192], dtype=torch.int32, device=DEV)
    keep = torch.rand(S, T, generator=g).to(DEV) < 0.5
    keep[0, 0] = True
    keep[2, 32:48] = False
    want = c.attend(q, ln, beams=beams, keep=keep)
    there = keep & (torch.arange(T, device=DEV) < ln[:, None])
    c.k.masked_fill_(~there[:, None, :, None], 0x7f)
    v = c.v.view(S, H, T // 64, D, 4, 4, 4).permute(0, 1, 2, 5, 4, 6, 3).reshape(S, H, T, D).masked_fill(~there[:, None, :, None], 0x7f)
    c.v.copy_(v.view(S, H, T // 64, 4, 4, 4, D).permute(0, 1, 2, 6, 4, 3, 5).reshape(c.v.shape))
    for t, bad in ((c.k_scale, float("nan")), (c.v_scale, float("inf"))):
        t[2, :, 2] = bad                                  # (the block whose tokens are all masked)
        t[0, :, 1:] = bad
        t[1, :, 7:] = bad
    assert torch.equal(c.attend(q, ln, beams=beams, keep=keep), want)
    assert torch.equal(c.attend(q, ln, beams=beams, keep=keep.to(torch.uint8) * 200), want)


def test_attend_shows_a_nan_that_counts():
    g = torch.Generator().manual_seed(22)
    c = _filled(2, 1, 1024, 64, 16, g)
    q, ln = torch.randn(2, 1, 64, generator=g).to(DEV), torch.tensor([1000, 1000], dtype=torch.int32, device=DEV)
    want = c.attend(q, ln)
    c.k[1, 0, 500, 3] = 0x7f
    got = c.attend(q, ln)
    assert torch.isnan(got[1]).all() and torch.equal(got[0], want[0])


def test_attend_strided_queries_scale_and_parts():
    """q as a part of a fused projection and with rows of an odd stride; a scale of one's own; the same slots in one part and in many agree to the bound"""
    g = torch.Generator().manual_seed(23)
    S, H, T, D, beams = 2, 4, 1024, 64, 3
    c = _filled(S, H, T, D, 32, g)
    ln = torch.tensor([1024, 333], dtype=torch.int32, device=DEV)
    wide = torch.randn(S * beams, 3 * H * D + 1, generator=g).to(DEV) * 0.3
    q = wide[:, 1:1 + H * D].unflatten(1, (H, D))
    want = c.attend(q.contiguous(), ln, beams=beams)
    assert torch.equal(c.attend(q, ln, beams=beams), want)
    half = c.attend(q * 2, ln, beams=beams, scale=D ** -0.5 / 2)
    assert torch.equal(half, want)                        # (a power of two moves nothing)
    k, v = _refs(c)
    exact, mag, vmax = ref.attend(q.double().cpu().numpy(), k.values(), v.values(), ln.tolist(), beams)
    from seal_amd import kv8
    for wanted in (1, 1 << 14):
        old, kv8.PARTS_WANTED = kv8.PARTS_WANTED, wanted
        try:
            got = c.attend(q, ln, beams=beams).double().cpu().numpy()
        finally:
            kv8.PARTS_WANTED = old
        assert (np.abs(got - exact) <= _attend_bound(mag, T, exact, D, vmax, F32)).all()


def test_a_cache_of_more_than_four_billion_codes():
    """offsets that pass 32 bits: the last slots of a large cache, written and read"""
    S, H, T, D = 33, 16, 131072, 64                       # 4.4 GB of keys, as much of values
    c = KV8Cache.empty(S, H, T, D, block=64, device=DEV)
    g = torch.Generator().manual_seed(31)
    n = 100
    new = torch.randn(S, n, H, D, generator=g)
    at = torch.full((S,), T - 80, dtype=torch.int32)
    c.append(new.to(DEV), (new * 2).to(DEV), at.to(DEV))
    lo = (T - 80) // 64 * 64
    k = ref.Cache(np.zeros((1, H, 128, D)), np.full((1, H, 2), 2.0 ** -64), 64)
    v = ref.Cache(np.zeros((1, H, 128, D)), np.full((1, H, 2), 2.0 ** -64), 64)
    k.append(new[-1:].double().numpy(), [T - 80 - lo])
    v.append(2 * new[-1:].double().numpy(), [T - 80 - lo])
    assert np.array_equal(c.k[-1, :, lo:].cpu().view(torch.float8_e4m3fn).double().numpy(), k.codes[0])
    tail = KV8Cache(c.k[-1:, :, lo:].contiguous(), c.v[-1:, :, lo // 64:].contiguous(), c.k_scale[-1:, :, lo // 64:].contiguous(), c.v_scale[-1:, :, lo // 64:].contiguous())
    assert np.array_equal(tail.values()[1].transpose(1, 2).double().cpu().numpy(), v.values())
    q = torch.randn(S, H, D, generator=g)
    keep = torch.zeros(S, T, dtype=torch.bool, device=DEV)
    keep[:, T - 80:] = True
    got = c.attend(q.to(DEV), torch.full((S,), T, dtype=torch.int32, device=DEV), keep=keep)[-1:].double().cpu().numpy()
    kp = np.zeros((1, 128), dtype=bool)
    kp[0, T - 80 - lo:] = True
    want, mag, vmax = ref.attend(q[-1:].double().numpy(), k.values(), v.values(), [128], 1, kp)
    assert (np.abs(got - want) <= _attend_bound(mag, 128, want, D, vmax, F32)).all()


# ---------------------------------------------------------------------------
# sampling
# ---------------------------------------------------------------------------
def _pack(ok):
    w = torch.zeros(ok.shape[0], -(-ok.shape[1] // 32) * 32, dtype=torch.int64)
    w[:, :ok.shape[1]] = ok
    w = (w.view(ok.shape[0], -1, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _check_samples(logits, u, allowed=None, **kw):
    """tokens: equal.  Log-probabilities: a term of the sum is exp2 of a rounded product of a rounded difference (two half steps of the exponent, at most 1.45 x the gap),
    exp2 itself two steps; adding them up 1 + vocab / 1024 + 6 half steps; then the store."""
    bits = None if allowed is None else _pack(allowed).to(DEV)
    dkw = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    tok, lp = sample_tokens(logits.to(DEV), u.to(DEV), allowed_bits=bits, **dkw)
    assert tok.shape == u.shape == lp.shape and tok.dtype == torch.int64 and lp.dtype == F32
    tok, lp = tok.cpu().numpy().reshape(len(u), -1), lp.cpu().numpy().reshape(len(u), -1)
    x = logits.float().numpy()
    for r in range(len(u)):
        row = {k: (v[r].item() if isinstance(v, torch.Tensor) else v) for k, v in kw.items()}
        want, wl = ref.sample(x[r], u[r].numpy(), allowed=None if allowed is None else allowed[r].numpy(), **row)
        assert np.array_equal(tok[r], want), (r, tok[r], want)
        fin = x[r][np.isfinite(x[r])]
        gap = float(fin.max() - fin.min()) if fin.size else 0.0
        tol = (4 * min(gap, 120.0) + 16 + x.shape[1] / 1024) * U32 + U32 * np.abs(np.where(np.isfinite(wl), wl, 0))
        assert np.array_equal(np.isfinite(lp[r]), np.isfinite(wl)) and (np.abs(lp[r] - wl)[np.isfinite(wl)] <= (tol if np.ndim(tol) == 0 else tol[np.isfinite(wl)])).all()
    return tok


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("R,V", [(1, 1), (3, 2), (2, 31), (5, 80), (2, 1023), (3, 4096), (2, 4097), (4, 50265), (2, 65537), (1, 131072), (1, 262144)])
def test_sample_sizes_and_filters(R, V, dt):
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(R, V, generator=g) * 3).to(dt)
    u = torch.rand(R, 5, generator=g)
    allowed = torch.rand(R, V, generator=g) < 0.4
    allowed[0, V - 1] = True
    for kw in (dict(), dict(temperature=0.6), dict(top_k=3), dict(top_k=40, temperature=1.3), dict(top_p=0.9), dict(top_p=0.3, temperature=2.0), dict(min_p=0.05),
               dict(top_k=500, top_p=0.8, min_p=0.01, temperature=0.9), dict(temperature=0.0), dict(top_p=0.0), dict(top_k=1), dict(min_p=1.0)):
        _check_samples(logits, u, **kw)
        _check_samples(logits, u, allowed=allowed, **kw)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
def test_sample_ties(dt):
    """equal logits: all of them, a few levels, and a border inside a group of equals: the lower index stays"""
    g = torch.Generator().manual_seed(2)
    V = 5000
    flat = torch.zeros(1, V)
    steps = torch.randint(0, 6, (1, V), generator=g).float()
    signs = torch.where(torch.rand(1, V, generator=g) < 0.5, 0.0, -0.0)          # +0 and -0 are equal
    u = torch.rand(1, 64, generator=g)
    u[0, 0], u[0, 1], u[0, 2] = 0.0, 1 - 2.0 ** -24, 2.0 ** -40
    for x in (flat, steps, signs, -steps * 1e30):
        for kw in (dict(), dict(top_k=7), dict(top_k=4096), dict(top_p=0.5), dict(top_k=100, top_p=0.25), dict(top_p=0.999, top_k=4999), dict(temperature=0.0), dict(min_p=0.5)):
            _check_samples(x.to(dt), u, **kw)


@pytest.mark.parametrize("dt", [F32, BF16], ids=["fp32", "bf16"])
@pytest.mark.parametrize("V", [32768, 40001, 262144])
def test_sample_spread_over_the_card_draws_the_same_tokens(V, dt, monkeypatch):
    """the three kernels of few rows of a large vocabulary against the one of many, where the lists of the largest tokens are the hardest to make: all in one
    place, in every last place, none but a few allowed, all alike, a handful of values, nearly no spread"""
    g = torch.Generator().manual_seed(V)
    rows = [torch.randn(V, generator=g) * 3 for _ in range(7)]
    rows[1][:1500] += 30
    rows[2][1023::1024] += 12
    rows[3][:] = -2.5
    rows[4] = torch.randint(0, 3, (V,), generator=g).float()
    rows[5] = rows[5] * 1e-3
    rows[6][torch.randperm(V, generator=g)[20:]] = -float("inf")
    x = torch.stack(rows).to(dt).to(DEV)
    u = torch.rand(len(rows), 9, generator=g).to(DEV)
    few = torch.rand(len(rows), V, generator=g) < 2e-3
    few[5, 1:] = False
    few[5, 0] = True
    own = dict(temperature=torch.tensor([1.0, 0.5, 0.0, 1.3, 0.8, 2.0, 1.0], device=DEV), top_k=torch.tensor([0, 513, 5, 0, 40, -1, 512], dtype=torch.int32, device=DEV),
               top_p=torch.tensor([1.0, 0.9, 0.2, 0.6, 0.95, 1.0, 0.0], device=DEV), min_p=torch.tensor([0.0, 0.0, 0.5, 0.1, 0.01, 0.02, 0.0], device=DEV))
    for bits in (None, _pack(few).to(DEV)):
        for kw in (dict(), dict(min_p=0.1), dict(top_p=0.9), dict(top_p=0.999, temperature=1.4), dict(top_k=1), dict(top_k=60), dict(top_k=512, top_p=0.7), dict(top_k=513),
                   dict(top_k=V - 1, top_p=0.5, min_p=0.001), dict(temperature=0.0), own):
            monkeypatch.undo()
            spread = sample_tokens(x, u, allowed_bits=bits, **kw)
            monkeypatch.setattr("seal_amd.sampling.SPLIT_ROWS", 0)
            one = sample_tokens(x, u, allowed_bits=bits, **kw)
            assert torch.equal(spread[0], one[0]), kw
            # (each within its own bound, see _check_samples: twice 4 x 120 gaps, 16 and the adding up)
            assert torch.allclose(spread[1], one[1], rtol=2 * U32, atol=2 * (4 * 120 + 16 + V / 1024) * U32), kw


def test_sample_values_that_are_not_finite():
    inf, nan = float("inf"), float("nan")
    V = 300
    x = torch.randn(8, V, generator=torch.Generator().manual_seed(5))
    x[0] = -inf                                            # nothing can be drawn
    x[1, :], x[1, 7] = -inf, 2.0
    x[2, 5] = nan
    x[3, 9], x[3, 200] = inf, inf
    x[4] = torch.finfo(F32).min                            # masks of the type's lowest value: all equal
    x[5, 1:] = torch.finfo(F32).min
    x[6] = nan
    x[7, ::2], x[7, 1::2] = -3e38, 3e38
    u = torch.rand(8, 9, generator=torch.Generator().manual_seed(6))
    for kw in (dict(), dict(top_k=2), dict(top_p=0.7), dict(top_k=200, top_p=0.9, min_p=0.1, temperature=0.5), dict(temperature=0.0)):
        tok = _check_samples(x, u, **kw)
        assert (tok[[0, 6]] == -1).all() and (tok[1] == 7).all() and set(tok[3]) <= {9, 200}
    none = torch.ones(8, V, dtype=torch.bool)
    none[2:4] = False
    assert (_check_samples(x, u, allowed=none, top_p=0.5)[2:4] == -1).all()


@pytest.mark.parametrize("V", [20000, 40000])
def test_sample_values_that_are_not_finite_in_long_rows(V):
    """the same in rows of several turns, and numbers beyond 1e30 of either sign"""
    g = torch.Generator().manual_seed(V)
    x = torch.randn(8, V, generator=g) * 3
    x[0, ::777] = float("nan")
    x[1, [17, V - 2]] = float("inf")
    x[2, :] = -float("inf")
    x[2, [3, 9000, V - 1]] = torch.tensor([0.5, 1.0, 0.25])
    x[3] = -2e30 + x[3] * 1e28
    x[4, 12345] = 2e30
    x[5, ::2] = -float("inf")
    x[6, :] = float("nan")
    x[6, 8191] = 2.0
    x[7, :] = float("nan")
    u = torch.rand(8, 3, generator=g)
    allowed = torch.rand(8, V, generator=g) < 0.3
    allowed[2, 9000] = allowed[6, 8191] = True
    for kw in (dict(), dict(top_k=5, top_p=0.9), dict(top_p=0.5), dict(min_p=0.05), dict(temperature=0.0)):
        assert (_check_samples(x, u, **kw)[7] == -1).all()
        assert (_check_samples(x, u, allowed=allowed, **kw)[7] == -1).all()


def test_sample_settings_row_by_row_and_strides():
    g = torch.Generator().manual_seed(7)
    R, V = 40, 777
    x = torch.randn(R, V, generator=g) * 4
    u = torch.rand(R, generator=g)
    kw = dict(temperature=torch.rand(R, generator=g) * 2, top_k=torch.randint(0, 60, (R,), generator=g).to(torch.int32), top_p=torch.rand(R, generator=g) * 1.2,
              min_p=torch.rand(R, generator=g) * 0.4)
    kw["temperature"][3], kw["top_k"][4], kw["top_p"][5], kw["min_p"][6] = 0.0, -2, 1.0, 0.0
    a = _check_samples(x, u, **kw)
    wide = torch.zeros(R, V + 13, device=DEV)
    wide[:, 5:5 + V] = x.to(DEV)
    bits = torch.full((R, 40), -1, dtype=torch.int32, device=DEV)
    tok, _ = sample_tokens(wide[:, 5:5 + V], u.to(DEV), allowed_bits=bits[:, 3:30], **{k: v.to(DEV) for k, v in kw.items()})
    assert np.array_equal(tok.cpu().numpy(), a[:, 0])
    assert sample_tokens(wide[:0, :V], u.to(DEV)[:0])[0].shape == (0,)
    assert sample_tokens(wide[:, :V], torch.zeros(R, 0, device=DEV))[0].shape == (R, 0)


@pytest.mark.parametrize("draws", [63, 64, 65, 1500])
def test_sample_many_draws(draws):
    """more draws than a wave has lanes, than a workgroup has waves and threads; rows that one wave finishes and rows that need them all"""
    g = torch.Generator().manual_seed(draws)
    x, u = torch.randn(3, 700, generator=g) * 4, torch.rand(3, draws, generator=g)
    for kw in (dict(top_k=6), dict(top_k=50, top_p=0.9), dict(min_p=0.2), dict(top_p=0.9), dict()):
        _check_samples(x, u, **kw)


def test_sample_follows_the_distribution():
    """an even grid of u is a stratified sample: a token's share of the draws is off its probability by less than one draw at each end"""
    x = torch.tensor([[0.0, 1.0, -1.0, 2.0, 0.5]])
    n = 4096
    u = ((torch.arange(n) + 0.5) / n)[None]
    tok = sample_tokens(x.to(DEV), u.to(DEV), temperature=0.7)[0].cpu()
    share = torch.bincount(tok[0], minlength=5).double() / n
    assert ((share - torch.softmax(x[0].double() / 0.7, 0)).abs() <= 1.0 / n).all()


# ---------------------------------------------------------------------------
# as programs call them
# ---------------------------------------------------------------------------
@pytest.mark.parametrize("dt,V", [(F32, 3000), (BF16, 3000), (BF16, 40000)], ids=["fp32", "bf16", "bf16-large"])
def test_replayed_graphs_equal_eager_calls(dt, V):
    g = torch.Generator().manual_seed(41)
    S, H, T, D = 6, 2, 1024, 64
    w = quantize_w4(torch.randn(V, H * D, generator=g).to(DEV), 64)
    cache = _filled(S, H, T, D, 16, g)
    ln = torch.zeros(S, dtype=torch.int32, device=DEV)
    x, u = torch.zeros(S, 3, H, D, dtype=dt, device=DEV), torch.zeros(S, 2, device=DEV)
    sets = [(torch.randn(S, 3, H, D, generator=g), torch.rand(S, 2, generator=g), torch.randint(0, T, (S,), generator=g)) for _ in range(3)]
    held = [t.clone() for t in (cache.k, cache.v, cache.k_scale, cache.v_scale)]

    def change(i):
        x.copy_(sets[i][0]); u.copy_(sets[i][1]); ln.copy_(sets[i][2])
        for t, h in zip((cache.k, cache.v, cache.k_scale, cache.v_scale), held):
            t.copy_(h)

    def call():
        cache.append(x[:, 1:2], x[:, 2:3], ln)
        a = cache.attend(x[:, 0], ln + 1)
        y = w4_linear(a.view(S, H * D), w)
        tok, lp = sample_tokens(y, u, temperature=0.8, top_k=50, top_p=0.9)
        return a, y, tok, lp, cache.k, cache.v, cache.k_scale, cache.v_scale
    for got, want in _replayed(call, change):
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_calls_on_two_streams_at_once():
    """each call has its own workspace and outputs: two streams that run the same operators over one cache at once do not meet"""
    g = torch.Generator().manual_seed(42)
    S, H, T, D = 2, 2, 8192, 64
    cache = _filled(S, H, T, D, 64, g)
    ln = torch.tensor([8000, 5000], dtype=torch.int32, device=DEV)
    qs = [torch.randn(S, H, D, generator=g).to(DEV) for _ in range(2)]
    x, us = torch.randn(16, 40000, generator=g).to(DEV), [torch.rand(16, generator=g).to(DEV) for _ in range(2)]
    want = [(cache.attend(q, ln), *sample_tokens(x, u, top_p=0.9)) for q, u in zip(qs, us)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append((cache.attend(qs[i], ln), *sample_tokens(x, us[i], top_p=0.9)))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(a, b) for one in got[i] for a, b in zip(one, want[i]))
