"""The quantised, sampled decode's operators as far as the CPU goes: layouts, rounding, refusals (Python and C ABI), and the references that
the GPU tests use against torch's own rounding."""
import ctypes

import numpy as np
import pytest
import torch

from seal_amd._lib import SealFMError, check, lib, uint64s
from seal_amd.kv8 import KV8Cache
from seal_amd.sampling import sample_tokens
from seal_amd.w4 import W4Weight, quantize_w4, w4_linear
from tests import quant_refs as ref


# ---- 4-bit weights ----
@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (16, 128, 64), (21, 130, 32), (40, 300, 128), (33, 257, 64)])
def test_quantized_weights_are_the_nearest_multiples(N, K, group):
    g = torch.Generator().manual_seed(N * K)
    w = torch.randn(N, K, generator=g)
    if N > 1:
        w[1] = 0
    q = quantize_w4(w, group)
    assert q.group == group and q.out_features == N and q.in_features == K
    got = ref.w4_values(q.codes.numpy(), q.scales.float().numpy(), N, K)
    assert np.array_equal(got, q.dequantize().double().numpy())
    scale = q.scales.double().transpose(1, 2).reshape(-1, q.scales.shape[1]).numpy()
    for n in range(N):
        for k in range(K):
            s = scale[n, k // group]
            best = np.abs(ref.E2M1 * s - float(w[n, k])).min()
            assert abs(got[n, k] - float(w[n, k])) == best


def test_weight_ties_go_to_the_even_code():
    w = torch.zeros(1, 128)
    w[0, :8] = torch.tensor([6.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])      # scale 1: every entry but the first is a tie
    got = quantize_w4(w, 128).dequantize()[0, :8].tolist()
    assert got == [6.0, 0.0, 1.0, 1.0, 2.0, 2.0, 4.0, 4.0]


def test_weight_refusals():
    with pytest.raises(ValueError):
        quantize_w4(torch.zeros(4, 4), 48)
    with pytest.raises(ValueError):
        quantize_w4(torch.full((4, 4), float("nan")))
    q = quantize_w4(torch.randn(32, 128))
    with pytest.raises(ValueError):
        W4Weight(q.codes, q.scales, 64, 128)
    with pytest.raises(ValueError):
        W4Weight(q.codes, q.scales.float(), 32, 128)
    with pytest.raises(ValueError):
        W4Weight(q.codes.transpose(4, 5), q.scales, 32, 128)
    for x, b in ((torch.zeros(2, 127), None), (torch.zeros(2, 128, dtype=torch.float16), None), (torch.zeros(128), None),
                 (torch.zeros(128, 2).t(), None), (torch.zeros(2, 128), torch.zeros(31)), (torch.zeros(2, 128), torch.zeros(32, dtype=torch.bfloat16))):
        with pytest.raises(ValueError):
            w4_linear(x, q, b)
    with pytest.raises(RuntimeError):
        w4_linear(torch.zeros(2, 128), q)


# ---- the cache ----
def test_e4m3_reference_is_torchs_rounding():
    g = torch.Generator().manual_seed(0)
    x = torch.cat([torch.randn(20000, generator=g) * torch.exp2(torch.randint(-12, 7, (20000,), generator=g).float()), torch.arange(-448, 449) * 1.0,
                   torch.arange(0, 64) * 2.0 ** -10]).clamp(-448, 448)
    assert np.array_equal(ref.e4m3(x.double().numpy()), x.to(torch.float8_e4m3fn).double().numpy())


def test_cache_layout():
    S, H, T, D = 2, 3, 128, 64
    c = KV8Cache.empty(S, H, 100, D, block=32, device="cpu")
    assert c.k.shape == (S, H, T, D) and c.v.shape == (S, H, 2, D, 64) and c.k_scale.shape == (S, H, 4) and c.block == 32
    c.k.copy_(torch.randint(0, 127, c.k.shape, dtype=torch.uint8))
    c.v.copy_(torch.randint(0, 127, c.v.shape, dtype=torch.uint8))
    c.k_scale.copy_(torch.exp2(torch.randint(-3, 3, c.k_scale.shape).float()))
    c.v_scale.copy_(torch.exp2(torch.randint(-3, 3, c.k_scale.shape).float()))
    k, v = c.values()
    for s, h, t, d in ((0, 0, 0, 0), (1, 2, 127, 63), (0, 1, 77, 5), (1, 0, 64, 33), (0, 2, 18, 1)):
        fp = lambda b: float(b.view(torch.float8_e4m3fn))  # noqa: E731
        assert float(k[s, t, h, d]) == fp(c.k[s, h, t, d]) * float(c.k_scale[s, h, t // 32])
        assert float(v[s, t, h, d]) == fp(c.v[s, h, t // 64, d, ref.place(t % 64)]) * float(c.v_scale[s, h, t // 32])


def test_cache_refusals():
    c = KV8Cache.empty(2, 3, 64, 64, device="cpu")
    with pytest.raises(ValueError):
        KV8Cache.empty(2, 3, 64, 32, device="cpu")
    with pytest.raises(ValueError):
        KV8Cache.empty(2, 3, 64, 64, block=8, device="cpu")
    with pytest.raises(ValueError):
        KV8Cache(c.k, c.v, c.k_scale, c.v_scale[:, :, :2])
    with pytest.raises(ValueError):
        KV8Cache(c.k[:, :, :32], c.v, c.k_scale, c.v_scale)
    with pytest.raises(ValueError):
        KV8Cache(c.k.view(torch.int8), c.v, c.k_scale, c.v_scale)
    n = torch.zeros(2, dtype=torch.int32)
    kv = torch.zeros(2, 1, 3, 64)
    for k, v, ln, cn in ((kv[:1], kv[:1], n, None), (kv, kv.bfloat16(), n, None), (kv.half(), kv.half(), n, None), (kv, kv, n.long(), None),
                         (kv, kv, n[:1], None), (kv, kv, n, n.long()), (kv[..., :32], kv[..., :32], n, None), (kv, kv[:, :, :2], n, None),
                         (torch.zeros(2, 1, 64, 3).transpose(2, 3), kv, n, None)):
        with pytest.raises(ValueError):
            c.append(k, v, ln, cn)
    q = torch.zeros(4, 3, 64)
    for bad in (dict(q=q, beams=1), dict(q=q[:, :2], beams=2), dict(q=q.half(), beams=2), dict(q=q, beams=0), dict(q=q, beams=2, lengths=n.long()),
                dict(q=q, beams=2, keep=torch.ones(2, 63, dtype=torch.bool)), dict(q=q, beams=2, keep=torch.ones(2, 64)), dict(q=q[..., :32], beams=2),
                dict(q=torch.zeros(4, 64, 3).transpose(1, 2), beams=2)):
        with pytest.raises(ValueError):
            c.attend(bad["q"], bad.get("lengths", n), beams=bad["beams"], keep=bad.get("keep"))
    with pytest.raises(RuntimeError):
        c.append(kv, kv, n)
    with pytest.raises(RuntimeError):
        c.attend(q, n, beams=2)


# ---- sampling ----
def test_sampling_refusals():
    x, u = torch.zeros(3, 70), torch.zeros(3)
    for kw in (dict(logits=x.half()), dict(logits=x[0]), dict(logits=torch.zeros(70, 3).t()), dict(u=u[:2]), dict(u=u.double()), dict(u=torch.zeros(3, 1, 1)),
               dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_k=1.5), dict(top_p=1.5),
               dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=float("nan")), dict(temperature=torch.ones(2)), dict(top_k=torch.ones(3)),
               dict(allowed_bits=torch.zeros(3, 2, dtype=torch.int32)), dict(allowed_bits=torch.zeros(3, 3)), dict(logits=torch.zeros(3, (1 << 18) + 1)),
               dict(logits=torch.zeros(3, 0)), dict(logits=torch.zeros(1, 70).expand(3, 70))):
        with pytest.raises(ValueError):
            sample_tokens(kw.pop("logits", x), kw.pop("u", u), **kw)
    with pytest.raises(RuntimeError):
        sample_tokens(x, u)


def test_c_entries_refuse_before_they_launch():
    """the C ABI's own checks (a caller without the Python layer): an error and its text, no launch, so they run without a GPU"""
    L = lib()
    p = ctypes.cast(ctypes.create_string_buffer(64), ctypes.c_void_p).value & ~15
    st = uint64s(64, 64, 64, 64, 64, 64)
    for sfx in ("", "_bf16"):
        w4 = getattr(L, "sealnn_w4_linear" + sfx)
        ap, at, sm = getattr(L, "sealnn_kv8_append" + sfx), getattr(L, "sealnn_kv8_attend" + sfx), getattr(L, "sealnn_sample_tokens" + sfx)
        bad = [lambda: w4(None, p, 128, p, p, None, 1, 16, 128, 48, 0, p), lambda: w4(None, None, 128, p, p, None, 1, 16, 128, 32, 0, p),
               lambda: w4(None, p, 128, p + 4, p, None, 1, 16, 128, 32, 0, p), lambda: w4(None, p, 128, p, p, None, 1, 16, 0, 32, 0, p),
               lambda: w4(None, p + 1, 128, p, p, None, 1, 16, 128, 32, 0, p), lambda: w4(None, p, 128, p, p, None, (1 << 19) + 1, 16, 128, 32, 0, p),
               lambda: ap(None, p, p, st, 1, p, None, p, p, p, p, 1, 1, 64, 16, 32), lambda: ap(None, p, p, st, 1, p, None, p, p, p, p, 1, 1, 65, 16, 64),
               lambda: ap(None, p, p, st, 1, p, None, p, p, p, p, 1, 1, 64, 24, 64), lambda: ap(None, p, p, st, 1, None, None, p, p, p, p, 1, 1, 64, 16, 64),
               lambda: ap(None, p, p, st, 1, p, None, p + 8, p, p, p, 1, 1, 64, 16, 64), lambda: ap(None, p, None, st, 1, p, None, p, p, p, p, 1, 1, 64, 16, 64),
               lambda: at(None, p, 64, 64, p, p, p, p, p, None, 0, 1, 1, 1, 1, 64, 16, 64, 1.0, 2, None, 0, p),
               lambda: at(None, p, 64, 64, p, p, p, p, p, None, 0, 1, 1, 1, 1, 128, 16, 64, 1.0, 2, p, 64, p),
               lambda: at(None, p, 64, 64, p, p, p, p, p, p + 1, 64, 1, 1, 1, 1, 64, 16, 64, 1.0, 1, None, 0, p),
               lambda: at(None, None, 64, 64, p, p, p, p, p, None, 0, 1, 1, 1, 1, 64, 16, 64, 1.0, 1, None, 0, p),
               lambda: at(None, p, 64, 64, p, p, p, p, p, None, 0, 1, 1, 1, 1, 64, 16, 96, 1.0, 1, None, 0, p),
               lambda: at(None, p, 64, 64, p, p, p, p, p, None, 0, 1 << 20, 1 << 10, 64, 1, 64, 16, 64, 1.0, 1, None, 0, p),
               lambda: sm(None, p, 10, 1, (1 << 18) + 1, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, None, 0),
               lambda: sm(None, p, 10, 1, 0, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, None, 0),
               lambda: sm(None, None, 10, 1, 10, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, None, 0),
               lambda: sm(None, p, 10, 1, 10, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, p, 96 + 16448 - 1),
               lambda: sm(None, p, 10, 1, 10, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, p + 8, 1 << 20),
               lambda: sm(None, p, 10, 65536, 10, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, p, 1 << 40),
               lambda: sm(None, p, 10, 1, 3, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, p, 1 << 20)]
        for i, f in enumerate(bad):
            with pytest.raises(SealFMError) as e:
                check(f())
            assert "sealnn_" in str(e.value), i
        # nothing to do is not an error
        check(w4(None, p, 128, p, p, None, 0, 16, 128, 32, 0, p))
        check(ap(None, p, p, st, 0, p, None, p, p, p, p, 1, 1, 64, 16, 64))
        check(at(None, p, 64, 64, p, p, p, p, p, None, 0, 0, 1, 1, 1, 64, 16, 64, 1.0, 1, None, 0, p))
        check(sm(None, p, 10, 0, 10, p, 1, None, 0, 1.0, 0, 1.0, 0.0, None, None, None, None, p, p, None, 0))
