"""What the quantised, sampled decode's Python entries refuse beyond shapes and types, and what quantising has to get right at the edge of a type's range.  No GPU."""
import pytest
import torch

from seal_amd.kv8 import KV8Cache
from seal_amd.sampling import sample_tokens
from seal_amd.w4 import quantize_w4, w4_linear


def _calls():
    c, n = KV8Cache.empty(2, 1, 64, 64, device="cpu"), torch.zeros(2, dtype=torch.int32)
    kv, w = torch.zeros(2, 1, 1, 64), quantize_w4(torch.randn(16, 128))
    return {
        "sample_tokens": (lambda t: sample_tokens(t, torch.zeros(2)), torch.zeros(2, 70)),
        "w4_linear": (lambda t: w4_linear(t, w), torch.zeros(2, 128)),
        "w4_linear bias": (lambda t: w4_linear(torch.zeros(2, 128), w, t), torch.zeros(16)),
        "KV8Cache.append keys": (lambda t: c.append(t, kv, n), kv.clone()),
        "KV8Cache.append values": (lambda t: c.append(kv, t, n), kv.clone()),
        "KV8Cache.attend": (lambda t: c.attend(t, n), torch.zeros(2, 1, 64)),
    }


@pytest.mark.parametrize("name", list(_calls()))
def test_a_gradient_is_refused_not_lost(name):
    call, t = _calls()[name]
    t.requires_grad_(True)
    with pytest.raises(RuntimeError, match="backward"):
        call(t)
    with pytest.raises(RuntimeError, match="backward"):
        call(t * 2)                                       # (a result with history)
    # without a gradient to lose the call goes on, here as far as the missing GPU
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):
        call(t)
    with torch.inference_mode(), pytest.raises(RuntimeError, match="GPU"):
        call(t)
    with pytest.raises(RuntimeError, match="GPU"):
        call(t.detach())


def test_reorder_takes_a_row_for_every_slot():
    """a single row would be copied into every slot"""
    c = KV8Cache.empty(3, 2, 64, 64, device="cpu")
    for t in (c.k, c.v):
        t.copy_(torch.randint(0, 127, t.shape, dtype=torch.uint8))
    for t in (c.k_scale, c.v_scale):
        t.copy_(torch.exp2(torch.randint(-3, 3, t.shape).float()))
    held = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]
    for bad in (torch.tensor([1]), torch.tensor([0, 1]), torch.tensor([[0, 1, 2]]), torch.tensor([0.0, 1.0, 2.0]), torch.tensor([True, False, True]), torch.tensor(1)):
        with pytest.raises(ValueError):
            c.reorder(bad)
        assert all(torch.equal(a, b) for a, b in zip((c.k, c.v, c.k_scale, c.v_scale), held))
    for dt in (torch.int64, torch.int32):
        c.reorder(torch.tensor([2, 2, 0], dtype=dt))
        assert all(torch.equal(a, b[[2, 2, 0]]) for a, b in zip((c.k, c.v, c.k_scale, c.v_scale), held))
        held = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)]


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("size", [1e-36, 1e-38, 3e-39, 1e-40, 3e-41, 1e-44, 3e38])
def test_tiny_and_huge_weights_are_the_nearest_multiples_too(size, group):
    """scales below the smallest normal number (bf16 has fp32's subnormals, with 8 bits less), scales that round to zero, weights up to the largest number"""
    from tests import quant_refs as ref
    g = torch.Generator().manual_seed(3)
    w = (torch.rand(20, 300, generator=g) * 2 - 1) * size
    w[0, :40] = 0
    q = quantize_w4(w, group)
    got = ref.w4_values(q.codes.numpy(), q.scales.float().numpy(), 20, 300)
    s = q.scales.double().transpose(1, 2).reshape(-1, q.scales.shape[1]).numpy().repeat(group, 1)[:20, :300]
    best = abs(ref.E2M1[:, None, None] * s - w.double().numpy()).min(0)
    assert (abs(got - w.double().numpy()) == best).all()
    assert torch.equal(q.dequantize().double(), torch.from_numpy(got))


def test_weights_beyond_fp32_are_refused():
    w = torch.zeros(4, 64, dtype=torch.float64)
    w[1, 2] = 1e300
    with pytest.raises(ValueError):
        quantize_w4(w)
