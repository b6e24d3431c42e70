"""What the operators of a quantised, sampled decode are measured on: drawing the next token from the logits, the 8-bit
key / value cache (writing into it and attending to it) and products with 4-bit weights.

``run`` computes them in elementary torch operations (``own = False``) or through ``seal_amd`` (``own = True``); ``exact``
computes the same from the definitions in 64 bits.

Layouts, shared by both sides:

* cache: ``k`` [slots, heads, T, dh] e4m3 codes; ``v`` [slots, heads, T / 64, dh, 64] e4m3 codes, where the 64 tokens of a tile
  stand in the order (g, j, r) of token 16 j + 4 g + r; ``k_scale`` / ``v_scale`` [slots, heads, T / block] fp32 powers of two.
* weights: ``codes`` [N / 16, K / 128, 4, 16, 4, 4] uint8 -- (chunk position g, row, s, byte): the four bytes hold the eight
  e2m1 codes of columns 32 s + 8 g .. + 7 of the 128-column chunk, the even column in the low nibble; ``scales``
  [N / 16, K / group, 16] bf16; N padded to 16 and K to 128 with zeros.
"""
import math

import numpy as np
import torch

own = False

FLT_MAX = torch.finfo(torch.float32).max
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # one interactive row over BART's vocabulary, nucleus sampling: latency
        dict(name="sample, one row", op="sample", rows=1, vocab=50265, dtype="fp32", draws=1, temperature=0.7, top_k=0, top_p=0.9, min_p=0.0, allowed=1.0),
        # a batch of 20 queries x 15 samples, constrained to a corpus: one token in a hundred is allowed
        dict(name="sample, constrained", op="sample", rows=300, vocab=50265, dtype="fp32", draws=1, temperature=0.8, top_k=50, top_p=0.95, min_p=0.0, allowed=0.01),
        # a large bf16 batch over a large vocabulary, four draws from each row
        dict(name="sample, large", op="sample", rows=512, vocab=131072, dtype="bf16", draws=4, temperature=1.0, top_k=0, top_p=1.0, min_p=0.02, allowed=1.0),
        # a decode step's new token, 20 queries x 15 samples of BART-large
        dict(name="append, one token", op="append", slots=300, heads=16, head_dim=64, tokens=64, block=16, new=1, low=1, high=40, dtype="fp32"),
        # the encoder states of long inputs, ragged, written into an empty cache
        dict(name="append, long inputs", op="append", slots=24, heads=16, head_dim=64, tokens=1024, block=64, new=1000, low=0, high=0, dtype="bf16"),
        # self-attention of a decode step over the short history of every sample
        dict(name="attend, own history", op="attend", slots=300, heads=16, head_dim=64, tokens=64, block=16, q_heads=16, beams=1, low=1, high=17, keep=1.0, dtype="fp32"),
        # cross-attention of a decode step: 15 samples share a query's encoder states
        dict(name="attend, short inputs", op="attend", slots=20, heads=16, head_dim=64, tokens=64, block=16, q_heads=16, beams=15, low=12, high=30, keep=1.0, dtype="fp32"),
        # the same over inputs of up to BART's 1024 positions, with holes in the mask
        dict(name="attend, long inputs", op="attend", slots=40, heads=16, head_dim=64, tokens=1024, block=32, q_heads=16, beams=15, low=500, high=1024, keep=0.9, dtype="fp32"),
        # one sequence with a long history: the work has to be split over its length
        dict(name="attend, one long row", op="attend", slots=1, heads=16, head_dim=64, tokens=32768, block=64, q_heads=16, beams=1, low=32001, high=32001, keep=1.0, dtype="bf16"),
        # many long histories, four query heads on every cached head
        dict(name="attend, large", op="attend", slots=32, heads=8, head_dim=128, tokens=8192, block=64, q_heads=32, beams=1, low=4001, high=8192, keep=1.0, dtype="bf16"),
        # the output projection for one row
        dict(name="product, one row", op="product", rows=1, out=50265, inner=1024, group=64, dtype="fp32", gelu=False),
        # the first feed-forward product of four queries x 15 samples
        dict(name="product, 60 rows", op="product", rows=60, out=4096, inner=1024, group=32, dtype="bf16", gelu=True),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("sample", "append", "attend", "product"))
    dtype = rng.choice(("fp32", "bf16"))
    if op == "sample":
        vocab = _log(rng, 80, 131072)
        rows = _log(rng, 1, min(640, (512 * 131072) // vocab))
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, draws=rng.choice((1, 1, 1, 3, 16)), temperature=round(rng.uniform(0.3, 1.6), 3),
                    top_k=rng.choice((0, 0, 1, _log(rng, 2, 1000))), top_p=rng.choice((1.0, round(rng.uniform(0.05, 0.99), 3))),
                    min_p=rng.choice((0.0, 0.0, round(rng.uniform(0.001, 0.3), 4))), allowed=rng.choice((1.0, 0.3, 0.01)))
    if op == "product":
        rows, inner = _log(rng, 1, 64), _log(rng, 64, 4096)
        return dict(op=op, rows=rows, out=_log(rng, 16, (50265 * 1024) // max(1024, inner)), inner=inner, group=rng.choice((32, 64, 128)), dtype=dtype, gelu=rng.random() < 0.3)
    head_dim, heads, block = rng.choice((64, 64, 128)), rng.choice((1, 2, 8, 12, 16)), rng.choice((16, 32, 64))
    if op == "append":
        new = rng.choice((1, _log(rng, 2, 1000)))
        old = rng.choice((0, _log(rng, 1, 1000)))
        slots = _log(rng, 1, max(1, min(300, (24 * 16 * 64 * 1000) // (heads * head_dim * new))))
        tokens = -(-(new + old) // 64) * 64
        return dict(op=op, slots=slots, heads=heads, head_dim=head_dim, tokens=tokens, block=block, new=new, low=min(old, 1), high=old, dtype=dtype)
    high = _log(rng, 1, 32768)
    low = max(1, int(high * rng.uniform(0.1, 1.0)))
    tokens = -(-high // 64) * 64
    slots = _log(rng, 1, max(1, min(300, (1 << 28) // (heads * head_dim * tokens))))
    q_heads = heads * rng.choice((1, 1, 2, 4))
    return dict(op=op, slots=slots, heads=heads, head_dim=head_dim, tokens=tokens, block=block, q_heads=q_heads, beams=rng.choice((1, 1, 5, 15, 30)) if q_heads == heads else 1,
                low=low, high=high, keep=rng.choice((1.0, 1.0, 0.7)), dtype=dtype)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _rng(seed, dev):
    return torch.Generator(device=dev).manual_seed(int(seed))


def _lengths(case, seed, g, dev):
    """lengths spread evenly over low .. high (so that the work of a case does not hang on the seed), in an order of the seed's"""
    n = case["slots"]
    v = torch.linspace(case["low"], case["high"], n, dtype=torch.float64, device=dev).round().to(torch.int32) if n > 1 else torch.full((1,), case["high"], dtype=torch.int32, device=dev)
    return v[torch.randperm(n, generator=g, device=dev)].contiguous()


def _codes(shape, g, dev):
    """e4m3 codes of normal values"""
    x = torch.empty(shape, dtype=torch.float8_e4m3fn, device=dev)
    flat = x.view(-1)
    for a in range(0, flat.numel(), 1 << 26):
        b = min(flat.numel(), a + (1 << 26))
        flat[a:b] = (torch.randn(b - a, generator=g, device=dev) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return x.view(torch.uint8)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = _rng(seed, dev)
    op, dt = case["op"], DTYPES[case["dtype"]]
    if op == "sample":
        R, V = case["rows"], case["vocab"]
        # a decoder's logits: a broad normal bulk and a handful of likely tokens in every row
        x = torch.randn(R, V, generator=g, device=dev) * 2.5
        at = torch.randint(0, V, (R, 8), generator=g, device=dev)
        x.scatter_add_(1, at, torch.rand(R, 8, generator=g, device=dev) * 10)
        bits = None
        if case["allowed"] < 1:
            words = (V + 31) // 32
            ok = torch.rand(R, words * 32, generator=g, device=dev) < case["allowed"]
            ok.view(-1)[torch.randint(0, V, (R,), generator=g, device=dev) + torch.arange(R, device=dev) * words * 32] = True
            w = ok.view(R, words, 32).to(torch.int64) << torch.arange(32, device=dev)
            w = w.sum(-1)
            bits = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
        return dict(case=case, logits=x.to(dt), u=torch.rand(R, case["draws"], generator=g, device=dev), bits=bits)
    if op == "product":
        N, K, G = case["out"], case["inner"], case["group"]
        Np, Kp = -(-N // 16) * 16, -(-K // 128) * 128
        # normal weights in e2m1 with a scale for each group of columns: the group's largest magnitude becomes 6
        w = torch.zeros(Np, Kp, device=dev)
        w[:N, :K] = torch.randn(N, K, generator=g, device=dev) * (K ** -0.5)
        wg = w.view(Np, Kp // G, G)
        sc = (wg.abs().amax(-1) / 6).to(torch.bfloat16)
        y = (wg / sc.float().clamp_min(1e-30).unsqueeze(-1)).clamp(-6, 6).view(Np, Kp)
        lut = torch.tensor(E2M1, device=dev)
        c = torch.bucketize(y.abs(), (lut[1:] + lut[:-1]) / 2).to(torch.uint8) | (torch.signbit(y).to(torch.uint8) << 3)
        c = c.view(Np // 16, 16, Kp // 128, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)           # (tile, chunk, g, row, s, byte, nibble)
        codes = (c[..., 0] | (c[..., 1] << 4)).contiguous()
        scales = sc.view(Np // 16, 16, Kp // G).transpose(1, 2).contiguous()
        x = torch.randn(case["rows"], K, generator=g, device=dev) * torch.exp(torch.randn(K, generator=g, device=dev) * 0.5)
        return dict(case=case, codes=codes, scales=scales, x=x.to(dt), bias=(torch.randn(N, generator=g, device=dev) * 0.1).to(dt))
    S, H, T, D, blk = case["slots"], case["heads"], case["tokens"], case["head_dim"], case["block"]
    # caches as a running program holds them: codes everywhere (what lies behind a slot's length is old), power-of-two scales of a few sizes
    k, v = _codes((S, H, T, D), g, dev), _codes((S, H, T // 64, D, 64), g, dev)
    ks, vs = (torch.exp2(torch.randint(-9, -5, (S, H, T // blk), generator=g, device=dev).float()) for _ in range(2))
    st = dict(case=case, k=k, v=v, k_scale=ks, v_scale=vs, lengths=_lengths(case, seed, g, dev))
    if op == "append":
        n = case["new"]
        # k and v are parts of one fused projection's output [slots, new, 3, heads, dh]
        qkv = torch.randn(S, n, 3, H, D, generator=g, device=dev) * torch.exp2(torch.randint(-3, 4, (S, n, 1, H, 1), generator=g, device=dev).float())
        qkv = qkv.to(dt)
        st.update(k_new=qkv[:, :, 1], v_new=qkv[:, :, 2], counts=None)
        if n > 1:                                   # ragged: every slot brings its own number of tokens
            c = torch.linspace(n / 2, n, S, device=dev).round().to(torch.int32)
            st["counts"] = c[torch.randperm(S, generator=g, device=dev)].contiguous()
        return st
    st["q"] = (torch.randn(S * case["beams"], case["q_heads"], D, generator=g, device=dev) * 1.5).to(dt)
    st["keep"] = (torch.rand(S, T, generator=g, device=dev) < case["keep"]) if case["keep"] < 1 else None
    return st


# ---------------------------------------------------------------------------
# the operators in plain torch operations
# ---------------------------------------------------------------------------
def _sample_plain(s):
    """weights, filters and draws in 64 bits: the border of a nucleus and the token that a random number falls on hang on long sums
    (the settings are fp32 numbers: temperature, top_p and min_p are rounded to that first)"""
    c = s["case"]
    x = s["logits"].double()
    x = torch.where(x != x, -math.inf, x).clamp(max=FLT_MAX)
    R, V = x.shape
    top = x.amax(-1, keepdim=True)
    lse = torch.log(torch.exp(x - top).sum(-1, keepdim=True)) + top
    z = x
    if s["bits"] is not None:
        ok = (s["bits"][:, :, None] >> torch.arange(32, device=x.device)) & 1
        z = torch.where(ok.view(R, -1)[:, :V] != 0, x, -math.inf)
    val, idx = torch.sort(z, dim=-1, descending=True, stable=True)
    best = val[:, :1]
    some = best > -math.inf
    w = torch.where(val > -math.inf, torch.exp((val - torch.where(some, best, 0.0)) / float(np.float32(c["temperature"]))), 0.0)
    kept = w > 0
    if c["top_k"] > 0:
        kept &= torch.arange(V, device=x.device) < c["top_k"]
    if c["top_p"] < 1:
        wk = torch.where(kept, w, 0.0)
        cum = torch.cumsum(wk, -1)
        kept &= (cum - wk) < float(np.float32(c["top_p"])) * cum[:, -1:]
    if c["min_p"] > 0:
        kept &= w >= float(np.float32(c["min_p"]))
    w = torch.zeros_like(w).scatter_(1, idx, torch.where(kept, w, 0.0))        # back into the order of the vocabulary
    cum = torch.cumsum(w, -1)
    t = s["u"].double() * cum[:, -1:]
    tok = torch.searchsorted(cum, t, right=True)                               # the first token whose cumulative weight passes u * total
    last = V - 1 - torch.argmax((w > 0).flip(-1).to(torch.int8), -1, keepdim=True)
    tok = torch.minimum(tok, last)
    lp = x.gather(1, tok) - lse
    return torch.where(some, tok, -1), torch.where(some, lp, -math.inf).float()


def _v_tokens(v):
    """[slots, heads, T / 64, dh, 64] -> [slots, heads, T, dh] (any type)"""
    S, H, n, D, _ = v.shape
    return v.view(S, H, n, D, 4, 4, 4).permute(0, 1, 2, 5, 4, 6, 3).reshape(S, H, n * 64, D)


def _v_tiles(v):
    """[slots, heads, T, dh] -> [slots, heads, T / 64, dh, 64]"""
    S, H, T, D = v.shape
    return v.view(S, H, T // 64, 4, 4, 4, D).permute(0, 1, 2, 6, 4, 3, 5).reshape(S, H, T // 64, D, 64)


def _values(codes, scale):
    S, H, T, D = codes.shape
    return (codes.view(torch.float8_e4m3fn).float().view(S, H, scale.shape[2], -1) * scale.unsqueeze(-1)).view(S, H, T, D)


def _pow2(e):
    return ((e + 127) << 23).to(torch.int32).view(torch.float32)


def _append_codes(old, scale, new, lengths, counts):
    """(codes [slots, heads, T, dh], scale) after ``new`` [slots, n, heads, dh] went to positions lengths .. lengths + counts - 1"""
    S, H, T, D = old.shape
    n, nb = new.shape[1], scale.shape[2]
    blk = T // nb
    pos = torch.arange(T, device=old.device)
    rel = pos[None, :] - lengths[:, None]                                          # [slots, T]: which new token stands at a position
    fresh = (rel >= 0) & (rel < (counts[:, None] if counts is not None else n))
    x = torch.gather(new.float().permute(0, 2, 1, 3), 2, rel.clamp(0, n - 1)[:, None, :, None].expand(S, H, T, D))
    x = x.view(S, H, nb, blk, D)
    fb = fresh.view(S, 1, nb, blk, 1)
    mag = torch.where(fb & x.isfinite(), x.abs(), 0.0).amax((-1, -2))                # [slots, heads, nb]
    m, e = torch.frexp(mag)
    need = torch.where(mag > 0, e - torch.where(m <= 0.875, 9, 8), -64).clamp(min=-64)
    held = ((pos.view(nb, blk)[None, :, 0] < lengths[:, None]))[:, None, :]           # the block had tokens before
    touched = fb.any(3).view(S, 1, nb)
    e_old = (scale.view(torch.int32) >> 23) - 127
    e_new = torch.where(touched, torch.where(held, torch.maximum(need, e_old), need), e_old)
    y = torch.where(x != x, x, (x * _pow2(-e_new)[..., None, None]).clamp(-448, 448))
    kept = old.view(torch.float8_e4m3fn).float().view(S, H, nb, blk, D) * _pow2((e_old - e_new).clamp(min=-126))[..., None, None]
    before = (pos[None, :] < lengths[:, None]).view(S, 1, nb, blk, 1) & touched[..., None, None]
    codes = torch.where(fb, y, kept).to(torch.float8_e4m3fn).view(torch.uint8)
    codes = torch.where(fb | before, codes, old.view(S, H, nb, blk, D))
    return codes.view(S, H, T, D), _pow2(e_new)


def _append_plain(s):
    k, ks = _append_codes(s["k"], s["k_scale"], s["k_new"], s["lengths"], s["counts"])
    v, vs = _append_codes(_v_tokens(s["v"]), s["v_scale"], s["v_new"], s["lengths"], s["counts"])
    s["k"].copy_(k)
    s["k_scale"].copy_(ks)
    s["v"].copy_(_v_tiles(v))
    s["v_scale"].copy_(vs)
    return _cache_outputs(s)


def _cache_outputs(s):
    return s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn), s["k_scale"], s["v_scale"]


def _attend_plain(s):
    c, q = s["case"], s["q"]
    k, v = _values(s["k"], s["k_scale"]), _values(_v_tokens(s["v"]), s["v_scale"])
    S, H, T, D = k.shape
    n = c["beams"] * (c["q_heads"] // H)
    qf = q.float().view(S, c["beams"], H, c["q_heads"] // H, D).permute(0, 2, 1, 3, 4).reshape(S, H, n, D)
    ok = torch.arange(T, device=q.device)[None, :] < s["lengths"][:, None]
    if s["keep"] is not None:
        ok = ok & s["keep"]
    sc = torch.matmul(qf, k.transpose(-1, -2)) * D ** -0.5
    sc = torch.where(ok[:, None, None, :], sc, -math.inf)
    m = sc.amax(-1, keepdim=True)
    p = torch.exp(sc - torch.where(m > -math.inf, m, 0.0))
    out = torch.matmul(p, torch.where(ok[:, None, :, None], v, 0.0)) / p.sum(-1, keepdim=True).clamp_min(1e-30)
    return out.view(S, H, c["beams"], -1, D).permute(0, 2, 1, 3, 4).reshape(S * c["beams"], c["q_heads"], D).to(q.dtype)


def _weights(s, dt):
    c = s["case"]
    b = s["codes"]
    nib = torch.stack([b & 15, b >> 4], -1).long()                                   # (tile, chunk, g, row, s, byte, nibble)
    val = torch.tensor(E2M1 + tuple(-t for t in E2M1), dtype=dt, device=b.device)[nib]
    w = val.permute(0, 3, 1, 4, 2, 5, 6).reshape(b.shape[0] * 16, b.shape[1] * 128)
    sc = s["scales"].transpose(1, 2).reshape(w.shape[0], -1, 1).to(dt)
    return (w.view(w.shape[0], -1, c["group"]) * sc).view_as(w)[:c["out"], :c["inner"]]


def _product_plain(s):
    y = torch.matmul(s["x"].float(), _weights(s, torch.float32).t()) + s["bias"].float()
    if s["case"]["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * 0.5 ** 0.5))
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    c = state["case"]
    if own:
        return _run_own(state)
    return {"sample": _sample_plain, "append": _append_plain, "attend": _attend_plain, "product": _product_plain}[c["op"]](state)


def _run_own(s):
    c = s["case"]
    if c["op"] == "sample":
        from seal_amd.sampling import sample_tokens
        return sample_tokens(s["logits"], s["u"], temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"], allowed_bits=s["bits"])
    if c["op"] == "product":
        from seal_amd.w4 import W4Weight, w4_linear
        return w4_linear(s["x"], W4Weight(s["codes"], s["scales"], c["out"], c["inner"]), s["bias"], gelu=c["gelu"])
    from seal_amd.kv8 import KV8Cache
    cache = KV8Cache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    if c["op"] == "append":
        cache.append(s["k_new"], s["v_new"], s["lengths"], s["counts"])
        return _cache_outputs(s)
    return cache.attend(s["q"], s["lengths"], beams=c["beams"], keep=s["keep"])


def _sum_lengths(case):
    return int(np.round(np.linspace(case["low"], case["high"], case["slots"])).sum()) if case["slots"] > 1 else case["high"]


def work(case):
    op, size = case["op"], 4 if case["dtype"] == "fp32" else 2
    if op == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size + (n / 8 if case["allowed"] < 1 else 0) + case["rows"] * case["draws"] * 16, "flops": 4 * n}
    if op == "product":
        n = case["out"] * case["inner"]
        return {"bytes": n / 2 + 2 * n / case["group"] + size * (case["rows"] * (case["inner"] + case["out"]) + case["out"]), "flops": 2 * n * case["rows"]}
    H, D = case["heads"], case["head_dim"]
    if op == "append":
        # the new values read, their codes written; the block that a slot's tokens end in is read and written again where it is not empty
        n = case["slots"] * (0.75 if case["new"] > 1 else 1) * case["new"]
        again = case["slots"] * case["block"] / 2 if case["high"] > 0 else 0
        return {"bytes": 2 * H * D * (n * (size + 1) + 2 * again), "flops": 6 * H * D * n}
    n = _sum_lengths(case)
    return {"bytes": 2 * n * H * (D + 4 / case["block"]) + 2 * size * case["slots"] * case["beams"] * case["q_heads"] * D,
            "flops": 4 * n * case["beams"] * case["q_heads"] * D}


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"sample": _sample_exact, "append": _append_exact, "attend": _attend_exact, "product": _product_exact}[case["op"]](s)


def _sample_exact(s):
    """row by row on the host, with numpy"""
    c = s["case"]
    R, V = s["logits"].shape
    if R * V > 70_000_000:
        return None
    u = s["u"].cpu().numpy().astype(np.float64)
    toks, lps = np.zeros((R, c["draws"]), np.int64), np.zeros((R, c["draws"]))
    bits = None if s["bits"] is None else np.unpackbits(s["bits"].cpu().numpy().view(np.uint8), axis=1, bitorder="little")[:, :V].astype(bool)
    logits = s["logits"].float().cpu().numpy()
    for r in range(R):
        x = logits[r].astype(np.float64)
        may = np.isfinite(x) if bits is None else np.isfinite(x) & bits[r]
        at = np.flatnonzero(may)
        if not at.size:
            toks[r], lps[r] = -1, -np.inf
            continue
        z = x[at]
        w = np.exp((z - z.max()) / float(np.float32(c["temperature"])))
        if c["top_k"] > 0 or c["top_p"] < 1:
            order = np.lexsort((at, -z))
            n = min(at.size, c["top_k"]) if c["top_k"] > 0 else at.size
            if c["top_p"] < 1:
                mass = np.cumsum(w[order[:n]])
                n = int(np.searchsorted(mass, float(np.float32(c["top_p"])) * mass[-1], side="left")) + 1
            sel = np.sort(order[:n])
            at, w = at[sel], w[sel]
        if c["min_p"] > 0:
            sel = w >= float(np.float32(c["min_p"]))
            at, w = at[sel], w[sel]
        mass = np.cumsum(w)
        got = at[np.minimum(np.searchsorted(mass, u[r] * mass[-1], side="right"), at.size - 1)]
        toks[r] = got
        lps[r] = x[got] - (x.max() + np.log(np.exp(x - x.max()).sum()))
    return torch.from_numpy(toks), torch.from_numpy(lps)


def _e4m3(y):
    """round to the nearest e4m3 value, ties to even, in 64 bits (|y| <= 448)"""
    _, e = np.frexp(y)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(y / step) * step


def _append_exact(s):
    """slot by slot on the host, with numpy, from the definition: a block's scale is the smallest power of two that holds its new tokens,
    or its old scale where that is larger and the block had tokens"""
    c = s["case"]
    S, H, T, D, blk = c["slots"], c["heads"], c["tokens"], c["head_dim"], c["block"]
    if S * H * T * D > 60_000_000:
        return None
    out = []
    lengths = s["lengths"].cpu().numpy()
    counts = np.full(S, c["new"]) if s["counts"] is None else s["counts"].cpu().numpy()
    token = np.array([16 * j + 4 * g + r for g in range(4) for j in range(4) for r in range(4)])   # the token at each place of a tile
    for name in ("k", "v"):
        val = s[name].view(torch.float8_e4m3fn).double().cpu().numpy().copy()
        sc = s[name + "_scale"].double().cpu().numpy().copy()
        new = s[name + "_new"].double().cpu().numpy()
        for i in range(S):
            a, b = int(lengths[i]), min(T, int(lengths[i] + counts[i]))
            for at in range(a // blk, -(-b // blk)):
                lo, hi = max(a, at * blk), min(b, (at + 1) * blk)
                if lo >= hi:
                    continue
                x = new[i, lo - a:hi - a].transpose(1, 0, 2)                              # [heads, tokens, dh]
                big = np.abs(x).max((1, 2))
                e = np.maximum(np.ceil(np.log2(np.maximum(big, 2.0 ** -60) / 448)), -64)
                e = np.where(big > 448 * np.exp2(e), e + 1, np.where(big <= 448 * np.exp2(e - 1), e - 1, e)).clip(-64)
                e = np.where(big > 0, e, -64)
                if lo > at * blk:
                    e = np.maximum(e, np.log2(sc[i, :, at]))
                    ratio = (sc[i, :, at] / np.exp2(e))[:, None, None]
                    if name == "k":
                        val[i, :, at * blk:lo] = _e4m3(val[i, :, at * blk:lo] * ratio)
                    else:
                        t0, cols = at * blk // 64, np.flatnonzero((token >= at * blk % 64) & (token < at * blk % 64 + lo - at * blk))
                        val[i, :, t0, :, cols] = _e4m3(val[i, :, t0, :, cols] * ratio.transpose(1, 0, 2))
                sc[i, :, at] = np.exp2(e)
                y = _e4m3(x / np.exp2(e)[:, None, None])
                if name == "k":
                    val[i, :, lo:hi] = y
                else:
                    t0 = lo // 64
                    cols = np.flatnonzero((token >= lo % 64) & (token < lo % 64 + hi - lo))
                    val[i, :, t0, :, cols] = y[:, token[cols] - lo % 64].transpose(1, 0, 2)
        out.append((val, sc))
    return tuple(torch.from_numpy(t) for t in (out[0][0], out[1][0], out[0][1], out[1][1]))


def _attend_exact(s):
    """one slot at a time, only the tokens that are there"""
    c, q = s["case"], s["q"].double()
    S, H, blk = c["slots"], c["heads"], c["block"]
    share = c["q_heads"] // H
    out = torch.zeros_like(q)
    place = torch.tensor([(t % 16 // 4) * 16 + t // 16 * 4 + t % 4 for t in range(64)], device=q.device)
    for i in range(S):
        n = int(s["lengths"][i])
        at = torch.arange(n, device=q.device)
        if s["keep"] is not None:
            at = at[s["keep"][i, :n]]
        if not at.numel():
            continue
        k = s["k"][i].view(torch.float8_e4m3fn).double()[:, at] * s["k_scale"][i][:, at // blk].double()[..., None]
        v = s["v"][i].view(torch.float8_e4m3fn).double()[:, at // 64, :, place[at % 64]]                # (advanced indices around a slice: the tokens come first)
        v = v.permute(1, 0, 2) * s["v_scale"][i][:, at // blk].double()[..., None]
        qi = q[i * c["beams"]:(i + 1) * c["beams"]]
        for h in range(H):
            p = torch.softmax(qi[:, h * share:(h + 1) * share] @ k[h].t() * c["head_dim"] ** -0.5, -1)
            out[i * c["beams"]:(i + 1) * c["beams"], h * share:(h + 1) * share] = p @ v[h]
    return out


def _product_exact(s):
    """the weights from their bytes one nibble at a time: column 32 s + 8 g + i of a chunk is nibble i of word (g, row, s)"""
    c = s["case"]
    b = s["codes"].cpu().numpy()
    tiles, chunks = b.shape[:2]
    w = np.zeros((tiles, 16, chunks, 128))
    lut = np.array(E2M1 + tuple(-t for t in E2M1))
    for g in range(4):
        for part in range(4):
            for i in range(8):
                w[:, :, :, 32 * part + 8 * g + i] = lut[(b[:, :, g, :, part, i // 2] >> (4 * (i % 2))) & 15].transpose(0, 2, 1)
    w = w.reshape(tiles * 16, chunks * 128)
    sc = s["scales"].double().cpu().numpy()
    for n in range(chunks * 128 // c["group"]):
        w[:, n * c["group"]:(n + 1) * c["group"]] *= sc[:, n].reshape(-1, 1)
    w = torch.from_numpy(w[:c["out"], :c["inner"]]).to(s["x"].device)
    y = s["x"].double() @ w.t() + s["bias"].double()
    if c["gelu"]:
        y = y / 2 * torch.special.erfc(-y / math.sqrt(2))
    return y
