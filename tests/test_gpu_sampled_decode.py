"""The operators as a decode runs them: ``fm_index_sample`` (drawing under the FM-index constraint) and ``QuantStepDecoder`` (4-bit weights, 8-bit caches),
alone and together, on seeded models -- against the CPU oracle's masks, HF's forward and the step written out in 64 bits."""
import numpy as np
import pytest
import torch

from tests import quant_refs as ref
from tests.helpers import make_docs, tiny_bart

pytestmark = pytest.mark.gpu
VOCAB = 130


def _index(seed=0, n=40):
    from oracle.seal_oracle import OracleFMIndex
    from seal_amd import FMIndex
    docs = make_docs(seed, n, VOCAB - 8)
    ix, orc = FMIndex(), OracleFMIndex()
    ix.initialize(docs)
    orc.initialize(docs)
    return ix, orc


def _model(**kw):
    return tiny_bart(VOCAB, **{**dict(d_model=128, heads=2, max_positions=160), **kw}).to("cuda:0")


def _inputs(B, S, seed=3):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(4, VOCAB - 8, (B, S), generator=g)
    mask = torch.ones_like(ids)
    for b in range(1, B):
        mask[b, S - 3 * b:] = 0
    return ids.to("cuda:0"), mask.to("cuda:0")


class _Fixed:
    """a decoder whose logits are given"""

    def __init__(self, logits):
        self.logits, self.t, self.logit_bias, self.lm_w = logits, 0, None, logits

    def encode(self, ids, mask):
        return None

    def start(self, *a):
        self.t = 0

    def step(self, tokens, beams_identical=False):
        self.t += 1
        return self.logits[self.t - 1]


@pytest.mark.parametrize("kw", [dict(), dict(force_decoding_from=[5]), dict(always_allow_eos=True), dict(stop_at_count=3), dict(disable_fm_index=True)],
                         ids=["plain", "forced", "eos", "stop", "free"])
def test_sampling_under_the_index_follows_the_oracle(kw):
    """every draw of every row replayed on the host: the oracle's mask for the row's prefix, then the definition of the draw"""
    from oracle.beam_oracle import oracle_logits_mask
    from seal_amd import fm_index_sample
    ix, orc = _index()
    B, K, T = 3, 5, 9
    R = B * K
    g = torch.Generator().manual_seed(7)
    logits = torch.randn(T - 1, R, VOCAB, generator=g) * 2
    logits[:, :, 0] = float("-inf")
    u = torch.rand(T - 1, R, generator=g)
    model = _model()
    cfg = model.config
    ids, mask = _inputs(B, 6)
    settings = dict(temperature=0.8, top_k=40, top_p=0.95, min_p=0.001)
    got = fm_index_sample(model, ix, ids, mask, num_samples=K, max_length=T, u=u.to("cuda:0"), decoder=_Fixed(logits.to("cuda:0")), **settings, **kw)
    assert len(got) == B and all(len(q) == K for q in got)
    got = [s for q in got for s in q]
    okw = {k: v for k, v in kw.items() if k != "disable_fm_index"}
    rows = [[cfg.decoder_start_token_id] for _ in range(R)]
    score, ended = np.zeros(R), [False] * R
    for t in range(1, T):
        padded = [r + [cfg.pad_token_id] * (t - len(r)) for r in rows]
        if kw.get("disable_fm_index"):
            allowed = np.ones((R, VOCAB), dtype=bool)
        else:
            allowed = np.asarray(oracle_logits_mask(orc, padded, VOCAB, K, pad_token_id=cfg.pad_token_id, eos_token_id=cfg.eos_token_id, **okw), dtype=bool)
        for r in range(R):
            if ended[r]:
                continue
            tok, lp = ref.sample(logits[t - 1, r].numpy(), u[t - 1, r].numpy(), allowed=allowed[r], **settings)
            if tok[0] < 0:
                ended[r] = True
                continue
            rows[r].append(int(tok[0]))
            score[r] += lp[0]
            ended[r] = int(tok[0]) == cfg.eos_token_id
    assert [s[1] for s in got] == rows
    assert len({len(r) for r in rows}) > 1 or kw.get("disable_fm_index")
    # T - 1 fp32 additions of log-probabilities that are each within 2^-19 (see the operator's own test) of the definition
    assert np.allclose([s[0] for s in got], score, rtol=(T + 1) * 2.0 ** -24, atol=T * 2.0 ** -19)


@pytest.mark.parametrize("geom", [dict(d_model=32, heads=4), dict(d_model=128, heads=2)], ids=["dh8", "dh64"])
def test_sampled_sequences_are_in_the_corpus_and_scored_by_the_model(geom):
    from seal_amd import fm_index_sample
    ix, _ = _index()
    model = _model(**geom)
    cfg = model.config
    ids, mask = _inputs(3, 10)
    g = torch.Generator(device="cuda:0").manual_seed(5)
    a = fm_index_sample(model, ix, ids, mask, num_samples=6, max_length=8, generator=g, temperature=1.3)
    g.manual_seed(5)
    assert fm_index_sample(model, ix, ids, mask, num_samples=6, max_length=8, generator=g, temperature=1.3) == a
    for q, samples in enumerate(a):
        assert len({tuple(t) for _, t in samples}) > 1
        for score, toks in samples:
            assert toks[0] == cfg.decoder_start_token_id and len(toks) > 1 and cfg.pad_token_id not in toks
            body = toks[1:]
            assert ix.get_count(body) > 0
            with torch.no_grad():
                lg = model(input_ids=ids[q:q + 1], attention_mask=mask[q:q + 1], decoder_input_ids=torch.tensor([toks[:-1]], device="cuda:0")).logits[0]
            lp = torch.log_softmax(lg.double(), -1)
            want = sum(float(lp[i, t]) for i, t in enumerate(body))
            assert abs(score - want) <= 1e-4                      # (the tolerance of hypothesis scores against HF's fp32 forward)


def test_sample_refusals_of_the_loop():
    from seal_amd import fm_index_sample
    ix, _ = _index()
    model = _model()
    ids, mask = _inputs(2, 6)
    for kw in (dict(num_samples=0), dict(max_length=1), dict(u=torch.zeros(3, 2, device="cuda:0")), dict(u=torch.zeros(7, 2, dtype=torch.float64, device="cuda:0"), max_length=8)):
        with pytest.raises(ValueError):
            fm_index_sample(model, ix, ids, mask, **kw)


# ---------------------------------------------------------------------------
# the quantised step
# ---------------------------------------------------------------------------
def _ln(x, m):
    x = x.double()
    mu = x.mean(-1, keepdim=True)
    return (x - mu) / torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + m.eps) * m.weight.double().cpu() + m.bias.double().cpu()


def _act(x):
    return 0.5 * x * torch.special.erfc(-x / 2 ** 0.5)


def _step64(dec, tokens, t, own, cross, cross_mask):
    """one decoder step in 64 bits with the weights that the codes stand for, over the keys and values that the caches hold (position t included);
    also returns every layer's unrounded new keys and values"""
    H, dh, R = dec.h, dec.dh, tokens.numel()

    def lin(x, key, w, b):
        W = dec._w4[key].dequantize() if dec.quantized else w
        return x @ W.double().cpu().t() + b.double().cpu()

    def att(q, k, v, ok):
        s = torch.einsum("rhd,rthd->rht", q, k) * dec.scale
        p = torch.softmax(torch.where(ok[:, None, :], s, -float("inf")), -1)
        return torch.einsum("rht,rthd->rhd", p, v).reshape(R, H * dh)
    x = _ln(dec.embed(tokens).cpu() + dec.pos.weight[t + dec.pos_offset].cpu(), dec.ln_emb)
    new = []
    for i, L in enumerate(dec.layers):
        qkv = lin(x, (id(L), "qkv"), L["qkv_w"], L["qkv_b"]).view(R, 3, H, dh)
        new.append((qkv[:, 1], qkv[:, 2]))
        k, v = (z[:, :t + 1].double().cpu() for z in own[i].values())
        a = att(qkv[:, 0], k, v, torch.ones(R, t + 1, dtype=torch.bool))
        x = _ln(x + lin(a, (id(L), "so"), L["so"].weight, L["so"].bias), L["ln1"])
        q = lin(x, (id(L), "cq"), L["cq"].weight, L["cq"].bias).view(R, H, dh)
        k, v = (z.double().cpu().repeat_interleave(dec.beams, 0) for z in cross[i].values())
        c = att(q, k, v, cross_mask)
        x = _ln(x + lin(c, (id(L), "co"), L["co"].weight, L["co"].bias), L["ln2"])
        h = _act(lin(x, (id(L), "fc1"), L["fc1"].weight, L["fc1"].bias))
        x = _ln(x + lin(h, (id(L), "fc2"), L["fc2"].weight, L["fc2"].bias), L["ln3"])
    return lin(x, "lm", dec.lm_w, dec.lm_b.view(-1)), new


@pytest.mark.parametrize("weights", ["w4", None])
@pytest.mark.parametrize("geom", [dict(d_model=128, heads=2), dict(d_model=128, heads=1)], ids=["dh64", "dh128"])
def test_quantised_step_is_the_step_over_its_codes(weights, geom):
    """inputs of 100 tokens and 40 positions (beyond the fp32 step's 64 and 17).  The logits: fp32 arithmetic of a few thousand terms a value through two
    layers, against 64 bits over the same codes.  The cached keys and values: within e4m3's half step (2^-4 relative, or 2^-10 of the scale below its normal
    range) of the unrounded ones, twice where a growing scale re-encoded them."""
    from seal_amd.quant_decoder import QuantStepDecoder
    model = _model(**geom)
    dec = QuantStepDecoder(model, weights=weights, group=64)
    B, K, S, T = 3, 2, 100, 40
    ids, mask = _inputs(B, S)
    enc = dec.encode(ids, mask)
    dec.start(enc, mask, K, T)
    st = dec._cur
    ok = torch.zeros(B, st.keep.shape[1], dtype=torch.bool)
    ok[:, :S] = mask.cpu() != 0
    ok = ok.repeat_interleave(K, 0)
    kv = [dec._ckv(enc, L).view(B, S, 2, dec.h, dec.dh) for L in dec.layers]
    for c, z in zip(st.cross, kv):
        for got, want in zip(c.values(), (z[:, :, 0], z[:, :, 1])):
            tol = want.abs() * 2.0 ** -4 + 2.0 ** -10 * max(c.k_scale.max().item(), c.v_scale.max().item())
            assert ((got[:, :S] - want).abs() <= tol).all()
    g = torch.Generator().manual_seed(9)
    for t in range(T):
        tokens = torch.randint(4, VOCAB, (B * K,), generator=g).to("cuda:0")
        logits = dec.step(tokens)
        if t not in (0, 1, 15, 16, 39):
            continue
        want, new = _step64(dec, tokens, t, st.own, st.cross, ok)
        fin = torch.isfinite(want)
        assert torch.equal(torch.isfinite(logits.cpu()), fin)
        # (values of order 1 through ~30 fp32 roundings of sums of <= 256 terms: 2^-24 * 256 * 30 is 5e-4; seen: ~2e-6)
        assert (logits.cpu().double() - want)[fin].abs().max() <= 5e-4
        for c, (k, v) in zip(st.own, new):
            for got, w, sc in zip(c.values(), (k, v), (c.k_scale, c.v_scale)):
                tol = w.abs() * 2.0 ** -3 + 2.0 ** -9 * sc.max().item() + 1e-5
                assert ((got[:, t].double().cpu() - w).abs() <= tol).all()
    with pytest.raises(RuntimeError):
        dec.step(tokens)


def test_graph_reorder_and_narrow():
    """the captured step equals the launched one; re-ranked rows carry their history; the queries that stay after ``narrow`` go on as if alone"""
    from seal_amd.quant_decoder import QuantStepDecoder
    model = _model()
    B, K, T = 3, 4, 20
    ids, mask = _inputs(B, 30)
    g = torch.Generator().manual_seed(2)
    toks = [torch.randint(4, VOCAB, (B * K,), generator=g).to("cuda:0") for _ in range(T)]
    perm = torch.cat([torch.randperm(K, generator=g) + K * b for b in range(B)]).to("cuda:0")
    dup = torch.zeros(B * K, dtype=torch.long, device="cuda:0") + torch.arange(B, device="cuda:0").repeat_interleave(K) * K      # (every beam continues the first)

    def run(dec, plan, cuts=(), orders=()):
        out = []
        dec.start(dec.encode(ids, mask), mask, K, T, narrow_plan=plan)
        gone = 0
        for t in range(T):
            out.append(dec.step(toks[t][gone * K:]).clone())
            if t in orders:
                dec.reorder(orders[t][gone * K:] - gone * K)
            if t in cuts:
                dec.narrow(cuts[t])
                gone += cuts[t]
        return out
    plain = QuantStepDecoder(model)
    base = run(plain, ())
    again = run(plain, ())
    assert all(torch.equal(a, b) for a, b in zip(base, again))
    eager = QuantStepDecoder(model)
    eager.use_graph = False
    assert all(torch.equal(a, b) for a, b in zip(base, run(eager, ())))
    cut = run(plain, (1, 2), cuts={3: 1, 9: 1})
    for t in range(T):
        gone = 0 if t <= 3 else 1 if t <= 9 else 2
        assert torch.equal(cut[t], base[t][gone * K:]), t
    assert all(torch.equal(a, b) for a, b in zip(cut, run(plain, (), cuts={3: 1, 9: 1})))           # (not announced)
    moved = run(plain, (), orders={4: perm, 11: dup})
    assert all(torch.equal(a, b) for a, b in zip(moved[:5], base[:5])) and not torch.equal(moved[5], base[5])
    # rows as their own histories would have made them
    hist = [[] for _ in range(B * K)]
    for t in range(5):
        for r in range(B * K):
            hist[r].append(int(toks[t][r]))
    hist = [list(hist[int(p)]) for p in perm]
    dec = QuantStepDecoder(model)
    dec.start(dec.encode(ids, mask), mask, K, T)
    for t in range(5):
        dec.step(torch.tensor([h[t] for h in hist], device="cuda:0"))
    assert torch.equal(dec.step(toks[5]), moved[5])


def test_beam_search_and_sampling_with_the_quantised_step():
    """all of it together: both loops of the framework over ``QuantStepDecoder``, constrained by the index -- hypotheses are n-grams of the corpus, scores are the
    sums of the quantised model's own log-probabilities (its logits, row by row, from a second decoder that is fed the sequence)"""
    from seal_amd import fm_index_generate, fm_index_sample
    from seal_amd.quant_decoder import QuantStepDecoder
    ix, _ = _index()
    model = _model()
    dec = QuantStepDecoder(model)
    ids, mask = _inputs(2, 70)
    K, T = 4, 7
    hyps = fm_index_generate(model, ix, ids, mask, min_length=1, max_length=T, num_beams=K, keep_history=True, decoder=dec)
    drawn = fm_index_sample(model, ix, ids, mask, num_samples=K, max_length=T, temperature=1.2, top_p=0.98, decoder=dec, generator=torch.Generator(device="cuda:0").manual_seed(1))
    check = QuantStepDecoder(model)
    n = 0
    for q in range(2):
        assert len(hyps[q]) > K
        for score, toks in [h for h in hyps[q] if ix.get_count([x for x in h[1][1:]]) > 0][:6] + drawn[q]:
            assert ix.get_count(toks[1:]) > 0
            check.start(check.encode(ids, mask), mask, K, T)
            total = 0.0
            for t, tok in enumerate(toks[1:]):
                lg = check.step(torch.full((2 * K,), toks[t], device="cuda:0"))[q * K]
                total += float(torch.log_softmax(lg.double(), -1)[tok])
            assert abs(score - total) <= 1e-4
            n += 1
    assert n >= 2 * K


def test_quantised_decoder_refusals():
    from seal_amd.quant_decoder import QuantStepDecoder
    with pytest.raises(ValueError):
        QuantStepDecoder(_model(d_model=32, heads=4))
    with pytest.raises(ValueError):
        QuantStepDecoder(_model(), weights="int8")
    with pytest.raises(ValueError):
        QuantStepDecoder(_model().half())
    with pytest.raises(RuntimeError):
        QuantStepDecoder(tiny_bart(VOCAB, d_model=128, heads=2))
    dec = QuantStepDecoder(_model(max_positions=32))
    ids, mask = _inputs(1, 6)
    with pytest.raises(ValueError):
        dec.start(dec.encode(ids, mask), mask, 1, 33)


def test_quantised_step_in_bf16():
    """a bf16 model: the step's activations round to bf16, so its logits sit as far from the 64-bit step over the same codes as a bf16 chain does: 2 x 2^-8 of
    the logits' own size for each of the ~14 roundings on the way"""
    from seal_amd.quant_decoder import QuantStepDecoder
    model = _model().to(torch.bfloat16)
    dec = QuantStepDecoder(model)
    B, K, S, T = 2, 3, 20, 18
    ids, mask = _inputs(B, S)
    dec.start(dec.encode(ids, mask), mask, K, T)
    ok = torch.zeros(B, dec._cur.keep.shape[1], dtype=torch.bool)
    ok[:, :S] = mask.cpu() != 0
    g = torch.Generator().manual_seed(9)
    for t in range(T):
        tokens = torch.randint(4, VOCAB, (B * K,), generator=g).to("cuda:0")
        logits = dec.step(tokens)
    want, _ = _step64(dec, tokens, T - 1, dec._cur.own, dec._cur.cross, ok.repeat_interleave(K, 0))
    fin = torch.isfinite(want)
    assert logits.dtype == torch.float32
    assert (logits.cpu().double() - want)[fin].abs().max() <= 28 * 2.0 ** -8 * want[fin].abs().max()
