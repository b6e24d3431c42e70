"""The decoder step with 4-bit weights and an 8-bit cache: ``BartStepDecoder``'s interface for decodes that the fp32 step is not made for.

``BartStepDecoder``'s fused step holds at most 17 decoder positions and 64 encoder tokens and reads its weights at 16 or 32 bits.  ``QuantStepDecoder`` keeps the
self-attention history and the encoder's keys and values in ``KV8Cache`` (any length, a quarter of the bytes of fp32) and, with ``weights="w4"``, runs every product
of a step through ``w4_linear`` (an eighth of the bytes): for long inputs, long outputs and few rows, where a step is bound by reading them.
BART-large, us a step, fp32 step / this one: 1 row 1324 / 639, 60 rows 1318 / 955, inputs of 1000 tokens 1828 / 689 (1 row) and 4945 / 2066 (300 rows), 200 positions
5508 / 2241 (300 rows) -- but 300 rows of 30 tokens and 16 positions 1570 / 1935, and 1575 / 2496 where a beam search reorders the rows (``reorder`` copies whole caches): such decodes
are the fp32 step's.  Both
round: the scores are those of a model whose weights have 4 and whose keys and values have 8 bits.  The encoder, the projection of its states and the rescoring
forward (``keys.py``) stay what ``BartStepDecoder`` runs.

    decoder = QuantStepDecoder(model)
    fm_index_sample(model, index, input_ids, attention_mask, num_samples=15, decoder=decoder)
    fm_index_generate(model, index, input_ids, attention_mask, keep_history=True, decoder=decoder, ...)
"""
from collections import OrderedDict
from typing import Optional

import torch
import torch.nn.functional as F

from .bart_decoder import BartStepDecoder
from .kv8 import KV8Cache
from .utils import captured, collector_held
from .w4 import quantize_w4, w4_linear


class QuantStepDecoder(BartStepDecoder):
    """``weights``: "w4" (e2m1 with a scale for every ``group`` columns, quantised here, once) or None (the model's own); ``block``: tokens per scale of the cache.
    The model must be fp32 or bf16, on the GPU, with a head_dim of 64 or 128."""

    shared_first_step = False          # (every row is drawn or ranked on its own from the first step on)

    # What the shapes that were decoded keep between decodes (caches, graphs and their logits), the least recently used going first: 300 rows of 1024 positions are 7.5 GB
    # of history at BART-large, 64 positions 0.5 GB, and a graph holds at least the segments of a memory pool of its own.  The shape in use always stays.
    STATE_BYTES, MAX_STATES = 16 << 30, 32

    def __init__(self, model, weights: Optional[str] = "w4", group: int = 32, block: int = 16):
        super().__init__(model)
        w = self.lm_w
        if w.dtype not in self.FUSED_DTYPES or self.dh not in (64, 128):
            raise ValueError(f"QuantStepDecoder: an fp32 or bf16 model with a head_dim of 64 or 128, got {w.dtype} and {self.dh}")
        if weights not in ("w4", None):
            raise ValueError(f"QuantStepDecoder: weights = {weights!r}")
        if not w.is_cuda:
            raise RuntimeError("QuantStepDecoder: the model must live on the GPU (seal_amd has no CPU path)")
        self.block, self.quantized = block, weights is not None
        self._states, self._cur, self._side, self._last_stream = OrderedDict(), None, None, None
        self._w4 = {}
        if self.quantized:
            for L in self.layers:
                for name, m in (("qkv", L["qkv_w"]), ("so", L["so"].weight), ("cq", L["cq"].weight), ("co", L["co"].weight), ("fc1", L["fc1"].weight), ("fc2", L["fc2"].weight)):
                    self._w4[id(L), name] = quantize_w4(m.detach(), group)
            self._w4["lm"] = quantize_w4(w.detach(), group)

    def _product(self, x, key, weight, bias, gelu=False):
        if self.quantized:
            return w4_linear(x, self._w4[key], bias, gelu=gelu)
        return F.linear(x, weight, bias)

    def _in_order(self, dev) -> None:
        """the buffers of a shape go from call to call: one that is made on another stream than the call before waits for what that stream has been given (a caller who
        captures orders its streams itself)"""
        if torch.cuda.is_current_stream_capturing():
            return
        now = torch.cuda.current_stream(dev)
        if self._last_stream is not None and self._last_stream != now:
            now.wait_stream(self._last_stream)
        self._last_stream = now

    # -- one decode's buffers and graph; the narrower continuations of a loop over several decodes are views of them --
    class _State:
        pass

    def _new_state(self, B, K, S, T, dev):
        st = self._State()
        R = B * K
        st.B, st.K = B, K
        st.tokens = torch.zeros(R, dtype=torch.long, device=dev)
        st.t = torch.zeros(1, dtype=torch.long, device=dev)
        st.lengths = torch.zeros(R, dtype=torch.int32, device=dev)
        st.own = [KV8Cache.empty(R, self.h, T, self.dh, block=self.block, device=dev) for _ in self.layers]
        st.cross = [KV8Cache.empty(B, self.h, S, self.dh, block=self.block, device=dev) for _ in self.layers]
        st.cross_lengths = torch.zeros(B, dtype=torch.int32, device=dev)
        st.keep = torch.zeros(B, st.cross[0].tokens, dtype=torch.uint8, device=dev)
        st.dropped, st.graph, st.logits, st.tails = 0, None, None, {}
        return st

    def _state_bytes(self, key, tails=()) -> int:
        """what a shape holds: its caches, and the logits of its graphs (of all rows, and of the queries behind each of ``tails``)"""
        B, K, S, T = key[:4]
        codes = 2 * len(self.layers) * self.h * (B * K * T + B * S)
        return codes * self.dh + codes // self.block * 4 + 4 * self.lm_w.shape[0] * K * (B + sum(B - dropped for dropped in tails))

    def _make_room(self, key, dev) -> None:
        """drop the least recently used shapes that ``key``'s leaves no room for"""
        held = {k: self._state_bytes(k, st.tails) for k, st in self._states.items()}
        held.setdefault(key, self._state_bytes(key))
        total, drop = sum(held.values()), []
        for k in self._states:                       # (the longest unused first)
            if len(held) - len(drop) <= self.MAX_STATES and total <= self.STATE_BYTES:
                break
            if k != key:
                drop.append(k)
                total -= held[k]
        if drop:
            with collector_held():                   # (no graph may be freed under another thread's capture)
                if dev.type == "cuda":
                    torch.cuda.synchronize(dev)      # (a decode on another stream may still use what goes)
                for k in drop:
                    del self._states[k]

    @staticmethod
    def _tail(root, dropped):
        """the state of the queries behind the first ``dropped``"""
        st = QuantStepDecoder._State()
        a = dropped * root.K

        def part(c, n):
            return KV8Cache(c.k[n:], c.v[n:], c.k_scale[n:], c.v_scale[n:])
        st.B, st.K = root.B - dropped, root.K
        st.tokens, st.t, st.lengths = root.tokens[a:], root.t, root.lengths[a:]
        st.own, st.cross = [part(c, a) for c in root.own], [part(c, dropped) for c in root.cross]
        st.cross_lengths, st.keep = root.cross_lengths[dropped:], root.keep[dropped:]
        st.dropped, st.graph, st.logits, st.tails = dropped, None, None, {}
        return st

    def _forward(self, st):
        R, H, dh = st.B * st.K, self.h, self.dh
        x = self.embed(st.tokens) + self.pos.weight.index_select(0, st.t + self.pos_offset)
        x = self.ln_emb(x)
        L_ = self._nn(x.dtype)
        stream = torch.cuda.current_stream(x.device).cuda_stream
        reach = st.lengths + 1

        def add_ln(res, y, ln):
            return self._add_ln(L_, stream, res, y, ln, R, False)[0]
        for L, own, cross in zip(self.layers, st.own, st.cross):
            key = id(L)
            qkv = self._product(x, (key, "qkv"), L["qkv_w"], L["qkv_b"]).view(R, 3, H, dh)
            own.append(qkv[:, 1:2], qkv[:, 2:3], st.lengths)
            a = own.attend(qkv[:, 0], reach, scale=self.scale)
            x = add_ln(x, self._product(a.view(R, self.d), (key, "so"), L["so"].weight, L["so"].bias), L["ln1"])
            q = self._product(x, (key, "cq"), L["cq"].weight, L["cq"].bias).view(R, H, dh)
            c = cross.attend(q, st.cross_lengths, beams=st.K, keep=st.keep, scale=self.scale)
            x = add_ln(x, self._product(c.view(R, self.d), (key, "co"), L["co"].weight, L["co"].bias), L["ln2"])
            erf_gelu = type(L["act"]).__name__ in ("GELUActivation", "GELU") and getattr(L["act"], "approximate", "none") == "none"
            if self.quantized and erf_gelu:
                h = self._product(x, (key, "fc1"), L["fc1"].weight, L["fc1"].bias, gelu=True)
            else:
                h = L["act"](self._product(x, (key, "fc1"), L["fc1"].weight, L["fc1"].bias))
            x = add_ln(x, self._product(h, (key, "fc2"), L["fc2"].weight, L["fc2"].bias), L["ln3"])
        st.t.add_(1)
        st.lengths.add_(1)
        bias = self.lm_b.view(-1)
        return self._product(x, "lm", self.lm_w, bias if bias.dtype == x.dtype else bias.to(x.dtype)).float()

    def _capture(self, st, dev):
        """warm up, then capture (both write the caches: the caller resets the lengths, and a block starts over with its first token)"""
        with torch.inference_mode(False), torch.no_grad():
            side = self._side
            if side is None or side.device != dev:
                side = self._side = torch.cuda.Stream(device=dev)
            side.wait_stream(torch.cuda.current_stream(dev))
            with torch.cuda.stream(side):
                for _ in range(2):
                    st.t.zero_()
                    st.lengths.zero_()
                    self._forward(st)
            torch.cuda.current_stream(dev).wait_stream(side)
            g = torch.cuda.CUDAGraph()
            # (on a stream of the model's device: torch's own capture stream is on the device that was current when it was made, and what runs elsewhere is not captured)
            with captured(g, stream=side, capture_error_mode="thread_local"):
                st.logits = self._forward(st)
            st.graph = g

    @torch.no_grad()
    def start(self, enc_hidden: torch.Tensor, attention_mask: torch.Tensor, num_beams: int, max_len: int, narrow_plan=()) -> None:
        B, S, _ = enc_hidden.shape
        dev = enc_hidden.device
        if max_len + self.pos_offset > self.pos.weight.shape[0]:
            raise ValueError(f"QuantStepDecoder: {max_len} positions, the model has {self.pos.weight.shape[0] - self.pos_offset}")
        self.batch, self.beams, self.rows, self.max_len, self.t = B, num_beams, B * num_beams, max_len, 0
        S64, T64 = -(-S // 64) * 64, -(-max_len // 64) * 64
        key = (B, num_beams, S64, T64, enc_hidden.dtype, str(dev))
        self._in_order(dev)
        self._root = self._cur = None                # (the last decode is over: its shape may go)
        self._make_room(key, dev)
        st = self._states.get(key)
        if st is None:
            with torch.inference_mode(False):
                st = self._states[key] = self._new_state(B, num_beams, S64, T64, dev)
        self._states.move_to_end(key)
        for dropped in narrow_plan:
            if dropped not in st.tails:
                st.tails[dropped] = self._tail(st, dropped)
        if self.use_graph:
            for s in [st] + [st.tails[d] for d in narrow_plan]:
                if s.graph is None:
                    self._capture(s, dev)
        st.t.zero_()
        st.lengths.zero_()
        st.keep.zero_()
        st.keep[:, :S] = attention_mask != 0
        st.cross_lengths.copy_((torch.arange(1, S + 1, device=dev, dtype=torch.int32) * (attention_mask != 0)).amax(1))       # up to the last token that counts
        first = torch.zeros(B, dtype=torch.int32, device=dev)
        for L, cross in zip(self.layers, st.cross):
            kv = self._ckv(enc_hidden, L).view(B, S, 2, self.h, self.dh)
            cross.append(kv[:, :, 0], kv[:, :, 1], first)
        self._root = self._cur = st

    @torch.no_grad()
    def step(self, tokens: torch.Tensor, beams_identical: bool = False) -> torch.Tensor:
        """tokens [rows] at the next position -> next-token logits [rows, vocab] (fp32; the buffer of a graph: valid until the next step)"""
        st = self._cur
        if self.t >= self.max_len:
            raise RuntimeError(f"QuantStepDecoder: a decode of {self.max_len} positions is over")
        self._in_order(st.tokens.device)
        st.tokens.copy_(tokens)
        if st.graph is not None:
            st.graph.replay()
            logits = st.logits
        else:
            logits = self._forward(st)
        self.t += 1
        if self.logit_bias is not None:
            logits = (logits.view(st.B, st.K, -1) + self.logit_bias[:, None, :]).view(st.B * st.K, -1)
        return logits

    @torch.no_grad()
    def reorder(self, beam_idx: torch.Tensor) -> None:
        """new row r continues old row beam_idx[r] (HF ``_reorder_cache``): the rows' codes move"""
        self._in_order(beam_idx.device)
        for own in self._cur.own:
            own.reorder(beam_idx)

    @torch.no_grad()
    def narrow(self, nq: int) -> None:
        if nq <= 0:
            return
        dropped = self._cur.dropped + nq
        if dropped not in self._root.tails:
            self._root.tails[dropped] = self._tail(self._root, dropped)        # (not announced to ``start``: launched eagerly)
        self._cur = self._root.tails[dropped]
        self.batch -= nq
        self.rows = self.batch * self.beams
        if self.logit_bias is not None:
            self.logit_bias = self.logit_bias[nq:]

    def step_buffers(self):
        return None, None

    def steps_are_library_free(self) -> bool:
        return False
