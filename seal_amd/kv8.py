"""A key / value cache in 8 bits for decode steps: e4m3 codes with a power-of-two scale for every block of tokens and head.

``KV8Cache.append`` writes the keys and values of new tokens (a prompt's or encoder's states, or one token of a step) and ``attend`` is the
attention of single positions over it: ``sealnn_kv8_append`` / ``sealnn_kv8_attend`` of include/sealnn.h, where the rounding is defined.  The
cross-attention of a decode (the ``beams`` rows of a query share its encoder states), the self-attention over a row's own history and query heads
that share a cached head are the same call.  ``QuantStepDecoder`` (quant_decoder.py) decodes with it."""
from typing import Optional

import torch

from ._lib import launch, lib, refuse_gradient, uint64s

TILE = 64                                  # tokens of a tile of the layout
# Workgroups (of four waves) that a call splits long slots into when it has few: one a CU is enough for many items (32 slots x 8 heads of up to 8192 tokens: 79 us, in two
# parts 84), two a CU are better where every item is split anyway (1 slot x 16 heads of 32001 tokens: 16 parts 19.0 us, 32 18.0, 64 19.3).  Short caches are not split: the
# second launch and the workspace cost a caller 4 us (1 slot x 16 heads of 512 tokens: 8.3 us a call, split 12.2; in a graph 6.5 / 7.5; of 2048 tokens 16.0 / 12.1, 15.7 / 8.1)
ITEMS_ENOUGH, PARTS_WANTED, SPLIT_TOKENS = 256, 512, 1024


class KV8Cache:
    """``k`` [slots, heads, T, head_dim] and ``v`` [slots, heads, T / 64, head_dim, 64] uint8 (e4m3 codes; token 16 j + 4 g + r of a tile at place
    16 g + 4 j + r), ``k_scale`` / ``v_scale`` [slots, heads, T / block] fp32 powers of two.  T a multiple of 64, head_dim 64 or 128, block 16, 32 or 64.
    ``KV8Cache.empty`` makes the buffers.  For serving: ``append`` and ``attend`` have no gradient, and refuse inputs that require one unless called under
    ``torch.no_grad()``."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        shape, blocks = k.shape, k_scale.shape
        if len(shape) != 4 or shape[3] not in (64, 128) or shape[2] % TILE or not shape[2]:
            raise ValueError(f"KV8Cache: k is [slots, heads, T, head_dim] with T a multiple of {TILE} and head_dim 64 or 128, got {tuple(shape)}")
        S, H, T, D = shape
        if v.shape != (S, H, T // TILE, D, TILE):
            raise ValueError(f"KV8Cache: v is {(S, H, T // TILE, D, TILE)}, got {tuple(v.shape)}")
        if len(blocks) != 3 or blocks[0] != S or blocks[1] != H or blocks != v_scale.shape or blocks[2] not in (T // 16, T // 32, T // 64):
            raise ValueError(f"KV8Cache: the scales are [{S}, {H}, T / block] with a block of 16, 32 or 64 tokens, got {tuple(blocks)} and {tuple(v_scale.shape)}")
        if k.dtype != torch.uint8 or v.dtype != torch.uint8 or k_scale.dtype != torch.float32 or v_scale.dtype != torch.float32:
            raise ValueError("KV8Cache: codes are uint8 and scales fp32")
        dev = k.device
        if not (k.is_contiguous() and v.is_contiguous() and k_scale.is_contiguous() and v_scale.is_contiguous()
                and dev == v.device == k_scale.device == v_scale.device):
            raise ValueError("KV8Cache: the four tensors must be contiguous and on one device")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.slots, self.heads, self.tokens, self.head_dim, self.block, self.device = S, H, T, D, T // blocks[2], dev

    @classmethod
    def empty(cls, slots: int, heads: int, tokens: int, head_dim: int = 64, block: int = 16, device="cuda") -> "KV8Cache":
        """a cache for ``tokens`` tokens of every slot (rounded up to whole tiles), all codes 0"""
        if block not in (16, 32, 64):
            raise ValueError(f"KV8Cache: a block of 16, 32 or 64 tokens, got {block}")
        T = max(TILE, (tokens + TILE - 1) // TILE * TILE)
        return cls(torch.zeros(slots, heads, T, head_dim, dtype=torch.uint8, device=device),
                   torch.zeros(slots, heads, T // TILE, head_dim, TILE, dtype=torch.uint8, device=device),
                   torch.full((slots, heads, T // block), 2.0 ** -64, device=device), torch.full((slots, heads, T // block), 2.0 ** -64, device=device))

    def _lengths(self, t: torch.Tensor, name: str):
        if t.dtype != torch.int32 or t.dim() != 1 or t.shape[0] != self.slots or t.device != self.device or not t.is_contiguous():
            raise ValueError(f"KV8Cache: {name} is int32 [{self.slots}], contiguous, on {self.device}; got {t.dtype} {tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def _on_gpu(self) -> int:
        if not self.k.is_cuda:
            raise RuntimeError("KV8Cache: the cache must live on the GPU (seal_amd has no CPU path)")
        return self.k.get_device()

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor, lengths: torch.Tensor, counts: Optional[torch.Tensor] = None) -> None:
        """Write ``k_new`` / ``v_new`` [slots, n, heads, head_dim] (fp32 or bf16; any strides, dims contiguous) at positions ``lengths[slot]`` .. of every
        slot: all n tokens, or the first ``counts[slot]`` of them.  What would lie behind the cache's end is dropped.  ``lengths`` (int32 [slots], on the
        device) is left as it is: the caller counts."""
        shape, dt = k_new.shape, k_new.dtype
        if (len(shape) != 4 or shape[0] != self.slots or shape[2] != self.heads or shape[3] != self.head_dim or v_new.shape != shape or v_new.dtype != dt
                or k_new.device != self.device or v_new.device != self.device):
            raise ValueError(f"KV8Cache.append: keys and values are [{self.slots}, n, {self.heads}, {self.head_dim}] of one type on {self.device}, "
                             f"got {dt} {tuple(shape)} on {k_new.device} and {v_new.dtype} {tuple(v_new.shape)} on {v_new.device}")
        if dt != torch.float32 and dt != torch.bfloat16:
            raise ValueError(f"KV8Cache.append: fp32 or bf16, got {dt}")
        ks, vs = k_new.stride(), v_new.stride()
        if ks[3] != 1 or vs[3] != 1:
            raise ValueError("KV8Cache.append: the dims of a head must be contiguous")
        if k_new.requires_grad or v_new.requires_grad:
            refuse_gradient("KV8Cache.append", k_new, v_new)
        lengths_ptr, counts_ptr = self._lengths(lengths, "lengths"), None if counts is None else self._lengths(counts, "counts")
        launch(lib().sealnn_kv8_append if dt == torch.float32 else lib().sealnn_kv8_append_bf16, self._on_gpu(), k_new.data_ptr(), v_new.data_ptr(),
               uint64s(ks[0], ks[1], ks[2], vs[0], vs[1], vs[2]), shape[1], lengths_ptr, counts_ptr, self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(),
               self.v_scale.data_ptr(), self.slots, self.heads, self.tokens, self.block, self.head_dim)

    def attend(self, q: torch.Tensor, lengths: torch.Tensor, beams: int = 1, keep: Optional[torch.Tensor] = None,
               scale: Optional[float] = None) -> torch.Tensor:
        """softmax(scale q K^T) V: ``q`` [slots * beams, q_heads, head_dim] (fp32 or bf16; rows and heads may be strided; row r reads slot r // beams, head h
        reads cached head h // (q_heads / heads)) over the first ``lengths[slot]`` tokens, those of them for which ``keep`` (bool or uint8 [slots, T]) is set.
        ``scale`` defaults to head_dim ** -0.5.  A row with nothing to attend to is zeros.  Returns a new tensor shaped and typed like ``q``."""
        D, H, shape, dt = self.head_dim, self.heads, q.shape, q.dtype
        if (len(shape) != 3 or beams < 1 or shape[0] != self.slots * beams or shape[2] != D or shape[1] % H or not shape[1]
                or (dt != torch.float32 and dt != torch.bfloat16) or q.device != self.device):
            raise ValueError(f"KV8Cache.attend: q is fp32 or bf16 [{self.slots} * beams, a multiple of {H}, {D}] on {self.device}, "
                             f"got {dt} {tuple(shape)} on {q.device}")
        row_stride, head_stride, stride = q.stride()
        if stride != 1:
            raise ValueError("KV8Cache.attend: the dims of a head must be contiguous")
        if q.requires_grad:
            refuse_gradient("KV8Cache.attend", q)
        share = shape[1] // H
        keep_ptr, keep_stride = None, 0
        if keep is not None:
            if keep.shape != (self.slots, self.tokens) or keep.dtype not in (torch.bool, torch.uint8) or keep.device != self.device:
                raise ValueError(f"KV8Cache.attend: keep is bool or uint8 [{self.slots}, {self.tokens}] on {self.device}, got {keep.dtype} {tuple(keep.shape)}")
            keep = keep.contiguous()
            if keep.data_ptr() & 3:                  # (the kernel reads four tokens' bytes as a word: a view that starts between words is copied)
                keep = keep.clone()
            keep_ptr, keep_stride = keep.data_ptr(), self.tokens
        lengths_ptr, index = self._lengths(lengths, "lengths"), self._on_gpu()
        out = q.new_empty(shape)
        items = self.slots * H * ((beams * share + 15) // 16)
        splits = 1 if self.tokens < SPLIT_TOKENS or items >= ITEMS_ENOUGH or not items else max(1, min(self.tokens // TILE // 4, PARTS_WANTED // items))
        work, work_floats = None, 0
        if splits > 1:
            work_floats = shape[0] * shape[1] * splits * (D + 4)
            work = torch.empty(work_floats, dtype=torch.float32, device=self.device)
        launch(lib().sealnn_kv8_attend if dt == torch.float32 else lib().sealnn_kv8_attend_bf16, index, q.data_ptr(), row_stride, head_stride, self.k.data_ptr(),
               self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr(), lengths_ptr, keep_ptr, keep_stride, self.slots, beams, H, share, self.tokens,
               self.block, D, D ** -0.5 if scale is None else scale, splits, None if work is None else work.data_ptr(), work_floats * 4, out.data_ptr())
        return out

    def values(self):
        """(keys, values) as fp32 [slots, T, heads, head_dim]: the numbers that the codes stand for"""
        S, H, T, D = self.k.shape

        def scaled(codes, scale):
            x = codes.view(torch.float8_e4m3fn).float().view(S, H, scale.shape[2], self.block, D) * scale[..., None, None]
            return x.view(S, H, T, D).transpose(1, 2)
        v = self.v.view(S, H, T // TILE, D, 4, 4, 4).permute(0, 1, 2, 5, 4, 6, 3).reshape(S, H, T, D)
        return scaled(self.k, self.k_scale), scaled(v, self.v_scale)

    def reorder(self, rows: torch.Tensor) -> None:
        """slot i continues what slot ``rows[i]`` held (HF ``_reorder_cache``); ``rows`` int64 or int32 [slots], on the device, each 0 .. slots - 1"""
        if rows.shape != (self.slots,) or rows.dtype not in (torch.int64, torch.int32) or rows.device != self.device:
            raise ValueError(f"KV8Cache.reorder: rows are int64 or int32 [{self.slots}] on {self.device}, got {rows.dtype} {tuple(rows.shape)} on {rows.device}")
        for t in (self.k, self.v, self.k_scale, self.v_scale):
            t.copy_(t.index_select(0, rows))
