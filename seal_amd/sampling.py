"""Drawing tokens from logits on the GPU: temperature, top-k, top-p and min-p, under an optional allowed-token bitmap (the FM-index
constraint of a step, ``IndexBasedLogitsProcessor.allowed_bits``), from random numbers that the caller gives.

``sample_tokens`` is one kernel launch (``sealnn_sample_tokens``, include/sealnn.h); ``fm_index_sample`` (beam_search.py) is the decode loop
around it.  The reference draws with ``torch.multinomial`` over the softmax (reference beam_search.py:296, ``sample=True``)."""
from typing import Optional, Tuple, Union

import torch

from ._lib import check, launch_on, lib

MAX_VOCAB = 1 << 18
Setting = Union[float, int, torch.Tensor]


def _setting(value: Setting, name: str, rows: int, dtype: torch.dtype, like: torch.Tensor):
    """(number, address of a per-row tensor or None) of a sampling parameter"""
    if isinstance(value, torch.Tensor):
        if value.dtype != dtype or value.shape != (rows,) or value.device != like.device or not value.is_contiguous():
            raise ValueError(f"sample_tokens: {name} as a tensor is {dtype}, one value for each of the {rows} rows, contiguous, on {like.device} "
                             f"(got {value.dtype}, {tuple(value.shape)}, {value.device})")
        return 0, value.data_ptr()
    return value, None


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0, allowed_bits: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(tokens, logprobs)``, both shaped like ``u``: int64 and fp32.

    ``logits`` [rows, vocab] fp32 or bf16 (rows may be strided); ``u`` fp32 [rows] or [rows, draws], uniform in [0, 1): the draw is the first
    token, in the order of the vocabulary, whose cumulative weight ``exp(logit / temperature)`` passes ``u * total``.  The weights are those of
    the tokens that ``allowed_bits`` (int32 [rows, >= ceil(vocab / 32)], bit v of a row: token v may be drawn) allows, then of the ``top_k`` largest
    (0: all; of equal logits the lower index is the larger), then of the fewest that hold at least ``top_p`` of the weight left (1: all), then of those with at
    least ``min_p`` of the largest weight (0: all); the largest always stays.  ``temperature`` 0: the first of the largest logits.  Each setting is a number
    for all rows or a tensor with one for each row (fp32; ``top_k`` int32).  NaN logits are never drawn, +inf counts as the largest fp32 number.

    A row of which no token may be drawn gives token -1 and log-probability -inf.  ``logprobs`` are those of the model: ``logit - logsumexp`` of the whole
    row, without temperature, constraint or filters (what the decode loop carries, as the reference's beam scores carry unconstrained ones)."""
    if logits.dim() != 2 or logits.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError(f"sample_tokens: logits are fp32 or bf16 [rows, vocab], got {logits.dtype} {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"sample_tokens: a vocabulary of 1 .. {MAX_VOCAB} tokens, got {vocab}")
    if vocab > 1 and logits.stride(1) != 1:
        raise ValueError("sample_tokens: the logits of a row must be contiguous")
    if rows > 1 and logits.stride(0) < vocab:
        raise ValueError("sample_tokens: the rows of the logits overlap")
    if u.dtype != torch.float32 or u.dim() not in (1, 2) or u.shape[0] != rows or u.device != logits.device:
        raise ValueError(f"sample_tokens: u is fp32 [rows] or [rows, draws] on {logits.device}, got {u.dtype} {tuple(u.shape)} on {u.device}")
    u = u.contiguous()
    if not isinstance(temperature, torch.Tensor) and not 0 <= temperature < float("inf"):
        raise ValueError(f"sample_tokens: temperature = {temperature}")
    if not isinstance(top_k, torch.Tensor) and (top_k < 0 or top_k != int(top_k)):
        raise ValueError(f"sample_tokens: top_k = {top_k}")
    if not isinstance(top_p, torch.Tensor) and not 0 <= top_p <= 1:
        raise ValueError(f"sample_tokens: top_p = {top_p}")
    if not isinstance(min_p, torch.Tensor) and not 0 <= min_p <= 1:
        raise ValueError(f"sample_tokens: min_p = {min_p}")
    t, t_v = _setting(temperature, "temperature", rows, torch.float32, logits)
    k, k_v = _setting(top_k, "top_k", rows, torch.int32, logits)
    p, p_v = _setting(top_p, "top_p", rows, torch.float32, logits)
    m, m_v = _setting(min_p, "min_p", rows, torch.float32, logits)
    bits, bits_stride = None, 0
    if allowed_bits is not None:
        b = allowed_bits
        if (b.dtype != torch.int32 or b.dim() != 2 or b.shape[0] != rows or b.shape[1] < (vocab + 31) // 32 or b.device != logits.device
                or (b.shape[1] > 1 and b.stride(1) != 1)):
            raise ValueError(f"sample_tokens: allowed_bits is int32 [rows, >= {(vocab + 31) // 32}] with contiguous rows on {logits.device}, "
                             f"got {b.dtype} {tuple(b.shape)} on {b.device}")
        bits, bits_stride = b.data_ptr(), b.stride(0)
    if not logits.is_cuda:
        raise RuntimeError("sample_tokens: the logits must live on the GPU (seal_amd has no CPU path)")
    tokens = torch.empty(u.shape, dtype=torch.int64, device=u.device)
    logprobs = torch.empty_like(u)
    fn = lib().sealnn_sample_tokens if logits.dtype == torch.float32 else lib().sealnn_sample_tokens_bf16
    with launch_on(logits) as stream:
        check(fn(stream, logits.data_ptr(), logits.stride(0), rows, vocab, u.data_ptr(), u.shape[1] if u.dim() == 2 else 1, bits, bits_stride,
                 t, min(int(k), MAX_VOCAB), p, m, t_v, k_v, p_v, m_v, tokens.data_ptr(), logprobs.data_ptr()))
    return tokens, logprobs
