"""Drawing tokens from logits on the GPU: temperature, top-k, top-p and min-p, under an optional allowed-token bitmap (the FM-index
constraint of a step, ``IndexBasedLogitsProcessor.allowed_bits``), from random numbers that the caller gives.

``sample_tokens`` calls the library once (``sealnn_sample_tokens``, include/sealnn.h: one kernel, or three for few rows of a large vocabulary); ``fm_index_sample`` (beam_search.py) is the decode loop
around it.  The reference draws with ``torch.multinomial`` over the softmax (reference beam_search.py:296, ``sample=True``)."""
from typing import Optional, Tuple, Union

import torch

from ._lib import launch, lib, refuse_gradient

MAX_VOCAB = 1 << 18
# Few rows of a large vocabulary are spread over the card by three kernels instead of one workgroup each (include/sealnn.h).  us, one kernel / three, fp32, top-p 0.9: 1 x 16384
# 24.1 / 23.6, 1 x 50265 39.7 / 24.7, 32 x 50265 41 / 28, 128 x 50265 42.6 / 42.1, 1 x 131072 66 / 25; top-k 50: 1 x 50265 16.3 / 15.8, 32 x 50265 17.2 / 17.7, 32 x 131072 23.2 / 22.3
# (where every token has to be weighed -- no top-k, no min-p -- it pays up to twice the rows: 64 x 50265 top-p 0.9 41.5 / 34.1, without a filter 34.8 / 24.1,
# under a bitmap 28.6 / 28.6, but 128 x 50265 under a bitmap 29.4 / 35.3)
SPLIT_VOCAB, SPLIT_ROWS = 32768, 32
Setting = Union[float, int, torch.Tensor]


def _per_row(value: torch.Tensor, name: str, rows: int, dtype: torch.dtype, device) -> int:
    """the address of a sampling parameter that every row has its own of"""
    if value.dtype != dtype or value.shape != (rows,) or value.device != device or not value.is_contiguous():
        raise ValueError(f"sample_tokens: {name} as a tensor is {dtype}, one value for each of the {rows} rows, contiguous, on {device} "
                         f"(got {value.dtype}, {tuple(value.shape)}, {value.device})")
    return value.data_ptr()


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Setting = 1.0, top_k: Setting = 0, top_p: Setting = 1.0,
                  min_p: Setting = 0.0, allowed_bits: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """``(tokens, logprobs)``, both shaped like ``u``: int64 and fp32.

    ``logits`` [rows, vocab] fp32 or bf16 (rows may be strided); ``u`` fp32 [rows] or [rows, draws], uniform in [0, 1): the draw is the first
    token, in the order of the vocabulary, whose cumulative weight ``exp(logit / temperature)`` passes ``u * total``.  The weights are those of
    the tokens that ``allowed_bits`` (int32 [rows, >= ceil(vocab / 32)], bit v of a row: token v may be drawn) allows, then of the ``top_k`` largest
    (0: all; of equal logits the lower index is the larger), then of the fewest that hold at least ``top_p`` of the weight left (1: all), then of those with at
    least ``min_p`` of the largest weight (0: all); the largest always stays.  A weight below 2^-45 of the largest is none: its token is not drawn.  ``temperature`` 0: the first of the largest logits.  Each setting is a number
    for all rows or a tensor with one for each row (fp32; ``top_k`` int32).  NaN logits are never drawn, +inf counts as the largest fp32 number.

    A row of which no token may be drawn gives token -1 and log-probability -inf.  ``logprobs`` are those of the model: ``logit - logsumexp`` of the whole
    row, without temperature, constraint or filters (what the decode loop carries, as the reference's beam scores carry unconstrained ones).  No gradient: logits that require one are refused unless it is
    called under ``torch.no_grad()``."""
    dt, shape, dev, u_shape = logits.dtype, logits.shape, logits.device, u.shape
    if len(shape) != 2 or (dt != torch.float32 and dt != torch.bfloat16):
        raise ValueError(f"sample_tokens: logits are fp32 or bf16 [rows, vocab], got {dt} {tuple(shape)}")
    rows, vocab = shape
    if not 0 < vocab <= MAX_VOCAB:
        raise ValueError(f"sample_tokens: a vocabulary of 1 .. {MAX_VOCAB} tokens, got {vocab}")
    row_stride, stride = logits.stride()
    if stride != 1 and vocab > 1:
        raise ValueError("sample_tokens: the logits of a row must be contiguous")
    if row_stride < vocab and rows > 1:
        raise ValueError("sample_tokens: the rows of the logits overlap")
    if u.dtype != torch.float32 or not 0 < len(u_shape) < 3 or u_shape[0] != rows or u.device != dev:
        raise ValueError(f"sample_tokens: u is fp32 [rows] or [rows, draws] on {dev}, got {u.dtype} {tuple(u_shape)} on {u.device}")
    if logits.requires_grad:
        refuse_gradient("sample_tokens", logits)
    u = u.contiguous()
    t = k = p = m = 0
    t_v = k_v = p_v = m_v = None
    if isinstance(temperature, torch.Tensor):
        t_v = _per_row(temperature, "temperature", rows, torch.float32, dev)
    elif 0 <= temperature < float("inf"):
        t = temperature
    else:
        raise ValueError(f"sample_tokens: temperature = {temperature}")
    if isinstance(top_k, torch.Tensor):
        k_v = _per_row(top_k, "top_k", rows, torch.int32, dev)
    elif top_k >= 0 and top_k == int(top_k):
        k = min(int(top_k), MAX_VOCAB)
    else:
        raise ValueError(f"sample_tokens: top_k = {top_k}")
    if isinstance(top_p, torch.Tensor):
        p_v = _per_row(top_p, "top_p", rows, torch.float32, dev)
    elif 0 <= top_p <= 1:
        p = top_p
    else:
        raise ValueError(f"sample_tokens: top_p = {top_p}")
    if isinstance(min_p, torch.Tensor):
        m_v = _per_row(min_p, "min_p", rows, torch.float32, dev)
    elif 0 <= min_p <= 1:
        m = min_p
    else:
        raise ValueError(f"sample_tokens: min_p = {min_p}")
    bits, bits_stride = None, 0
    if allowed_bits is not None:
        b_shape = allowed_bits.shape
        if (allowed_bits.dtype != torch.int32 or len(b_shape) != 2 or b_shape[0] != rows or b_shape[1] < (vocab + 31) // 32 or allowed_bits.device != dev
                or (allowed_bits.stride(1) != 1 and b_shape[1] > 1)):
            raise ValueError(f"sample_tokens: allowed_bits is int32 [rows, >= {(vocab + 31) // 32}] with contiguous rows on {dev}, "
                             f"got {allowed_bits.dtype} {tuple(b_shape)} on {allowed_bits.device}")
        bits, bits_stride = allowed_bits.data_ptr(), allowed_bits.stride(0)
    if not logits.is_cuda:
        raise RuntimeError("sample_tokens: the logits must live on the GPU (seal_amd has no CPU path)")
    tokens, logprobs = u.new_empty(u_shape, dtype=torch.int64), u.new_empty(u_shape)
    work, work_bytes = None, 0
    if vocab >= SPLIT_VOCAB and rows <= (SPLIT_ROWS if k or m or k_v is not None or m_v is not None or (t_v is None and not t) else 2 * SPLIT_ROWS):
        work_bytes = rows * (-(-vocab // 1024) * 96 + 16448)
        work = torch.empty(work_bytes, dtype=torch.uint8, device=dev)
    launch(lib().sealnn_sample_tokens if dt == torch.float32 else lib().sealnn_sample_tokens_bf16, logits.get_device(), logits.data_ptr(), row_stride, rows, vocab,
           u.data_ptr(), u_shape[1] if len(u_shape) == 2 else 1, bits, bits_stride, t, k, p, m, t_v, k_v, p_v, m_v, tokens.data_ptr(), logprobs.data_ptr(),
           None if work is None else work.data_ptr(), work_bytes)
    return tokens, logprobs
