"""Linear layers with 4-bit weights: e2m1 codes with a bf16 scale for every group of 32, 64 or 128 columns of a row.

For decode steps of few rows, which are bound by reading the weights: an eighth of the fp32 bytes.  ``quantize_w4`` lays a weight out once,
``w4_linear`` is the product (``sealnn_w4_linear``, include/sealnn.h): the activations enter at full precision -- what 4 bits cost is the
rounding of the weights alone."""
from typing import Optional

import torch

from ._lib import launch, lib, refuse_gradient

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


class W4Weight:
    """A weight [out_features, in_features] as ``codes`` [ceil(out / 16), ceil(in / 128), 4, 16, 4, 4] uint8 and ``scales`` [ceil(out / 16), ceil(in / 128) * 128 / group,
    16] bf16 (include/sealnn.h says which byte is what)."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, out_features: int, in_features: int):
        tiles, chunks = -(-out_features // 16), -(-in_features // 128)
        if out_features < 1 or in_features < 1 or codes.dtype != torch.uint8 or codes.shape != (tiles, chunks, 4, 16, 4, 4):
            raise ValueError(f"W4Weight: the codes of a {out_features} x {in_features} weight are uint8 {(tiles, chunks, 4, 16, 4, 4)}, got {codes.dtype} {tuple(codes.shape)}")
        if scales.dtype != torch.bfloat16 or scales.dim() != 3 or scales.shape[0] != tiles or scales.shape[2] != 16 or scales.shape[1] not in (chunks, 2 * chunks, 4 * chunks):
            raise ValueError(f"W4Weight: the scales are bf16 [{tiles}, {chunks} * 128 / group, 16] with a group of 32, 64 or 128, got {scales.dtype} {tuple(scales.shape)}")
        if not codes.is_contiguous() or not scales.is_contiguous() or codes.device != scales.device:
            raise ValueError("W4Weight: codes and scales must be contiguous and on one device")
        self.codes, self.scales, self.out_features, self.in_features = codes, scales, out_features, in_features
        self.group = chunks * 128 // scales.shape[1]

    def dequantize(self) -> torch.Tensor:
        """the weight that the codes stand for, fp32 [out_features, in_features]"""
        c = self.codes
        nib = torch.stack([c & 15, c >> 4], -1).long()
        w = torch.tensor(E2M1 + tuple(-x for x in E2M1), device=c.device)[nib].permute(0, 3, 1, 4, 2, 5, 6).reshape(c.shape[0] * 16, c.shape[1] * 128)
        s = self.scales.float().transpose(1, 2).reshape(w.shape[0], -1, 1)
        return (w.view(w.shape[0], -1, self.group) * s).view_as(w)[:self.out_features, :self.in_features]


@torch.no_grad()
def quantize_w4(weight: torch.Tensor, group: int = 32) -> W4Weight:
    """Round a weight [out, in] to the nearest e2m1 multiples of its groups' scales; a scale is the group's largest magnitude / 6, rounded to bf16.  Ties go to the
    code with the even last bit.  Any device."""
    if weight.dim() != 2 or group not in (32, 64, 128):
        raise ValueError(f"quantize_w4: a weight [out, in] and a group of 32, 64 or 128, got {tuple(weight.shape)} and {group}")
    N, K = weight.shape
    Np, Kp = -(-N // 16) * 16, -(-K // 128) * 128
    w = torch.zeros(Np, Kp, dtype=torch.float32, device=weight.device)
    w[:N, :K] = weight
    if not bool(torch.isfinite(w).all()):
        raise ValueError("quantize_w4: the weight holds infinities or NaN, or numbers beyond fp32")
    g = w.view(Np, Kp // group, group)
    s = (g.abs().amax(-1) / 6).to(torch.bfloat16)
    y = (g / torch.where(s > 0, s, 1.0).float().unsqueeze(-1)).view(Np, Kp)      # (a scale of 0: every multiple is 0)
    mag = y.abs()
    lut = torch.tensor(E2M1, device=w.device)
    mid = (lut[1:] + lut[:-1]) / 2
    code = torch.bucketize(mag, mid)                                   # (a tie goes to the lower code ...)
    tie = (code < 7) & (mag == mid[code.clamp(max=6)]) & (code % 2 == 1)
    code = (code + tie.long()).to(torch.uint8)                          # (... unless that is odd)
    code = torch.where(mag > 0, code, torch.zeros_like(code)) | ((y < 0).to(torch.uint8) << 3)
    c = code.view(Np // 16, 16, Kp // 128, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 5, 6)
    return W4Weight((c[..., 0] | (c[..., 1] << 4)).contiguous(), s.view(Np // 16, 16, Kp // group).transpose(1, 2).contiguous(), N, K)


def w4_linear(x: torch.Tensor, weight: W4Weight, bias: Optional[torch.Tensor] = None, gelu: bool = False) -> torch.Tensor:
    """``F.linear(x, weight, bias)`` (and its erf GELU) for ``x`` fp32 or bf16 [rows, in_features], rows may be strided; ``bias`` of x's type.  Made for 1 .. 64 rows (a wide
    bf16 layer, 50265 x 1024, takes 35 us at 60 rows, the library's 16-bit product 20); up to 2^19 work.  Returns a new [rows, out_features] of x's type.  A row of x that is not finite gives
    a row that is not (fp32: NaN; bf16: what inf * w sums to).  No gradient: an input that requires one is refused unless it is called under ``torch.no_grad()``."""
    codes, dt = weight.codes, x.dtype
    if x.dim() != 2 or x.shape[1] != weight.in_features or (dt != torch.float32 and dt != torch.bfloat16) or x.device != codes.device:
        raise ValueError(f"w4_linear: x is fp32 or bf16 [rows, {weight.in_features}] on {codes.device}, got {dt} {tuple(x.shape)} on {x.device}")
    rows, N = x.shape[0], weight.out_features
    row_stride, stride = x.stride()
    if stride != 1 and weight.in_features > 1:
        raise ValueError("w4_linear: the columns of a row of x must be contiguous")
    if bias is not None and (bias.shape != (N,) or bias.dtype != dt or bias.device != x.device or not bias.is_contiguous()):
        raise ValueError(f"w4_linear: the bias is {dt} [{N}], contiguous, on {x.device}")
    if x.requires_grad or (bias is not None and bias.requires_grad):
        refuse_gradient("w4_linear", x, bias)
    if not x.is_cuda:
        raise RuntimeError("w4_linear: x must live on the GPU (seal_amd has no CPU path)")
    y = x.new_empty((rows, N))
    launch(lib().sealnn_w4_linear if dt == torch.float32 else lib().sealnn_w4_linear_bf16, x.get_device(), x.data_ptr(), row_stride, codes.data_ptr(),
           weight.scales.data_ptr(), None if bias is None else bias.data_ptr(), rows, N, weight.in_features, weight.group, gelu, y.data_ptr())
    return y
