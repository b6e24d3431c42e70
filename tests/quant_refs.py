"""The operators of the quantised, sampled decode written out in 64 bits on the CPU, straight from their definitions (include/sealnn.h): what
tests/test_quant_ops.py and tests/test_gpu_quant_ops.py hold the kernels to."""
import math

import numpy as np
import torch

E2M1 = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6])


def place(token):
    """where token 0 .. 63 of a tile stands in a row of V"""
    return token % 16 // 4 * 16 + token // 16 * 4 + token % 4


def e4m3(y):
    """to the nearest e4m3 value, ties to even; |y| <= 448 or NaN"""
    y = np.asarray(y, dtype=np.float64)
    _, e = np.frexp(np.where(np.isnan(y), 0, y))
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.rint(y / step) * step


def exponent_for(amax):
    e = -64
    while amax > 448 * 2.0 ** e:
        e += 1
    return e


class Cache:
    """values [slots][heads][T][dh] as codes (numbers on the e4m3 grid) and exponents [slots][heads][T / block], keys and values alike"""

    def __init__(self, codes, scale, block):
        self.codes, self.scale, self.block = np.array(codes, dtype=np.float64), np.array(scale, dtype=np.float64), block

    def append(self, new, lengths, counts=None):
        new = np.asarray(new, dtype=np.float64)
        S, H, T, D = self.codes.shape
        for s in range(S):
            n = new.shape[1] if counts is None else min(int(counts[s]), new.shape[1])
            at, end = int(lengths[s]), min(int(lengths[s]) + n, T)
            while at < end and at >= 0:
                b = at // self.block
                stop = min(end, (b + 1) * self.block)
                for h in range(H):
                    x = new[s, at - int(lengths[s]):stop - int(lengths[s]), h]
                    fin = np.abs(x[np.isfinite(x)])
                    e = exponent_for(fin.max() if fin.size else 0.0)
                    if at > b * self.block:
                        old = self.scale[s, h, b]
                        e = max(e, int(np.log2(old)))
                        held = self.codes[s, h, b * self.block:at]
                        self.codes[s, h, b * self.block:at] = e4m3(held * old / 2.0 ** e) if old != 2.0 ** e else held
                    self.scale[s, h, b] = 2.0 ** e
                    self.codes[s, h, at:stop] = e4m3(np.clip(x / 2.0 ** e, -448, 448))
                at = stop

    def values(self):
        return self.codes * np.repeat(self.scale, self.block, axis=2)[..., None]


def attend(q, k, v, lengths, beams, keep=None, scale=None):
    """q [slots * beams, q_heads, dh], k / v [slots][heads][T][dh] float64 -> (out, bound on |s|-errors' inputs: sum |q||k| scale, largest |v|)"""
    q = np.asarray(q, dtype=np.float64)
    S, H, T, D = k.shape
    share = q.shape[1] // H
    scale = D ** -0.5 if scale is None else scale
    out, mag, vmax = np.zeros_like(q), np.zeros(q.shape[:2]), np.zeros(q.shape[:2])
    for r in range(q.shape[0]):
        s = r // beams
        at = np.arange(min(max(int(lengths[s]), 0), T))
        if keep is not None:
            at = at[np.asarray(keep)[s, at] != 0]
        if not at.size:
            continue
        for h in range(q.shape[1]):
            kk, vv = k[s, h // share, at], v[s, h // share, at]
            sc = kk @ q[r, h] * scale
            p = np.exp(sc - sc.max())
            out[r, h] = p @ vv / p.sum()
            mag[r, h] = (np.abs(kk) @ np.abs(q[r, h])).max() * scale
            vmax[r, h] = np.abs(vv).max()
    return out, mag, vmax


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, allowed=None):
    """one row: (tokens, logprobs)"""
    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, float(torch.finfo(torch.float32).max)))
    u = np.atleast_1d(np.asarray(u, dtype=np.float64))
    ok = np.isfinite(x) if allowed is None else np.isfinite(x) & allowed
    at = np.flatnonzero(ok)
    if not at.size:
        return np.full(u.shape, -1), np.full(u.shape, -np.inf)
    order = sorted(at, key=lambda i: (-x[i], i))
    f32 = lambda t: float(np.float32(t))  # noqa: E731
    if f32(temperature) <= 0:
        order, w = order[:1], np.ones(1)
    else:
        w = np.exp((x[order] - x[order[0]]) / f32(temperature))
        n = len(order) if top_k <= 0 else min(len(order), top_k)
        if top_p < 1:
            mass = np.cumsum(w[:n])
            n = max(1, int(np.searchsorted(mass, f32(top_p) * mass[-1], side="left")) + 1)
        n = min(n, max(1, int((w >= min(f32(min_p), 1.0)).sum())) if min_p > 0 else n)
        order, w = order[:n], w[:n]
    back = np.argsort(order)
    at, mass = np.asarray(order)[back], np.cumsum(w[back])
    tok = at[np.minimum(np.searchsorted(mass, u * mass[-1], side="right"), at.size - 1)]
    lse = x.max() + math.log(math.fsum(np.exp(x - x.max())))
    return tok, x[tok] - lse


def w4_values(codes, scales, N, K):
    """codes [tiles, chunks, 4, 16, 4, 4], scales [tiles, groups, 16] -> W float64 [N, K]"""
    tiles, chunks = codes.shape[:2]
    group = chunks * 128 // scales.shape[1]
    w = np.zeros((tiles * 16, chunks * 128))
    for t in range(tiles):
        for c in range(chunks):
            for g in range(4):
                for row in range(16):
                    for s in range(4):
                        for i in range(8):
                            k = 128 * c + 32 * s + 8 * g + i
                            code = (int(codes[t, c, g, row, s, i // 2]) >> (4 * (i % 2))) & 15
                            w[16 * t + row, k] = E2M1[code] * float(scales[t, k // group, row])
    return w[:N, :K]
