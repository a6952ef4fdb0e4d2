"""8-bit cached rows and attention over them, from their definitions in 64
bits (numpy and torch on the CPU; none of the package's code)."""

from __future__ import annotations

import math

import numpy as np
import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}


def e4m3(y: np.ndarray) -> np.ndarray:
    """Nearest e4m3 values (ties to even) of y, |y| <= 448."""
    _, e = np.frexp(y)
    step = np.exp2(np.maximum(e - 1, -6) - 3.0)
    return np.clip(np.rint(y / step) * step, -448.0, 448.0)


def quantise(x: torch.Tensor, dtype: torch.dtype):
    """(codes as float64 values, float32 scales) of rows x [..., D].  The scale
    and the quotient are float32 values by definition."""
    x = x.detach().cpu().to(torch.float64).numpy()
    top = TOP[dtype]
    with np.errstate(all="ignore"):
        scale = (np.abs(x).max(-1) / top).astype(np.float32)
        scale[~np.isfinite(x).all(-1)] = np.nan
        live = scale > 0
        div = np.where(live, scale, 1).astype(np.float64)[..., None]
        y = np.where(live[..., None], x / div, 0.0).astype(np.float32).astype(np.float64)
    y = np.clip(y, -top, top)
    codes = np.rint(y) if dtype == torch.int8 else e4m3(y)
    return torch.from_numpy(codes), torch.from_numpy(scale)


def values(x: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """What rows x read back as, float64."""
    codes, scale = quantise(x, dtype)
    return codes * scale.double()[..., None]


def ancestors(parents) -> np.ndarray:
    """[n, n] of who sees whom in one tree: itself and its ancestors."""
    n = len(parents)
    sees = np.zeros((n, n), bool)
    for j in range(n):
        at = j
        while at >= 0:
            sees[j, at] = True
            at = parents[at] if parents[at] < at else -1
    return sees


def mask_words(sees: np.ndarray, words: int) -> np.ndarray:
    """int64 [n, words] of a [n, t] table of who sees whom."""
    bits = np.zeros((sees.shape[0], words * 64), bool)
    bits[:, :sees.shape[1]] = sees
    return np.packbits(bits, axis=1, bitorder="little").view(np.int64)


def attention(query, keys, values, sees, scale):
    """One sequence: query [n, H, D], keys / values [c, Hkv, D] float64, sees
    bool [n, c].  Returns (out, spread, reach): out [n, H, D]; spread, the
    weighted sum of |v|, which a relative error of the weights multiplies;
    reach [n, H], the largest scale * sum |q| |k|, whose roundings are the
    error of a score; floor [n, H], the number of seen keys times the largest
    |v| among them, which a fixed step of the weights multiplies."""
    q = query.detach().cpu().double()
    n, H, D = q.shape
    hkv = keys.shape[1]
    g = H // hkv
    out, spread = torch.zeros_like(q), torch.zeros_like(q)
    reach = torch.zeros(n, H, dtype=torch.float64)
    floor = torch.zeros(n, H, dtype=torch.float64)
    seen = torch.as_tensor(sees)
    # (a key that nobody sees may hold anything)
    used = seen.any(0)
    k, v = keys[used], values[used]
    seen = seen[:, used]
    for h in range(H):
        x = q[:, h] @ k[:, h // g].T * scale
        x = x.masked_fill(~seen, -math.inf)
        live = seen.any(1)
        w = torch.zeros_like(x)
        if live.any():
            w[live] = torch.softmax(x[live], -1)
            for j in torch.nonzero(live).flatten().tolist():
                m = seen[j]
                out[j, h] = w[j, m] @ v[m, h // g]
                spread[j, h] = w[j, m] @ v[m, h // g].abs()
                floor[j, h] = m.sum() * v[m, h // g].abs().max()
                reach[j, h] = (abs(scale) * (q[j, h].abs() @ k[m, h // g].abs().T)).max()
    return out, spread, reach, floor


def tolerance(out, spread, reach, floor, dtype: torch.dtype):
    """How far a result of `dtype` may be off.

    Its own rounding: half a step of the result.  A score of D products summed
    in fp32 is off by at most (D + 4) 2^-24 of its reach (products, sums, and
    the scale's roundings), the weight by that relative amount, twice over
    through the sum of the weights; exp2 and the sums of weights and products
    add at most 2^-20 for the lengths tested.
    16-bit types: the numerator may take each weight in two parts (the sum takes
    it unrounded).  Two bf16 parts, the first cut off after 8 significant bits,
    leave less than 2^-7 of it, which 8 bits again hold to 2^-8 of that: 2^-15.
    Two fp16 parts, rounded, are off by 2^-11 of 2^-11.
    The smallest step of fp16 is 2^-24 whatever the value: with a row's largest
    numerator weight held at 2^10 or more a weight is off by up to half of it,
    2^-35 of the largest, so the sum by 2^-35 of the largest times the sum of
    |v|.  (Over codes the numerator's weight is w_t s_t and the codes are at
    most `top`: 2^-35 max(w_t s_t) n top <= 2^-35 n max|v|, the same.)"""
    half = torch.finfo(dtype).eps / 2
    fixed = 0.0
    rel = 2 * (out.shape[-1] + 4) * 2.0 ** -24 * reach[..., None] + 2.0 ** -20
    if dtype != torch.float32:
        rel = rel + 2.0 ** -15
        fixed = 2.0 ** -35 * floor[..., None]
    tiny = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126}
    return half * out.abs() + (1 + half) * (rel * spread + fixed) + tiny[dtype]
