"""Microscaled 4-bit floating point in 64 bits: the codec of rows, the product, and the paged cache's rows.

Plain restatements of the definitions in include/wf_api.h (no reference counterpart: the reference has no 4-bit form).
"""

from __future__ import annotations

import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantize(x: torch.Tensor):
    """(codes uint8 [..., k], one a value; scale bytes uint8 [..., k / 32]) of bf16 x [..., k]."""
    f = x.double().unflatten(-1, (-1, 32))
    bad = ~torch.isfinite(f).all(-1)
    f = torch.where(torch.isfinite(f), f, torch.zeros_like(f))
    # the smallest power of two of which the largest magnitude is below 7
    e = (torch.floor(torch.log2(f.abs().amax(-1) / 7)) + 1).clamp(-125, 125)
    y = f / torch.exp2(e)[..., None]
    code = torch.zeros_like(y, dtype=torch.int64)
    for i in range(7):
        mid = (GRID[i] + GRID[i + 1]) / 2
        code += ((y.abs() >= mid) if i % 2 else (y.abs() > mid)).long()   # ties to the even code
    code = (code + 8 * torch.signbit(f).long()).masked_fill(bad[..., None], 0)
    return code.to(torch.uint8).flatten(-2), (e + 127).long().masked_fill(bad, 255).to(torch.uint8)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """64-bit values of codes [..., k] (one a value) under scale bytes [..., k / 32]."""
    grid = torch.tensor(GRID + tuple(-g for g in GRID), dtype=torch.float64, device=codes.device)
    s = torch.exp2(scales.double() - 127).masked_fill(scales == 255, math.nan)
    return (grid[codes.long()].unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def pack(codes: torch.Tensor) -> torch.Tensor:
    """Two codes to a byte, the even one low."""
    return codes[..., 0::2] | codes[..., 1::2] << 4


def unpack(b: torch.Tensor) -> torch.Tensor:
    return torch.stack((b & 15, b >> 4), -1).flatten(-2)


def panels(codes: torch.Tensor, scales: torch.Tensor):
    """Code bytes [rows, k / 2] and scale bytes [rows, k / 32] as panels of 16 rows by 128 values (include/wf_api.h)."""
    rows, n = scales.shape
    P, G = -(-rows // 16), -(-n // 4)
    c = torch.zeros((P, G, 4, 16, 16), dtype=torch.uint8, device=codes.device)
    s = torch.zeros((P, G, 16, 4), dtype=torch.uint8, device=codes.device)
    for p in range(P):
        m = min(16, rows - 16 * p)
        at = slice(16 * p, 16 * p + m)
        for i in range(n):
            c[p, i // 4, i % 4, :m] = codes[at, 16 * i:16 * i + 16]
            s[p, i // 4, :m, i % 4] = scales[at, i]
    return c, s


def gelu(y: torch.Tensor) -> torch.Tensor:
    return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))


def product(a: torch.Tensor, w: torch.Tensor, bias=None, act: bool = False):
    """(result, bound) of values a [m, k], w [n, k] in 64 bits: how far a bf16 result of fp32 sums may be from it.

    Each product is exact in fp32 (two significant bits by two).  A matrix instruction adds 64 or 128 of them to the sum so
    far with an error of at most 2^-23 of the magnitudes' sum S; the partial sums of at most 8 ranges of K are added in
    fp32: with k / 64 + 16 such steps the sum is off by at most (k / 64 + 16) 2^-23 S, and the bias adds 2^-24 of the result.
    GELU's slope is at most 1.13, its fp32 evaluation is off by at most 2^-18 of its argument's magnitude (an exponential,
    a reciprocal and four products of 2^-22 each, where the argument of the exponential, at most 2^5 before the result no
    longer changes, multiplies its relative error).  The result is rounded to bf16 once: 2^-8, and 2^-133 below 2^-126."""
    y = a @ w.t()
    off = (a.shape[1] / 64 + 16) * 2.0 ** -23 * (a.abs() @ w.abs().t())
    if bias is not None:
        y = y + bias.double()
        off = off + 2.0 ** -23 * (y.abs() + bias.double().abs())
    if act:
        off = 1.13 * off + 2.0 ** -18 * y.abs()
        y = gelu(y)
    return y, off * (1 + 2.0 ** -7) + 2.0 ** -8 * y.abs() + 2.0 ** -133


def cached(codes, scales, pages, n, page_tokens):
    """The n cached rows [n, heads, 128] of one sequence, in 64 bits; codes [pages, tokens, heads, 64], scales [pages, heads,
    tokens, 4]."""
    if n == 0:
        return torch.zeros((0, codes.shape[2], 128), dtype=torch.float64, device=codes.device)
    ids = torch.tensor(pages[:-(-n // page_tokens)], dtype=torch.int64, device=codes.device)
    return values(unpack(codes[ids]), scales[ids].transpose(1, 2)).reshape(-1, codes.shape[2], 128)[:n]
