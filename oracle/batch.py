"""Batched sequences in 64 bits: the paged cache of ragged rows in both formats, and attention over it.

Plain restatements of the operators' definitions (no reference counterpart: the reference serves one sequence per call).
"""

from __future__ import annotations

import torch


def row_positions(kv_lens, new_lens):
    """(sequence, position) of every new row, in order."""
    return [(b, t - n + i) for b, (t, n) in enumerate(zip(kv_lens, new_lens)) for i in range(n)]


def quantize(x: torch.Tensor, fmt: str):
    """Codes (uint8) and fp32 scales of bf16 rows [..., 128]."""
    f = x.float()
    amax = f.abs().amax(-1)
    if fmt == "int8":
        s = (amax / torch.full_like(amax, 127)).clamp(min=1e-8)   # a tensor: division by a number multiplies on a GPU
        c = torch.round(f / s[..., None]).clamp(-127, 127).nan_to_num(0).to(torch.int8).view(torch.uint8)
    else:
        s = (amax / torch.full_like(amax, 448)).bfloat16().clamp(min=1e-8).float()
        c = (f / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    bad = ~torch.isfinite(f).all(-1)
    return c.masked_fill(bad[..., None], 0), s.masked_fill(bad, float("nan"))


def values(codes: torch.Tensor, scales: torch.Tensor, fmt: str) -> torch.Tensor:
    """code * scale in 64 bits; scales broadcast over the last dim of codes."""
    c = codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)
    return c.float().double() * scales.double()[..., None]


def cached(codes, scales, fmt, pages, n, page_tokens):
    """The n cached rows [n, heads, 128] of one sequence, in 64 bits."""
    if n == 0:
        return torch.zeros((0, codes.shape[2], 128), dtype=torch.float64, device=codes.device)
    ids = torch.tensor(pages[:-(-n // page_tokens)], dtype=torch.int64, device=codes.device)
    v = values(codes[ids], scales[ids].transpose(1, 2), fmt)
    return v.reshape(-1, codes.shape[2], 128)[:n]


def limit(position: int, kv_len: int, block: int) -> int:
    return kv_len if block == 0 else min(kv_len, (position // block + 1) * block)


def attend(q, k, v, limits, scale):
    """Rows q [n, heads, 128] over keys k, v [t, key heads, 128] (64 bits); row i sees the keys before limits[i].

    Returns (out, bound): the output and how far a bf16 output of fp32 arithmetic with bf16 weights may be from it.
    With A = sum_j w_j |v_j| / sum_j w_j, every weight is off by at most 2^-8 of itself from its rounding and by the
    error of its exponent.  A score's error e: the queries may be held as sums of two 4-bit significands under the
    row's power-of-two scale (off by at most 2^-10 of the scale, which is at most 2 max|q| / 448: 2^-17.8 max|q|) and
    the fp32 sums of 128 products of the parts run in any order (256 roundings of 2^-24 of twice the sum of the
    magnitudes: 2^-15); 2^-20 more for the exponential, and 2^-14 for the fp32 running sums over the keys (up to
    2^10 tiles' roundings).  The quotient of two sums doubles e.  The result is rounded to bf16 once: 2^-8.

    Two absolute terms come with fp16 (many rows), whose numbers are 2^-24 apart below 2^-14, half a step 2^-25.  A
    weight times its key's scale of V is held as 64 times its ratio to the largest such product M that the row has
    seen, or more, so it is off by at most 2^-25 / 64 = 2^-31 of M, and multiplies an exact code.  For keys whose scale
    is not below that of M's key these errors are together at most 2^-31 w_max sum_j |v_j| over the seen keys.  Of a key
    of smaller scale the error is at most 2^-31 M |code| <= 2^-31 w_max max|V|, of either sign; 2^-33 max|V| is allowed
    for the mean of them, which a quarter of such a key reaches at the worst and hundreds of ordinary ones do not.
    """
    q, k, v = q.double(), k.double(), v.double()
    n, heads, _ = q.shape
    group = heads // k.shape[1]
    out = torch.zeros_like(q)
    bound = torch.zeros_like(q)
    key = torch.arange(k.shape[0], device=q.device)
    seen = key[None, :] < torch.as_tensor(limits, device=q.device)[:, None]
    some = seen.any(1)
    for h in range(heads):
        g = h // group
        kg, vg = k[:, g], v[:, g]
        kz = torch.where(torch.isnan(kg), torch.zeros_like(kg), kg)
        s = q[:, h] @ kg.t().contiguous() * scale
        e = (2.0 ** -17.8 * q[:, h].abs().amax(-1, keepdim=True) * kz.abs().sum(-1)
             + 2.0 ** -15 * (q[:, h].abs() @ kz.abs().t().contiguous())) * scale
        e = e.masked_fill(~seen, 0).amax(-1, keepdim=True) if len(key) else torch.zeros_like(q[:, h, :1])
        s = s.masked_fill(~seen, float("-inf"))
        w = torch.zeros_like(s)
        if len(key):
            w[some] = torch.softmax(s[some], -1)
        # a weight of an unseen key is no term of the sum, whatever the key holds
        vz = torch.where(torch.isfinite(vg), vg, torch.zeros_like(vg))
        out[:, h] = w @ vz
        bad = (seen.double() @ (~torch.isfinite(vg)).double()) > 0
        out[:, h] = out[:, h].masked_fill(bad, float("nan"))
        A = w @ vz.abs()
        small = torch.zeros_like(A)
        if len(key):
            small = 2.0 ** -31 * w.amax(-1, keepdim=True) * (seen.double() @ vz.abs()) + 2.0 ** -33 * vz.abs().max()
        bound[:, h] = small + A * (2.0 ** -8 + 2 * e * (1 + 2.0 ** -8) + 2.0 ** -13) + out[:, h].abs() * 2.0 ** -8 * (1 + 2.0 ** -6) + 1e-30
    return out, bound
