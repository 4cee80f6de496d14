"""The operators of the 4-bit path, as they are measured: microscaled 4-bit floating point (MXFP4: blocks of 32 e2m1 codes
under one power of two) for rows, linears and the paged cache of a batch of sequences.

A case is a dict of plain values; ``kind`` names the operator:

  quant   mxfp4.quant_mxfp4 and .dequant_mxfp4: rows into codes and scales, and read back
  linear  mxfp4.WaveMxfp4Linear: activations quantized, product with the 4-bit weight, bias, GELU(tanh) if ``gelu``
  cache   kv.PagedBatch.append and .gather over kv.Mxfp4PagePool: new K/V rows of every sequence into its pages and back
  attn    backend.attn_paged_batch over kv.Mxfp4PagePool: ragged new rows over the paged caches (``block`` 0: every key of
          the sequence; 1: causal; n: causal by blocks of n positions)

``m`` rows, ``k`` and ``n`` a linear's input and output width.  ``seqs`` sequences; ``new`` the most new rows of one; ``past``
the most cached positions before them; ``ragged``: the sequences' new rows differ.  The lengths follow from ``mix``; with
six sequences or more one of them has no new rows.  Sizes are those of the two presets (dim 1536, 12 heads, FFN 8960; dim
5120, 40 heads, FFN 13824; 1560 tokens per frame, chunks of 3 frames, up to 8 chunks of context) and generic ones.
Activations are N(0, 1) with 1 % of the channels 20 times larger, weights N(0, 0.02), K and V N(0, 1) with 8 heavy-tailed
(Student-t, 3 degrees) dims per head.
"""

import math
import random

import torch

own = False

DEV = "cuda:0"
D = 128
BLOCK = 32
FRAME = 1560
CHUNK = 3 * FRAME
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SCALE = 1 / math.sqrt(D)


def listed():
    return [
        # the activations of one token of each of 16 streams: all latency
        dict(name="quant_tokens_16", kind="quant", m=16, k=5120),
        # the input of fc_out of a 1.3B block, one chunk
        dict(name="quant_chunk_1p3b", kind="quant", m=CHUNK, k=8960),
        # one token through a 1.3B block's fused QKV projection: the smallest linear
        dict(name="linear_token", kind="linear", m=1, k=1536, n=4608, gelu=False, bias=True),
        # one token of each of 16 streams through fc_in of a 14B block with its GELU: the weight is read once
        dict(name="linear_tokens_16", kind="linear", m=16, k=5120, n=13824, gelu=True, bias=True),
        # a few frames' odd number of rows, a width that ends inside a tile, no bias
        dict(name="linear_odd", kind="linear", m=301, k=1568, n=2212, gelu=False, bias=False),
        # fc_out of a 14B block, one chunk
        dict(name="linear_chunk_14b", kind="linear", m=CHUNK, k=13824, n=5120, gelu=False, bias=True),
        # one new token of each of 64 streams: the smallest write
        dict(name="cache_tokens_64", kind="cache", seqs=64, new=1, past=4000, ragged=False, hkv=8, page=64, mix=1),
        # one layer's K/V of the chunks of four 1.3B streams, published and gathered back
        dict(name="cache_chunks_1p3b", kind="cache", seqs=4, new=CHUNK, past=16 * FRAME, ragged=False, hkv=12, page=FRAME, mix=2),
        # a single token of one stream over a short context: the smallest attention
        dict(name="attn_token", kind="attn", seqs=1, new=1, past=1559, ragged=False, hq=12, hkv=12, page=FRAME, block=1, mix=4),
        # single tokens of 64 streams, five query heads to a key head, pages of 64: the cache is read once
        dict(name="attn_tokens_64", kind="attn", seqs=64, new=1, past=8191, ragged=False, hq=40, hkv=8, page=64, block=1, mix=5),
        # causal prompts of odd lengths behind contexts of other lengths, grouped heads, small pages
        dict(name="attn_prompts", kind="attn", seqs=6, new=4001, past=6000, ragged=True, hq=16, hkv=4, page=16, block=1, mix=7),
        # three 1.3B streams' chunks at once over the contexts each has reached, up to the steady state's 8 chunks
        dict(name="attn_chunks_1p3b", kind="attn", seqs=3, new=CHUNK, past=7 * CHUNK, ragged=False, hq=12, hkv=12, page=FRAME,
             block=0, mix=8),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["quant", "linear", "linear", "linear", "cache", "attn", "attn", "attn"])
    if kind in ("quant", "linear"):
        c = dict(kind=kind, m=_log(rng, 1, CHUNK), k=BLOCK * _log(rng, 1, 432))
        if kind == "linear":
            c.update(n=4 * _log(rng, 8, 3456), gelu=rng.random() < 0.4, bias=rng.random() < 0.7)
            c["n"] = min(c["n"], max(32, CHUNK * 13824 * 5120 // (c["m"] * c["k"]) // 4 * 4))
        return c
    c = dict(kind=kind, seqs=_log(rng, 1, 64), mix=rng.randint(100, 1 << 30), ragged=rng.random() < 0.6,
             page=rng.choice([16, 48, 64, 390, FRAME]))
    if kind == "cache":
        c["hkv"] = rng.choice([1, 2, 5, 8, 12, 40])
        c["new"] = _log(rng, 1, max(1, min(CHUNK, 4 * CHUNK * 12 // (c["hkv"] * c["seqs"]))))
        c["past"] = _log(rng, 1, max(1, 8 * CHUNK // c["seqs"]))
        return c
    c["hkv"], group = rng.choice([(12, 1), (40, 1), (8, 5), (4, 6), (4, 4), (2, 8), (1, 16)])
    c["hq"] = c["hkv"] * group
    c["new"] = _log(rng, 1, 8) if rng.random() < 0.5 else _log(rng, 9, CHUNK)
    c["past"] = _log(rng, 1, 8 * CHUNK)
    c["block"] = rng.choice([0, 1, 1, FRAME, 100])
    # the largest listed attention bounds the work, and the padded scores and caches of the plain form stay in memory
    c["seqs"] = max(1, min(c["seqs"], 64 * 8192 * 8 // (c["hkv"] * (c["past"] + c["new"])),
                           CHUNK * 8 * CHUNK * 12 // (c["hq"] * c["new"] * (c["past"] + c["new"]))))
    c["past"] = max(1, min(c["past"], CHUNK * 8 * CHUNK * 12 // (c["hq"] * c["new"] * c["seqs"])))
    return c


# ------------------------------------------------------------------ inputs
def _lens(case):
    """(new rows, keys) of every sequence."""
    r = random.Random(case["mix"])
    new, kv = [], []
    for b in range(case["seqs"]):
        n = r.randint(1, case["new"]) if case["ragged"] and b else case["new"]
        if case["seqs"] >= 6 and b == 2:
            n = 0   # a stream with nothing to do this time
        new.append(n)
        kv.append(n + (r.randint(case["past"] // 8, case["past"]) if b else case["past"]))
    return new, kv


class _Draw:
    """Tensors of one seed, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(1000003 * (int(seed) % (1 << 40)) + 31)

    def normal(self, shape, std=1.0):
        return (torch.randn(shape, generator=self.g, device=DEV) * std).to(BF16)

    def activations(self, m, k):
        x = torch.randn((m, k), generator=self.g, device=DEV)
        big = torch.rand((k,), generator=self.g, device=DEV).argsort()[:max(1, k // 100)]
        x[:, big] *= 20
        return x.to(BF16)

    def kv(self, rows, heads):
        x = torch.randn((rows, heads, D), generator=self.g, device=DEV)
        dims = torch.rand((heads, D), generator=self.g, device=DEV).argsort(dim=1)[:, :8]
        chi2 = torch.randn((rows, heads, 8, 3), generator=self.g, device=DEV).square().sum(-1)
        at = dims.expand(rows, heads, 8)
        x.scatter_(2, at, x.gather(2, at) / (chi2 / 3).sqrt())
        return x.to(BF16)


def _steps(x):
    """x [..., 32 n] as multiples of their blocks' powers of two: (values of the codes [..., n, 32], exponents [..., n])."""
    x = x.float().unflatten(-1, (-1, BLOCK))
    m, e = torch.frexp(x.abs().amax(-1))                 # m in [1/2, 1)
    e = (e - 3 + (m >= 0.875).int()).clamp(-125, 125)    # the smallest power of two of which the largest value is below 7
    y = torch.ldexp(x, -e[..., None])
    step = torch.where(y.abs() < 2, 0.5, torch.where(y.abs() < 4, 1.0, 2.0))
    return (torch.round(y / step) * step).clamp(-6, 6), e


def _rounded(x):
    """fp32 values of x's 4-bit form."""
    v, e = _steps(x)
    return torch.ldexp(v, e[..., None]).flatten(-2)


def _pack(x):
    """(code bytes [..., k / 2], the even value in the low half; E8M0 bytes [..., k / 32]) of bf16 rows."""
    v, e = _steps(x)
    a = v.abs()
    code = torch.where(a < 2, 2 * a, torch.where(a < 4, a + 2, a / 2 + 4)).to(torch.uint8) | (torch.signbit(v).to(torch.uint8) << 3)
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), (e + 127).to(torch.uint8)


def _values(codes, scales):
    """fp32 values of code bytes [..., k / 2] under E8M0 bytes [..., k / 32]."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    m = (c & 7).float()
    a = torch.where(m < 4, m / 2, torch.where(m < 6, m - 2, 2 * m - 8))
    v = torch.where(c >= 8, -a, a).unflatten(-1, (-1, BLOCK))
    return torch.ldexp(v, scales.int()[..., None] - 127).flatten(-2)


def _inputs(case, seed):
    """The tensors of a case; of the cached kinds also the lengths and the page lists."""
    r = _Draw(seed)
    if case["kind"] == "quant":
        return dict(x=r.activations(case["m"], case["k"]))
    if case["kind"] == "linear":
        x = dict(x=r.activations(case["m"], case["k"]), w=r.normal((case["n"], case["k"]), 0.02))
        return dict(x, b=r.normal((case["n"],), 0.1) if case["bias"] else None)
    new, kv = _lens(case)
    page, hkv = case["page"], case["hkv"]
    counts = [-(-n // page) for n in kv]
    pool = sum(counts) + 3
    order = torch.randperm(pool, generator=r.g, device=DEV).tolist()
    pages, at = [], 0
    for n in counts:
        pages.append(order[at:at + n])
        at += n
    x = dict(new=new, kv=kv, pages=pages)
    if case["kind"] == "cache":
        x.update(k=r.kv(sum(new), hkv), v=r.kv(sum(new), hkv))
        for t in ("k", "v"):
            x[t + "_codes"] = torch.zeros((pool, page, hkv, D // 2), dtype=torch.uint8, device=DEV)
            x[t + "_scales"] = torch.zeros((pool, hkv, page, D // BLOCK), dtype=torch.uint8, device=DEV)
        return x
    x["q"] = r.normal((sum(new), case["hq"], D))
    for t in ("k", "v"):
        codes, scales = _pack(r.kv(pool * page, hkv))
        x[t + "_codes"] = codes.view(pool, page, hkv, D // 2)
        x[t + "_scales"] = scales.view(pool, page, hkv, D // BLOCK).transpose(1, 2).contiguous()
    return x


def prepare(case, seed):
    s = dict(case, **_inputs(case, seed))
    if own:   # what a user of the framework keeps: the quantized linear, or the pool and the batch's tables and lengths
        from waveforcing_amd import backend, mxfp4
        from waveforcing_amd import kv as wkv

        s["backend"], s["mxfp4"] = backend, mxfp4
        if s["kind"] == "linear":
            s["linear"] = mxfp4.WaveMxfp4Linear(s.pop("w"), s.pop("b"), gelu=s["gelu"])
        elif s["kind"] != "quant":
            pool = wkv.Mxfp4PagePool(s["k_codes"].shape[0], s["hkv"], D, s["page"], DEV)
            for t in ("k_codes", "v_codes", "k_scales", "v_scales"):
                getattr(pool, t).copy_(s.pop(t))
            s["batch"] = wkv.PagedBatch(pool, s["pages"], s["kv"], s["new"])
        return s
    if s["kind"] == "linear":
        s["w"] = _rounded(s["w"])
        if s["bias"]:
            s["b"] = s["b"].float()
    elif s["kind"] != "quant":
        as_dev = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)
        new, kv, pages = s["new"], s["kv"], s["pages"]
        s["seq"] = as_dev([b for b, n in enumerate(new) for _ in range(n)])
        s["row"] = as_dev([i for n in new for i in range(n)])
        s["new_lens"], s["kv_lens"] = as_dev(new), as_dev(kv)
        s["most"] = (max(new), max(kv))
        s["starts"] = as_dev([sum(new[:b]) for b in range(len(new))])
        wide = max(1, max(len(p) for p in pages))
        s["tables"] = as_dev([p + [0] * (wide - len(p)) for p in pages])
    return s


# -------------------------------------------------------------------- run
def _linear_plain(s):
    y = torch.matmul(_rounded(s["x"]), s["w"].t())
    if s["bias"]:
        y = y + s["b"]
    if s["gelu"]:
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y.to(BF16)


def _cache_plain(s):
    pos = s["kv_lens"][s["seq"]] - s["new_lens"][s["seq"]] + s["row"]
    page, at = s["tables"][s["seq"], pos // s["page"]], pos % s["page"]
    out = {}
    for t in ("k", "v"):
        codes, scales = s[t + "_codes"], s[t + "_scales"]
        codes[page, at], scales[page, :, at] = _pack(s[t])
        out[t] = _values(codes[page, at], scales[page, :, at]).to(BF16)
    return out


def _attn_plain(s):
    key = torch.arange(s["most"][1], device=DEV)
    page, at = s["tables"][:, key // s["page"]], key % s["page"]
    here = key < s["kv_lens"][:, None]
    k, v = (_values(s[t + "_codes"][page, at], s[t + "_scales"].transpose(1, 2)[page, at]).masked_fill_(~here[..., None, None], 0)
            for t in ("k", "v"))
    seen = here[:, None, :]
    if s["block"]:
        pos = (s["kv_lens"] - s["new_lens"])[:, None] + torch.arange(s["most"][0], device=DEV)
        seen = seen & (key < (pos // s["block"] + 1)[..., None] * s["block"])
    B, lq, hkv = len(s["new_lens"]), s["most"][0], s["hkv"]
    group = s["hq"] // hkv
    at = (s["starts"][:, None] + torch.arange(lq, device=DEV)).clamp(max=s["q"].shape[0] - 1)
    q = s["q"][at].float().view(B, lq, hkv, group, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, group * lq, D)
    p = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()).mul_(SCALE).view(B, hkv, group, lq, -1)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, group * lq, -1), v.transpose(1, 2).contiguous()).view(B, hkv, group, lq, D)
    o = o / torch.where(total > 0, total, torch.ones_like(total))
    return o.permute(0, 3, 1, 2, 4)[s["seq"], s["row"]].reshape(-1, s["hq"], D).to(BF16)


def run(s):
    if own:
        if s["kind"] == "quant":
            return s["mxfp4"].dequant_mxfp4(*s["mxfp4"].quant_mxfp4(s["x"]))
        if s["kind"] == "linear":
            return s["linear"](s["x"])[0]
        if s["kind"] == "cache":
            s["batch"].append(s["k"], s["v"])
            k, v = s["batch"].gather()
            return dict(k=k, v=v)
        return s["backend"].attn_paged_batch(s["q"], s["batch"], block=s["block"], softmax_scale=SCALE)
    if s["kind"] == "quant":
        return _values(*_pack(s["x"])).to(BF16)
    return {"linear": _linear_plain, "cache": _cache_plain, "attn": _attn_plain}[s["kind"]](s)


# ------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "quant":
        return dict(bytes=case["m"] * case["k"] * 4 + 2 * case["m"] * case["k"] * 17 // 32, flops=0)
    if case["kind"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        return dict(bytes=2 * m * k + n * k * 17 // 32 + 2 * m * n + (2 * n if case["bias"] else 0), flops=2 * m * k * n)
    new, kv = _lens(case)
    hkv, row = case["hkv"], D // 2 + D // BLOCK
    if case["kind"] == "cache":
        return dict(bytes=4 * sum(new) * hkv * (2 * D + row), flops=0)
    seen = 0
    for n, t in zip(new, kv):
        b = case["block"]
        seen += n * t if not b else sum(min(t, (p // b + 1) * b) for p in range(t - n, t))
    read = sum(t for n, t in zip(new, kv) if n)
    return dict(bytes=4 * D * sum(new) * case["hq"] + 2 * row * hkv * read, flops=4 * D * seen * case["hq"])


# ------------------------------------------------ the same in 64 bits
_GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest(x):
    """The 4-bit form of x [..., 32 n]: the nearest number of the grid times the block's power of two, an even code on a tie."""
    x = x.to(F64).unflatten(-1, (-1, BLOCK))
    s = torch.exp2((torch.floor(torch.log2(x.abs().amax(-1, keepdim=True) / 7)) + 1).clamp(-125, 125))
    y = (x / s).abs()
    out = torch.zeros_like(y)
    for i in range(7):
        mid = (_GRID[i] + _GRID[i + 1]) / 2
        out += ((y >= mid) if i % 2 else (y > mid)).to(F64) * (_GRID[i + 1] - _GRID[i])
    return (torch.where(x < 0, -out, out) * s).flatten(-2)


def _decode(codes, scales):
    """The numbers that the bytes stand for, from the formats' definitions."""
    grid = torch.tensor(_GRID + [-g for g in _GRID], dtype=F64, device=DEV)
    pair = torch.stack((grid[(codes & 15).long()], grid[(codes >> 4).long()]), -1).flatten(-2)
    return (pair.unflatten(-1, (-1, BLOCK)) * torch.exp2(scales.to(F64) - 127)[..., None]).flatten(-2)


def _softmax_product(q, k, v, limit):
    """q [n, Hq, D], k and v [t, Hkv, D] in 64 bits; row i sees the keys before limit[i]."""
    n, hq, _ = q.shape
    out = torch.zeros_like(q)
    group = hq // k.shape[1]
    key = torch.arange(k.shape[0], device=DEV)
    for h in range(hq):
        kh, vh = k[:, h // group].t().contiguous(), v[:, h // group].contiguous()
        for i in range(0, n, 4096):
            lim = limit[i:i + 4096, None]
            s = (q[i:i + 4096, h].contiguous() @ kh) * SCALE
            s = torch.where(key < lim, s, torch.full_like(s, -math.inf))
            w = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300))
            out[i:i + 4096, h] = (w @ vh) / w.sum(-1, keepdim=True).clamp(min=1e-300)
    return out


def exact(case, seed):
    x = _inputs(case, seed)
    if case["kind"] == "quant":
        return _nearest(x["x"])
    if case["kind"] == "linear":
        y = _nearest(x["x"]) @ _nearest(x["w"]).t()
        if case["bias"]:
            y = y + x["b"].to(F64)
        if case["gelu"]:
            y = y / (1 + torch.exp(-2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
        return y
    if case["kind"] == "cache":
        return dict(k=_nearest(x["k"]), v=_nearest(x["v"]))
    out, at = torch.zeros(x["q"].shape, dtype=F64, device=DEV), 0
    for n, t, pages in zip(x["new"], x["kv"], x["pages"]):
        pos = torch.arange(t - n, t, device=DEV)
        limit = torch.full_like(pos, t)
        if case["block"]:
            limit = torch.minimum(limit, (torch.div(pos, case["block"], rounding_mode="floor") + 1) * case["block"])
        ids = torch.tensor(pages, dtype=torch.int64, device=DEV)
        k, v = (_decode(x[y + "_codes"][ids], x[y + "_scales"][ids].transpose(1, 2)).reshape(-1, case["hkv"], D)[:t] for y in ("k", "v"))
        if n:
            out[at:at + n] = _softmax_product(x["q"][at:at + n].to(F64), k, v, limit)
        at += n
    return out
