"""The operators of batched streams, as they are measured: a paged quantized cache that several sequences write and read
at once, the attention over it, and the attention to encoder states of ragged lengths.

A case is a dict of plain values; ``kind`` names the operator:

  cache  kv.PagedBatch.append and .gather: new K/V rows of every sequence quantized into its pages, and read back
  attn   backend.attn_paged_batch: ragged new rows over the paged caches (``block`` 0: every key of the sequence;
         1: causal; n: causal by blocks of n positions)
  cross  backend.attn_cross_batch: ragged rows over dense bf16 rows of another length

``seqs`` sequences; ``new`` the most new rows of one; ``past`` the most cached positions before them; ``ragged``: the
sequences' new rows differ.  The lengths follow from ``mix``; with six sequences or more one of them has no new rows.
Sizes are those of the two presets (12 and 40 heads of 128, 1560 tokens per frame, chunks of 3 frames, a 21-frame
window, text of up to 512 tokens) and generic ones with grouped key heads and small pages.
"""

import math
import random

import torch

own = False

DEV = "cuda:0"
D = 128
FRAME = 1560
CHUNK = 3 * FRAME
BF16, F32, F64 = torch.bfloat16, torch.float32, torch.float64
SCALE = 1 / math.sqrt(D)


def listed():
    return [
        # one new token of each of 64 streams into int8 pages: the smallest write, all latency
        dict(name="cache_tokens_64", kind="cache", fmt="int8", seqs=64, new=1, past=4000, ragged=False, hkv=8, page=64, mix=1),
        # one layer's K/V of the chunks of four 1.3B streams, published and gathered back
        dict(name="cache_chunks_1p3b", kind="cache", fmt="e4m3", seqs=4, new=CHUNK, past=16 * FRAME, ragged=False, hkv=12,
             page=FRAME, mix=2),
        # prompts of odd lengths that begin and end inside odd pages
        dict(name="cache_odd", kind="cache", fmt="int8", seqs=9, new=777, past=3000, ragged=True, hkv=5, page=48, mix=3),
        # a single token of one stream over a short context: the smallest attention
        dict(name="attn_token", kind="attn", fmt="e4m3", seqs=1, new=1, past=1559, ragged=False, hq=12, hkv=12, page=FRAME,
             block=1, mix=4),
        # single tokens of 64 streams, five query heads to a key head, int8 pages of 64: the cache is read once
        dict(name="attn_tokens_64", kind="attn", fmt="int8", seqs=64, new=1, past=8191, ragged=False, hq=40, hkv=8, page=64,
             block=1, mix=5),
        # a few tokens each of 16 streams over pages of 16
        dict(name="attn_few", kind="attn", fmt="e4m3", seqs=16, new=7, past=5001, ragged=True, hq=24, hkv=4, page=16,
             block=1, mix=6),
        # causal chunks of prompts behind contexts of other lengths, grouped heads
        dict(name="attn_prompts", kind="attn", fmt="e4m3", seqs=6, new=4001, past=6000, ragged=True, hq=16, hkv=4, page=64,
             block=1, mix=7),
        # three 1.3B streams' chunks at once over the contexts each has reached, up to the steady state's 8 chunks
        dict(name="attn_chunks_1p3b", kind="attn", fmt="e4m3", seqs=3, new=CHUNK, past=7 * CHUNK, ragged=False, hq=12, hkv=12,
             page=FRAME, block=0, mix=8),
        # two clips of up to 7 frames read into the cache, causal by frames, int8 pages
        dict(name="attn_frames_int8", kind="attn", fmt="int8", seqs=2, new=7 * FRAME, past=0, ragged=True, hq=12, hkv=12,
             page=FRAME, block=FRAME, mix=9),
        # text cross-attention of four 1.3B streams' chunks, each with its prompt's own length
        dict(name="cross_chunks_1p3b", kind="cross", seqs=4, new=CHUNK, past=512, ragged=False, hq=12, hkv=12, mix=10),
        # single rows over the prompts of 32 streams (14B heads)
        dict(name="cross_tokens_32", kind="cross", seqs=32, new=1, past=512, ragged=False, hq=40, hkv=40, mix=11),
        # odd row counts over long encoder outputs, grouped heads
        dict(name="cross_long", kind="cross", seqs=8, new=301, past=4001, ragged=True, hq=16, hkv=4, mix=12),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["cache", "cache", "attn", "attn", "attn", "cross"])
    c = dict(kind=kind, seqs=_log(rng, 1, 64), mix=rng.randint(100, 1 << 30), ragged=rng.random() < 0.6)
    if kind != "cross":
        c.update(fmt=rng.choice(["e4m3", "int8"]), page=rng.choice([16, 48, 64, 390, FRAME]))
    if kind == "cache":
        c["hkv"] = rng.choice([1, 2, 5, 8, 12, 40])
        c["new"] = _log(rng, 1, max(1, min(CHUNK, 4 * CHUNK * 12 // (c["hkv"] * c["seqs"]))))
        c["past"] = _log(rng, 1, max(1, 8 * CHUNK // c["seqs"]))
        return c
    c["hkv"], group = rng.choice([(12, 1), (40, 1), (8, 5), (4, 6), (4, 4), (2, 8), (1, 16)])
    c["hq"] = c["hkv"] * group
    tokens = rng.random() < 0.5
    c["new"] = _log(rng, 1, 8) if tokens else _log(rng, 9, CHUNK)
    c["past"] = _log(rng, 1, 512 if kind == "cross" and rng.random() < 0.5 else 8 * CHUNK if kind == "attn" else 5000)
    if kind == "attn":
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
        past = r.randint(case["past"] // 8, case["past"]) if b else case["past"]
        if case["kind"] == "cross":
            kv.append(0 if case["seqs"] >= 6 and b == 1 else past)   # a stream without a prompt
        else:
            kv.append(past + n)
        new.append(n)
    return new, kv


class _Draw:
    """Tensors of one seed, in the order they are asked for."""

    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(1000003 * (int(seed) % (1 << 40)) + 29)

    def normal(self, shape):
        return torch.randn(shape, generator=self.g, device=DEV).to(BF16)

    def kv(self, rows, heads):
        """N(0, 1) rows with 8 heavy-tailed (Student-t, 3 degrees) dims per head, as the model's K and V have."""
        x = torch.randn((rows, heads, D), generator=self.g, device=DEV)
        dims = torch.rand((heads, D), generator=self.g, device=DEV).argsort(dim=1)[:, :8]
        chi2 = torch.randn((rows, heads, 8, 3), generator=self.g, device=DEV).square().sum(-1)
        at = dims.expand(rows, heads, 8)
        x.scatter_(2, at, x.gather(2, at) / (chi2 / 3).sqrt())
        return x.to(BF16)


def _quantize(x, fmt):
    """(codes as bytes, fp32 scales) of bf16 rows [..., D]."""
    x = x.float()
    amax = x.abs().amax(-1)
    if fmt == "int8":
        s = (amax / 127).clamp(min=1e-8)
        return torch.round(x / s[..., None]).clamp(-127, 127).to(torch.int8).view(torch.uint8), s
    s = (amax / 448).to(BF16).float().clamp(min=float(torch.tensor(1e-8, dtype=BF16)))
    return (x / s[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8), s


def _values(codes, fmt):
    return codes.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()


def _inputs(case, seed):
    """The tensors of a case, and its page lists: every page of the pool holds some sequence's rows or none's."""
    new, kv = _lens(case)
    r, x = _Draw(seed), {}
    if case["kind"] == "cross":
        x.update(q=r.normal((sum(new), case["hq"], D)), k=r.kv(sum(kv), case["hkv"]), v=r.kv(sum(kv), case["hkv"]))
        return new, kv, None, x
    page, hkv = case["page"], case["hkv"]
    counts = [-(-n // page) for n in kv]
    pool = sum(counts) + 3
    order = torch.randperm(pool, generator=r.g, device=DEV).tolist()
    pages, at = [], 0
    for n in counts:
        pages.append(order[at:at + n])
        at += n
    if case["kind"] == "cache":
        x.update(k=r.kv(sum(new), hkv), v=r.kv(sum(new), hkv))
        for t in ("k", "v"):
            x[t + "_codes"] = torch.zeros((pool, page, hkv, D), dtype=torch.uint8, device=DEV)
            x[t + "_scales"] = torch.zeros((pool, hkv, page), dtype=F32, device=DEV)
        return new, kv, pages, x
    x["q"] = r.normal((sum(new), case["hq"], D))
    for t in ("k", "v"):
        codes, scales = _quantize(r.kv(pool * page, hkv), case["fmt"])
        x[t + "_codes"] = codes.view(pool, page, hkv, D)
        x[t + "_scales"] = scales.view(pool, page, hkv).transpose(1, 2).contiguous()
    return new, kv, pages, x


def prepare(case, seed):
    new, kv, pages, x = _inputs(case, seed)
    s = dict(case, **x)
    if own:   # what a user of the framework keeps: the pool and the batch's tables and lengths
        from waveforcing_amd import backend
        from waveforcing_amd import kv as wkv

        if case["kind"] == "cross":
            s["batch"] = wkv.CrossBatch(new, kv, DEV)
        else:
            cls = wkv.Int8PagePool if case["fmt"] == "int8" else wkv.Fp8PagePool
            pool = cls(x["k_codes"].shape[0], case["hkv"], D, case["page"], DEV)
            for t in ("k_codes", "v_codes", "k_scales", "v_scales"):
                getattr(pool, t).copy_(s.pop(t))
            s["batch"] = wkv.PagedBatch(pool, pages, kv, new)
        s["ops"] = backend
        return s
    as_dev = lambda v: torch.tensor(v, dtype=torch.int64, device=DEV)
    s["seq"] = as_dev([b for b, n in enumerate(new) for _ in range(n)])
    s["row"] = as_dev([i for n in new for i in range(n)])
    s["new_lens"], s["kv_lens"] = as_dev(new), as_dev(kv)
    s["most"] = (max(new), max(kv))
    s["starts"] = as_dev([sum(new[:b]) for b in range(len(new))])
    if pages is None:
        s["k_starts"] = as_dev([sum(kv[:b]) for b in range(len(kv))])
    else:
        wide = max(1, max(len(p) for p in pages))
        s["tables"] = as_dev([p + [0] * (wide - len(p)) for p in pages])
    return s


# -------------------------------------------------------------------- run
def _cache_plain(s):
    pos = s["kv_lens"][s["seq"]] - s["new_lens"][s["seq"]] + s["row"]
    page, at = s["tables"][s["seq"], pos // s["page"]], pos % s["page"]
    out = {}
    for t in ("k", "v"):
        codes, scales = s[t + "_codes"], s[t + "_scales"]
        codes[page, at], scales[page, :, at] = _quantize(s[t], s["fmt"])
        out[t] = (_values(codes[page, at], s["fmt"]) * scales[page, :, at][..., None]).to(BF16)
    return out


def _attend_plain(s, k, v, seen):
    """k, v [B, Lk, Hkv, D] fp32, rows past a sequence's length zero; seen [B, Lq, Lk]."""
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


def _attn_plain(s):
    key = torch.arange(s["most"][1], device=DEV)
    page, at = s["tables"][:, key // s["page"]], key % s["page"]
    here = key < s["kv_lens"][:, None]
    kv = []
    for t in ("k", "v"):
        x = _values(s[t + "_codes"][page, at], s["fmt"]) * s[t + "_scales"].transpose(1, 2)[page, at][..., None]
        kv.append(x.masked_fill_(~here[..., None, None], 0))
    seen = here[:, None, :]
    if s["block"]:
        pos = (s["kv_lens"] - s["new_lens"])[:, None] + torch.arange(s["most"][0], device=DEV)
        seen = seen & (key < (pos // s["block"] + 1)[..., None] * s["block"])
    return _attend_plain(s, *kv, seen)


def _cross_plain(s):
    key = torch.arange(s["most"][1], device=DEV)
    here = key < s["kv_lens"][:, None]
    at = (s["k_starts"][:, None] + key).clamp(max=s["k"].shape[0] - 1)
    kv = [s[t][at].float().masked_fill_(~here[..., None, None], 0) for t in ("k", "v")]
    return _attend_plain(s, *kv, here[:, None, :])


def run(s):
    if own:
        if s["kind"] == "cache":
            s["batch"].append(s["k"], s["v"])
            k, v = s["batch"].gather()
            return dict(k=k, v=v)
        if s["kind"] == "attn":
            return s["ops"].attn_paged_batch(s["q"], s["batch"], block=s["block"], softmax_scale=SCALE)
        return s["ops"].attn_cross_batch(s["q"], s["k"], s["v"], s["batch"], softmax_scale=SCALE)
    return {"cache": _cache_plain, "attn": _attn_plain, "cross": _cross_plain}[s["kind"]](s)


# ------------------------------------------------------------------- work
def work(case):
    new, kv = _lens(case)
    hkv = case["hkv"]
    if case["kind"] == "cache":
        return dict(bytes=4 * sum(new) * hkv * (3 * D + 4), flops=0)
    seen = 0
    for n, t in zip(new, kv):
        if case["kind"] == "cross" or not case["block"]:
            seen += n * t
        else:
            b = case["block"]
            seen += sum(min(t, (p // b + 1) * b) for p in range(t - n, t))
    key = 4 * D if case["kind"] == "cross" else 2 * (D + 4)
    read = sum(t for n, t in zip(new, kv) if n)
    return dict(bytes=4 * D * sum(new) * case["hq"] + key * hkv * read, flops=4 * D * seen * case["hq"])


# ------------------------------------------------ the same in 64 bits
def _decode(codes, fmt):
    """The numbers that the bytes stand for, from the formats' definitions."""
    c = torch.arange(256, device=DEV)
    if fmt == "int8":
        table = torch.where(c < 128, c, c - 256).to(F64)
    else:
        e, m = (c >> 3) & 15, (c & 7).to(F64)
        mag = torch.where(e > 0, torch.ldexp(8 + m, (e - 10).to(F64)), torch.ldexp(m, torch.full_like(m, -9)))
        table = torch.where(c >= 128, -mag, mag)
        table[127] = table[255] = math.nan
    return table[codes.long()]


def _stored(x, fmt):
    """A K or V row after the cache: the nearest of its scale's multiples (int8) or of the e4m3 numbers times it."""
    x = x.to(F64)
    amax = x.abs().amax(-1, keepdim=True)
    if fmt == "int8":
        s = (amax / 127).to(F32).to(F64).clamp(min=1e-8)
        return torch.round((x / s).to(F32).to(F64)).clamp(-127, 127) * s
    s = (amax / 448).to(BF16).to(F64).clamp(min=float(torch.tensor(1e-8, dtype=BF16)))
    y = (x / s).clamp(-448, 448)
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * s


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
    new, kv, pages, x = _inputs(case, seed)
    if case["kind"] == "cache":
        return dict(k=_stored(x["k"], case["fmt"]), v=_stored(x["v"], case["fmt"]))
    out, at, k_at = torch.zeros(x["q"].shape, dtype=F64, device=DEV), 0, 0
    for b, (n, t) in enumerate(zip(new, kv)):
        pos = torch.arange(t - n, t, device=DEV)
        limit = torch.full_like(pos, t)
        if case["kind"] == "cross":
            k, v = (x[y][k_at:k_at + t].to(F64) for y in ("k", "v"))
            limit = torch.full((n,), t, device=DEV)
        else:
            if case["block"]:
                limit = torch.minimum(limit, (torch.div(pos, case["block"], rounding_mode="floor") + 1) * case["block"])
            ids = torch.tensor(pages[b], dtype=torch.int64, device=DEV)
            k, v = ((_decode(x[y + "_codes"][ids], case["fmt"]) * x[y + "_scales"][ids].transpose(1, 2).to(F64)[..., None])
                    .reshape(-1, case["hkv"], D)[:t] for y in ("k", "v"))
        if n and t:
            out[at:at + n] = _softmax_product(x["q"][at:at + n].to(F64), k, v, limit)
        at, k_at = at + n, k_at + t
    return out
