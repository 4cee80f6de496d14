"""Attention of many rows over MXFP4 pages: weights of 11 significant bits where V's scales lie in 2^-19 .. 2^12 (scale bytes 108 to
139), of 8 where one does not, and the same tiles, pages and splits with both."""

import math

import pytest
import torch

from oracle import batch as ob
from oracle import mxfp4 as om
from waveforcing_amd import backend
from waveforcing_amd.kv import Mxfp4PagePool, PagedBatch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SCALE = 128 ** -0.5


def make(hkv, page, kv, new, seed, spare=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    counts = [-(-t // page) for t in kv]
    pool = Mxfp4PagePool(sum(counts) + spare, hkv, 128, page, DEV)
    order = torch.randperm(sum(counts) + spare, generator=g, device=DEV).tolist()
    for t in "kv":
        codes = getattr(pool, t + "_codes")
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device=DEV, dtype=torch.int64).to(torch.uint8))
        getattr(pool, t + "_scales").fill_(125)
    return pool, PagedBatch(pool, [[order.pop() for _ in range(c)] for c in counts], kv, new), g


def queries(n, heads, g):
    return torch.randn((n, heads, 128), generator=g, device=DEV).bfloat16()


def check(out, q, pool, batch, block):
    """Each block of 32 dims against the definition, within the bound that the values of that block alone give."""
    at = 0
    for b, (t, n) in enumerate(zip(batch.kv_lens, batch.new_lens)):
        if not n:
            continue
        k, v = (om.cached(getattr(pool, x + "_codes"), getattr(pool, x + "_scales"), batch.pages[b], t, pool.page_tokens) for x in "kv")
        lim = [ob.limit(t - n + i, t, block) for i in range(n)]
        for i in range(0, 128, 32):
            vi = torch.zeros_like(v)
            vi[..., i:i + 32] = v[..., i:i + 32]
            ref, bound = (x[..., i:i + 32] for x in ob.attend(q[at:at + n], k, vi, lim, SCALE))
            off = (out[at:at + n, :, i:i + 32].double() - ref).abs() - bound
            assert bool((off <= 0).all()), f"sequence {b}, dims {i}..: over the bound by {float(off.nan_to_num(math.inf).max()):.3g}"
        at += n


@pytest.mark.parametrize("page", [16, 64])
def test_weights_of_two_keys(page):
    """Row i gives a key of V = 1 the weight 1 and one of V = -1 the weight p = 2^-d(i); the others have none.  The result is
    (1 - p) / (1 + p).

    fp16 rounds p by at most 2^-11 of it, which moves the result by at most 2 p / (1 + p)^2 <= 1/2 of that.  Q is exact to 2^-13 of its row's largest
    value, 1/4, and K is 1: d is off by at most 2^-15, fp32 steps included by 2^-14, and p by ln 2 times that, the result by half of it.  One
    rounding to bf16: 2^-8 of the result."""
    new = 256
    pool, batch, g = make(1, page, [new], [new], 1)
    ids = batch.pages[0]
    pool.k_codes.zero_()
    pool.v_codes.fill_(0x22)                           # 1
    pool.k_scales.fill_(127)
    pool.v_scales.fill_(127)
    pool.k_codes[:, :, :, 0] = 0xf0                    # dim 1 of every key: -6 times 2^20
    pool.k_scales[:, :, :, 0] = 147
    for key, code in ((5, 0x00), (9, 0x02)):           # dim 0: 0 and 1
        pool.k_codes[ids[key // page], key % page, 0, 0] = code
        pool.k_scales[ids[key // page], 0, key % page, 0] = 127
    pool.v_codes[ids[9 // page], 9 % page] = 0xaa      # -1
    q = torch.zeros((new, 1, 128), dtype=torch.bfloat16, device=DEV)
    q[:, 0, 0] = -0.25 * torch.arange(new, device=DEV).div(new)
    q[:, 0, 1] = 0.25
    out = backend.attn_paged_batch(q, batch, block=0, softmax_scale=math.log(2)).double()
    p = torch.exp2(q[:, 0, 0].double())
    ref = ((1 - p) / (1 + p))[:, None, None].expand_as(out)
    bound = 2.0 ** -12 + 0.5 * math.log(2) * 2.0 ** -14 + 2.0 ** -8 * ref + 2.0 ** -20
    off = (out - ref).abs() - bound
    assert bool((off <= 0).all()), f"over the bound by {float(off.max()):.3g}"


@pytest.mark.parametrize("page", [7, 16, 64, 390])
def test_scales_around_what_fp16_holds(page):
    for byte in (107, 108, 109, 139, 140, 3, 2, 1):
        pool, batch, g = make(2, page, [700, 131], [300, 100], byte)
        pool.v_scales.fill_(byte)
        pool.v_scales[..., 1] = 125
        q = queries(batch.n_new, 4, g)
        check(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)


@pytest.mark.parametrize("page", [1, 16, 64, 100])
@pytest.mark.parametrize("at", [0, 1, 63, 64, 200, 511, 512, 2047, 2048, 2999])
def test_one_far_scale_among_others(at, page):
    """One key of a scale that fp16 does not hold, in the first tile, at tiles' edges, in another split: rows before and behind it."""
    pool, batch, g = make(1, page, [3000, 300], [200, 90], at + page)
    q = queries(batch.n_new, 2, g)
    clean = backend.attn_paged_batch(q, batch, block=1)
    check(clean, q, pool, batch, 1)
    pool.v_scales[batch.pages[0][at // page], 0, at % page, 2] = 127 + 40
    out = backend.attn_paged_batch(q, batch, block=1)
    check(out, q, pool, batch, 1)
    assert torch.equal(out[200:], clean[200:])
    pool.v_scales[batch.pages[0][at // page], 0, at % page, 2] = 30
    check(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)


@pytest.mark.parametrize("page", [16, 64])
def test_far_scales_that_no_row_sees_change_nothing(page):
    pool, batch, g = make(2, page, [333, 150], [100, 150], 3, spare=4)
    q = queries(batch.n_new, 4, g)
    clean = backend.attn_paged_batch(q, batch, block=1)
    check(clean, q, pool, batch, 1)
    seen = torch.zeros((pool.pool_pages, page), dtype=torch.bool, device=DEV)
    for ids, t in zip(batch.pages, batch.kv_lens):
        for i, p in enumerate(ids):
            seen[p, :min(page, t - page * i)] = True
    pool.v_scales.masked_fill_(~seen[:, None, :, None], 230)
    assert torch.equal(backend.attn_paged_batch(q, batch, block=1), clean)
    batch.tables[1, 0] = pool.pool_pages               # no page: zeros, whatever the others hold
    out = backend.attn_paged_batch(q, batch, block=1)
    assert torch.equal(out[:100], clean[:100]) and bool((out[100:100 + min(page, 150)] == 0).all())


def test_captured_attention_follows_the_scales():
    """A captured call replayed while V's scales leave what fp16 holds and come back, on two streams' graphs in turn."""
    pool, batch, g = make(2, 64, [900, 200], [150, 70], 11)
    q = queries(batch.n_new, 4, g)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        backend.attn_paged_batch(q, batch, block=1)
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(backend.attn_paged_batch(q, batch, block=1))
    for byte in (125, 200, 125, 60, 252, 125):
        pool.v_scales[batch.pages[0][3], :, 17, 1] = byte
        q.copy_(queries(batch.n_new, 4, g))
        want = backend.attn_paged_batch(q, batch, block=1)
        check(want, q, pool, batch, 1)
        torch.cuda.synchronize()
        for i, graph in enumerate(graphs):
            with torch.cuda.stream(side if i else torch.cuda.current_stream()):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, want) for o in outs)
