"""Attention over MXFP4 pages whose V has the largest scales that pages hold: results as finite as the definition's, against
64 bits within the arithmetic's bound (oracle/batch.py: attend)."""

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


def make(hkv, page, kv, new, seed):
    """A pool of random codes, scales of 2^-2, and a batch over shuffled pages of it."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    counts = [-(-t // page) for t in kv]
    pool = Mxfp4PagePool(sum(counts), hkv, 128, page, DEV)
    order = torch.randperm(sum(counts), generator=g, device=DEV).tolist()
    for t in "kv":
        codes = getattr(pool, t + "_codes")
        codes.copy_(torch.randint(0, 256, codes.shape, generator=g, device=DEV, dtype=torch.int64).to(torch.uint8))
        getattr(pool, t + "_scales").fill_(125)
    return pool, PagedBatch(pool, [[order.pop() for _ in range(c)] for c in counts], kv, new), g


def queries(n, heads, g):
    return torch.randn((n, heads, 128), generator=g, device=DEV).bfloat16()


def check_blocks(out, q, pool, batch, block, scale=SCALE):
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
            ref, bound = (x[..., i:i + 32] for x in ob.attend(q[at:at + n], k, vi, lim, scale))
            off = (out[at:at + n, :, i:i + 32].double() - ref).abs() - bound
            assert bool((off <= 0).all()), f"sequence {b}, dims {i}..: over the bound by {float(off.nan_to_num(math.inf).max()):.3g}"
        at += n


@pytest.mark.parametrize("byte", [252, 240, 200])
@pytest.mark.parametrize("new", [1, 5, 24, 60, 65, 200])
def test_values_of_the_largest_scales(new, byte):
    pool, batch, g = make(2, 64, [400, 9001, 250], [new, new, 0], new)
    pool.v_scales.fill_(byte)
    q = queries(batch.n_new, 4, g)
    for block in (1, 0):
        check_blocks(backend.attn_paged_batch(q, batch, block=block), q, pool, batch, block)
    small, batch, g = make(1, 16, [333], [new], new + 1)   # pages below a tile
    small.v_scales.fill_(byte)
    q = queries(new, 2, g)
    check_blocks(backend.attn_paged_batch(q, batch, block=1), q, small, batch, 1)


@pytest.mark.parametrize("rise", [0.5, 2, 8, 16])
@pytest.mark.parametrize("new", [1, 60, 100])
def test_rising_scores_over_the_largest_values(new, rise):
    """Scores of 0 and, in one key of each page, of `rise` (a power of two, in log2 units), twice that, four times, ... up to 64 times;
    V is 2^125 in every key."""
    pool, batch, g = make(1, 64, [640], [new], 7)
    pool.k_codes.zero_()
    pool.k_scales.fill_(127)
    pool.v_codes.fill_(0x22)                           # 1
    pool.v_scales.fill_(252)
    key = torch.zeros((1, 128), dtype=torch.bfloat16, device=DEV)
    key[0, 0] = rise
    c, s = om.quantize(key)
    for i, page in enumerate(batch.pages[0]):
        pool.k_codes[page, 17, 0] = om.pack(c)[0]
        pool.k_scales[page, 0, 17] = s[0] + min(i, 6)
    q = torch.zeros((new, 1, 128), dtype=torch.bfloat16, device=DEV)
    q[:, 0, 0] = 1.0
    scale = math.log(2)
    check_blocks(backend.attn_paged_batch(q, batch, block=0, softmax_scale=scale), q, pool, batch, 0, scale)


@pytest.mark.parametrize("new", [1, 40, 100])
def test_one_late_key_of_a_large_value(new):
    """A first tile of scores 0, then one key 2^16 times as heavy with V = 2^112: its weight times V passes fp32."""
    pool, batch, g = make(1, 64, [200], [new], 8)
    pool.k_codes.zero_()
    pool.v_codes.zero_()
    page = batch.pages[0][2]
    pool.k_codes[page, 5, 0, 0] = 0x06                 # 4 in dim 0
    pool.k_scales[page, 0, 5, 0] = 129                 # times 4
    pool.v_codes[page, 5] = 0x22                       # 1 everywhere
    pool.v_scales[page, 0, 5] = 127 + 112
    q = torch.zeros((new, 1, 128), dtype=torch.bfloat16, device=DEV)
    q[:, 0, 0] = 1.0
    out = backend.attn_paged_batch(q, batch, block=0, softmax_scale=math.log(2))
    check_blocks(out, q, pool, batch, 0, math.log(2))
    assert bool(torch.isfinite(out).all()) and float(out.min()) > 2.0 ** 111


@pytest.mark.parametrize("new", [1, 60, 200])
def test_blocks_of_far_scales_keep_their_own(new):
    """Blocks of one row 2^30 apart, at both ends and the middle of the range, keys of each."""
    for top in (252, 160, 127, 100):
        pool, batch, g = make(2, 64, [500, 70], [new, min(new, 70)], 9)
        pool.v_scales.copy_(torch.tensor([top, top - 30, top - 3, top - 12], dtype=torch.uint8, device=DEV).expand_as(pool.v_scales))
        q = queries(batch.n_new, 4, g)
        check_blocks(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)


@pytest.mark.parametrize("new", [1, 40, 100])
def test_a_nan_scale_reaches_rows_of_zero_queries(new):
    pool, batch, g = make(1, 64, [150], [new], 10)
    q = queries(new, 2, g)
    q[0] = 0
    clean = backend.attn_paged_batch(q, batch, block=0)
    check_blocks(clean, q, pool, batch, 0)
    for t in "kv":
        for byte in (255, 253):
            keep = getattr(pool, t + "_scales").clone()
            getattr(pool, t + "_scales")[batch.pages[0][0], 0, 3, 2] = byte
            assert bool(torch.isnan(backend.attn_paged_batch(q, batch, block=0)).all())
            getattr(pool, t + "_scales").copy_(keep)
