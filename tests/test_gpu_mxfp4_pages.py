"""MXFP4 pages of batched sequences on the GPU: appended rows against the definition bit for bit, attention over them
against 64 bits within the arithmetic's bound (oracle/batch.py: attend), and a layer of 4-bit linears, cache and attention."""

import pytest
import torch

from oracle import batch as ob
from oracle import mxfp4 as om
from waveforcing_amd import backend
from waveforcing_amd.kv import Fp8PagePool, Mxfp4PagePool, PagedBatch
from waveforcing_amd.mxfp4 import WaveMxfp4Linear

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SCALE = 128 ** -0.5


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(n, heads, g, scale=1.0):
    return (torch.randn((n, heads, 128), generator=g, device=DEV) * scale).bfloat16()


def stored(x):
    """(code bytes, scale bytes) of rows [..., 128]: a row with a NaN or an infinity is NaN whole."""
    c, s = om.quantize(x)
    bad = (s == 255).any(-1)
    return om.pack(c.masked_fill(bad[..., None], 0)), s.masked_fill(bad[..., None], 255)


def read(codes, scales):
    return om.values(om.unpack(codes), scales)


def make(hkv, page, kv, new, seed, spare=2, fill=True):
    """A pool whose every page holds something, and a batch over shuffled pages of it."""
    g = gen(seed)
    counts = [-(-t // page) for t in kv]
    n = sum(counts) + spare
    pool = Mxfp4PagePool(n, hkv, 128, page, DEV)
    order = torch.randperm(n, generator=g, device=DEV).tolist()
    pages = [[order.pop() for _ in range(c)] for c in counts]
    if fill:
        for t in ("k", "v"):
            x = rows(n * page, hkv, g)
            x[:, :, 5] *= 9.0   # a heavy channel
            c, s = stored(x)
            getattr(pool, t + "_codes").copy_(c.view(n, page, hkv, 64))
            getattr(pool, t + "_scales").copy_(s.view(n, page, hkv, 4).transpose(1, 2))
    return pool, PagedBatch(pool, pages, kv, new), g


def cached(pool, batch, b, which, lens=None):
    return om.cached(getattr(pool, which + "_codes"), getattr(pool, which + "_scales"), batch.pages[b], (lens or batch.kv_lens)[b],
                     pool.page_tokens)


def same(x, y):
    differ = int((x != y).sum()) if x.shape == y.shape and x.dtype == y.dtype else -1
    assert differ == 0, f"{differ} of {x.numel()} values differ ({tuple(x.shape)}, {tuple(y.shape)})"


def check(out, ref, bound):
    out = out.double()
    if not out.numel():
        return
    assert bool((torch.isnan(out) == torch.isnan(ref)).all())
    off = ((out - ref).abs() - bound).nan_to_num(0)
    assert float(off.max()) <= 0, f"off by {float((out - ref).abs().nan_to_num(0).max()):.3g}, over the bound by {float(off.max()):.3g}"


def check_paged(out, q, pool, batch, block, scale=SCALE):
    at = 0
    for b, (t, n) in enumerate(zip(batch.kv_lens, batch.new_lens)):
        if n:
            lim = [ob.limit(t - n + i, t, block) for i in range(n)]
            check(out[at:at + n], *ob.attend(q[at:at + n], cached(pool, batch, b, "k"), cached(pool, batch, b, "v"), lim, scale))
        at += n


# ------------------------------------------------------------------- cache
@pytest.mark.parametrize("kv, new", [([1], [1]), ([1, 0, 70, 129], [1, 0, 1, 129]), ([50, 33, 200, 777], [5, 33, 0, 64]),
                                     ([9] * 70, [1, 2, 0, 3, 1] * 14), ([1600, 900], [1599, 700])])
@pytest.mark.parametrize("hkv, page", [(1, 16), (12, 390), (5, 7), (2, 1)])
def test_append_and_gather(hkv, page, kv, new):
    pool, batch, g = make(hkv, page, kv, new, 10 + len(kv), fill=False)
    n = sum(new)
    x = {"k": rows(n + 3, hkv, g, 2.0), "v": rows(n + 3, hkv, g, 0.01)}   # 3 padding rows
    x["k"][0, 0, 32:64] = 0                           # the smallest scale
    x["k"][n - 1, hkv - 1, 3] = float("nan")
    x["v"][n - 1, 0, 99] = float("inf")
    want = {t: (getattr(pool, t + "_codes").clone(), getattr(pool, t + "_scales").clone()) for t in x}
    pages = torch.tensor([batch.pages[b][p // page] for b, p in ob.row_positions(kv, new)], device=DEV)
    at = torch.tensor([p % page for _, p in ob.row_positions(kv, new)], device=DEV)
    for t in x:
        want[t][0][pages, at], want[t][1][pages, :, at] = stored(x[t][:n])
    batch.append(x["k"], x["v"])
    for t in x:
        same(getattr(pool, t + "_codes"), want[t][0])
        same(getattr(pool, t + "_scales"), want[t][1])
    for t, got in zip("kv", batch.gather()):
        ref = read(want[t][0][pages, at], want[t][1][pages, :, at]).float().bfloat16()
        torch.testing.assert_close(got, ref, rtol=0, atol=0, equal_nan=True)
        last = hkv - 1 if t == "k" else 0
        assert bool(torch.isnan(got[n - 1, last]).all())


def test_pages_hold_what_the_rows_quantizer_gives():
    from waveforcing_amd import mxfp4

    pool, batch, g = make(12, 390, [1000], [1000], 5, fill=False)
    k, v = rows(1000, 12, g, 3.0), rows(1000, 12, g)
    batch.append(k, v)
    whole = PagedBatch(pool, batch.pages, [1000], [1000])
    for x, got in zip((k, v), whole.gather()):
        same(got, mxfp4.dequant_mxfp4(*mxfp4.quant_mxfp4(x.view(12000, 128))).view(1000, 12, 128))


def test_strided_rows_k_only_and_views():
    pool, batch, g = make(3, 16, [40, 21], [10, 5], 3)
    before = pool.v_codes.clone()
    qkv = rows(15, 9, g)
    batch.append(qkv[:, 3:6], None)                    # a column slice of a fused projection, K only
    same(pool.v_codes, before)
    out = torch.full((20, 6, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    batch.gather(with_v=False, out_k=out[:, 1:4])
    assert bool((out[15:] == 7).all() & (out[:, 4:] == 7).all() & (out[:, 0] == 7).all())
    same(out[:15, 1:4], read(*stored(qkv[:, 3:6].contiguous())).float().bfloat16())
    view = Mxfp4PagePool.view_of(pool, 2, 3)
    assert view.k_codes.shape == (3, 16, 3, 64) and view.k_scales.shape == (3, 3, 16, 4)
    one = PagedBatch(view, [[1]], [16], [16])
    same(one.gather()[0], om.cached(pool.k_codes, pool.k_scales, [3], 16, 16).float().bfloat16())


def test_device_lengths_and_bad_pages_stay_in_bounds():
    pool, batch, g = make(2, 16, [30, 8], [4, 8], 6)
    keep = {t: getattr(pool, t).clone() for t in ("k_codes", "k_scales")}
    batch.tables[0, 1] = pool.pool_pages              # outside the pool
    batch.kv_lens_dev[1] = 5                          # 8 rows, 5 positions: three rows before position 0
    x = rows(12, 2, g)
    batch.append(x, x)
    k, v = (torch.full((12, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    batch.gather(out_k=k, out_v=v)
    assert bool((k[:7] == 7).all()) and bool((k[7:] != 7).any())
    fresh = batch.gather()[0]
    assert bool((fresh[:7] == 0).all())
    other = [i for i in range(pool.pool_pages) if i != batch.pages[1][0]]
    for t, c in keep.items():
        same(getattr(pool, t)[other], c[other])
    q = rows(12, 2, g)
    out = backend.attn_paged_batch(q, batch, block=1)
    none = torch.zeros((14, 2, 128), dtype=torch.float64, device=DEV)
    zk, zv = (torch.cat([cached(pool, batch, 0, t)[:16], none]) for t in "kv")
    check(out[:4], *ob.attend(q[:4], zk, zv, [27, 28, 29, 30], SCALE))
    assert bool((out[4:7] == 0).all())
    k1, v1 = (cached(pool, batch, 1, t)[:5] for t in "kv")
    check(out[7:], *ob.attend(q[7:], k1, v1, [1, 2, 3, 4, 5], SCALE))


@pytest.mark.parametrize("new", [1, 90])
def test_missing_pages_take_no_other_pages_scales(new):
    """Page 0 holds NaN everywhere; a table entry outside the pool, read in its place, still reads as zero."""
    for page in (16, 64):
        pool, batch, g = make(2, page, [200], [new], 7, spare=6)
        spare = next(i for i in range(pool.pool_pages) if i not in batch.pages[0])
        if 0 in batch.pages[0]:                       # move what page 0 holds
            i = batch.pages[0].index(0)
            for t in ("k_codes", "v_codes", "k_scales", "v_scales"):
                getattr(pool, t)[spare] = getattr(pool, t)[0]
            batch.pages[0][i] = spare
            batch.tables[0, i] = spare
        for t in ("k", "v"):
            getattr(pool, t + "_codes")[0] = 0x77
            getattr(pool, t + "_scales")[0] = 255
        batch.tables[0, 1] = -5
        q = rows(new, 4, g)
        out = backend.attn_paged_batch(q, batch, block=0)
        zk, zv = cached(pool, batch, 0, "k"), cached(pool, batch, 0, "v")
        zk[page:2 * page] = 0
        zv[page:2 * page] = 0
        check(out, *ob.attend(q, zk, zv, [200] * new, SCALE))


# --------------------------------------------------------------- attention
ATTN_LENS = [([1], [1]), ([1, 64, 70, 129, 3], [1, 1, 0, 1, 1]), ([5, 40, 0, 200, 777, 65], [5, 33, 0, 64, 1, 2]),
             ([700, 1000], [300, 17]), ([130], [130]), ([2000, 300], [40, 299]), ([257] * 66, [1] * 66)]


@pytest.mark.parametrize("lens", range(len(ATTN_LENS)))
@pytest.mark.parametrize("block", [0, 1, 48])
@pytest.mark.parametrize("hkv, group, page", [(3, 1, 390), (2, 1, 16), (1, 5, 16), (2, 4, 7), (2, 16, 64), (1, 3, 1), (2, 2, 33)])
def test_paged_attention(hkv, group, page, block, lens):
    kv, new = ATTN_LENS[lens]
    pool, batch, g = make(hkv, page, kv, new, 30 + lens)
    q = rows(sum(new), hkv * group, g)
    out = backend.attn_paged_batch(q, batch, block=block)
    check_paged(out, q, pool, batch, block)
    same(out, backend.attn_paged_batch(q, batch, block=block))


@pytest.mark.parametrize("new", [1, 3, 20, 70, 333])
def test_long_cache_splits(new):
    pool, batch, g = make(2, 64, [9001, 100, 5000, 64 * 70], [new, min(new, 100), 0, 1], 40)
    q = rows(batch.n_new, 8, g)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)


EDGES = [15, 16, 17, 32, 33, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257]


@pytest.mark.parametrize("group", [1, 3])
def test_row_counts_around_the_tiles(group):
    kv = [n + 64 - n % 64 + i % 3 - 1 for i, n in enumerate(EDGES)]
    for new, t in ((EDGES, [max(a, b) for a, b in zip(kv, EDGES)]), ([0, 3, 70, 1] * 40, [80 + i % 3 for i in range(160)])):
        pool, batch, g = make(2, 32, t, new, 140)
        q = rows(sum(new), 2 * group, g)
        for block in (1, 0):
            check_paged(backend.attn_paged_batch(q, batch, block=block), q, pool, batch, block)


@pytest.mark.parametrize("new", [2, 90])
def test_strides_padding_and_given_outputs(new):
    pool, batch, g = make(2, 48, [300, 150], [new, new], 60)
    n = batch.n_new
    wide = rows(n + 5, 9, g)
    q = wide[:, 1:5]                                   # 4 of 9 heads' columns
    out = torch.full((n + 5, 6, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    backend.attn_paged_batch(q, batch, block=1, out=out[:, :4])
    assert bool((out[n:] == 7).all()) and bool((out[:, 4:] == 7).all())
    check_paged(out[:n, :4], q[:n], pool, batch, 1)
    fresh = backend.attn_paged_batch(q, batch, block=1, softmax_scale=0.3)
    assert bool((fresh[n:] == 0).all())
    check_paged(fresh[:n], q[:n], pool, batch, 1, scale=0.3)


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("new", [1, 7, 150])
def test_nothing_unseen_reaches_a_row(new, page):
    """NaN scales behind a sequence's end, in pages of no sequence and in positions that a row's mask hides."""
    pool, batch, g = make(2, page, [200, 151], [new, new], 70)
    q = rows(batch.n_new, 4, g)
    clean = backend.attn_paged_batch(q, batch, block=1)
    check_paged(clean, q, pool, batch, 1)
    keep = torch.zeros((pool.pool_pages, page), dtype=torch.bool, device=DEV)
    for ids, t in zip(batch.pages, batch.kv_lens):
        for i, p in enumerate(ids):
            keep[p, :min(page, t - page * i)] = True
    for t in ("k", "v"):
        getattr(pool, t + "_codes").masked_fill_(~keep[:, :, None, None], 0x7f)
        getattr(pool, t + "_scales").masked_fill_(~keep[:, None, :, None], 255 if t == "k" else 254)
    same(backend.attn_paged_batch(q, batch, block=1), clean)
    # the last position of sequence 0: a NaN scale of one block of K, then of V: its last row alone sees it
    at, row = batch.pages[0][199 // page], 199 % page
    for t in ("k", "v"):
        for byte, block in ((255, 0), (254, 3), (253, 2)):
            save = getattr(pool, t + "_scales").clone()
            getattr(pool, t + "_scales")[at, :, row, block] = byte
            out = backend.attn_paged_batch(q, batch, block=1)
            assert bool(torch.isnan(out[new - 1]).all())
            out[new - 1] = clean[new - 1]
            same(out, clean)
            getattr(pool, t + "_scales").copy_(save)
    # and through append: an infinite row of K
    k, v = rows(batch.n_new, 2, g), rows(batch.n_new, 2, g)
    k[new - 1, 1, 77] = float("-inf")
    batch.append(k, v)
    out = backend.attn_paged_batch(q, batch, block=1)
    assert bool(torch.isnan(out[new - 1, 2:]).all()) and not bool(torch.isnan(out[new - 1, :2]).any())
    assert not bool(torch.isnan(out[:new - 1]).any()) and not bool(torch.isnan(out[new:]).any())


@pytest.mark.parametrize("new", [1, 40, 100])
def test_queries_that_are_not_finite(new):
    pool, batch, g = make(1, 64, [400], [new], 75)
    q = rows(new, 2, g)
    clean = backend.attn_paged_batch(q, batch, block=1)
    q[new - 1, 0, 3] = float("inf")
    q[new - 1, 1, 127] = float("nan")
    out = backend.attn_paged_batch(q, batch, block=1)
    assert bool(torch.isnan(out[new - 1]).all())
    same(out[:new - 1], clean[:new - 1])


@pytest.mark.parametrize("new", [1, 40, 100])
def test_extreme_scores_and_scales(new):
    """Scores of +-10^4, rows whose first keys are far below their last, ties, blocks of far apart scales, a scale of zero."""
    pool, batch, g = make(1, 64, [400], [new], 80)
    q = rows(new, 2, g, 300.0)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)
    ids = torch.tensor(batch.pages[0], device=DEV)
    ramp = torch.arange(7 * 64, device=DEV).view(7, 1, 64, 1).expand(7, 1, 64, 4) // 64   # rising keys: the reference moves
    pool.k_scales[ids] = (124 + ramp).to(torch.uint8)
    check_paged(backend.attn_paged_batch(q, batch, block=0), q, pool, batch, 0)
    pool.k_codes.fill_(0x77)                           # every key the same: the mean of the values
    pool.k_scales.fill_(130)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)
    check_paged(backend.attn_paged_batch(q, batch, block=1, softmax_scale=0.0), q, pool, batch, 1, scale=0.0)
    # blocks of V and K from 2^-100 to 2^90, keys of each
    pool.v_scales.copy_(torch.tensor([27, 100, 127, 217], dtype=torch.uint8, device=DEV).expand_as(pool.v_scales))
    pool.k_scales.copy_(torch.tensor([27, 90, 126, 2], dtype=torch.uint8, device=DEV).expand_as(pool.k_scales))
    q = rows(new, 2, g)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)


@pytest.mark.parametrize("new", [1, 100])
def test_pools_past_32_bit_offsets(new):
    """Code pools of more than 4 GiB: pages at both ends."""
    page, hkv = 1560, 40
    n = 1120                                           # 1120 * 1560 * 40 * 64 = 4.47e9 bytes
    pool = Mxfp4PagePool(n, hkv, 128, page, DEV)
    batch = PagedBatch(pool, [[n - 1, 0], [n - 2]], [2000, 700], [new, new])
    g = gen(90)
    k, v, q = rows(2 * new, hkv, g), rows(2 * new, hkv, g), rows(2 * new, hkv, g)
    batch.append(k, v)
    for x, y in zip((k, v), batch.gather()):
        same(y, read(*stored(x)).float().bfloat16())
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, 1)


def test_streams_do_not_share_scratch():
    made = [make(2, 64, [6000 + 64 * i], [1 + 4 * i], 110 + i) for i in range(2)]
    qs = [rows(b.n_new, 8, g) for _, b, g in made]
    want = [backend.attn_paged_batch(q, b, block=1) for q, (_, b, _) in zip(qs, made)]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in made], [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(backend.attn_paged_batch(qs[i], made[i][1], block=1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


def test_captured_decode_follows_the_device_lengths():
    """One captured step (4-bit projection, append, attention, read-back) replayed while the lengths advance on the device."""
    pool, batch, g = make(2, 64, [250, 70, 1], [1, 1, 1], 120)
    capacity = PagedBatch(pool, batch.pages, batch.kv_lens, [1, 1, 1], max_kv=256)
    qkv = WaveMxfp4Linear(torch.randn((12 * 128, 256), generator=g, device=DEV).bfloat16() * 0.06, None)
    x = rows(3, 2, g)

    def step(over):
        y = qkv(x.view(3, 256))[0].view(3, 12, 128)
        over.append(y[:, 8:10], y[:, 10:])
        return backend.attn_paged_batch(y[:, :8], over, block=1), *over.gather()

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(capacity)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(capacity)
    for i in range(4):
        x.copy_(rows(3, 2, g))
        lens = [250 + i, 70 + i, 1 + i]
        capacity.kv_lens_dev.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        got = [o.clone() for o in outs]
        eager = PagedBatch(pool, batch.pages, lens, [1, 1, 1], max_kv=256)
        for a, b in zip(got, step(eager)):
            same(a, b)


def test_a_layer_in_four_bits_as_it_is_used():
    """Prompts, then single tokens, then idle and active streams through one layer: projection, append, attention, output
    projection, all in 4 bits, against 64 bits stage by stage; and the pages of an 8-bit pool side by side."""
    page, hkv, heads, dim = 64, 2, 4, 512
    g = gen(130)
    weight = lambda n, k: (torch.randn((n, k), generator=g, device=DEV) * k ** -0.5).bfloat16()
    qkv_w, o_w, bias = weight((heads + 2 * hkv) * 128, dim), weight(dim, heads * 128), weight(1, (heads + 2 * hkv) * 128)[0]
    qkv, o = WaveMxfp4Linear(qkv_w, bias), WaveMxfp4Linear(o_w, None)
    pool, wide = Mxfp4PagePool(40, hkv, 128, page, DEV), Fp8PagePool(40, hkv, 128, page, DEV)
    assert pool.nbytes == Mxfp4PagePool.bytes_for(40, hkv, 128, page) and 1.9 < wide.nbytes / pool.nbytes < 2
    pages = [list(range(0, 8)), list(range(8, 20)), list(range(20, 24))]
    exact = lambda x: om.values(*om.quantize(x))
    kv, batch = [0, 0, 0], None
    for new in ([300, 129, 1], [1, 1, 1], [1, 0, 60], [0, 250, 2]):
        kv = [t + n for t, n in zip(kv, new)]
        if batch is None:
            batch = PagedBatch(pool, pages, kv, new)
        else:
            batch.set_lens(kv, new)
        n = sum(new)
        x = (torch.randn((n, dim), generator=g, device=DEV)).bfloat16()
        y = qkv(x)[0]
        check(y, *om.product(exact(x), exact(qkv_w), bias))
        y = y.view(n, -1, 128)
        batch.append(y[:, heads:heads + hkv], y[:, heads + hkv:])
        for z, got in zip((y[:, heads:heads + hkv], y[:, heads + hkv:]), batch.gather()):
            same(got, read(*stored(z.contiguous())).float().bfloat16())
        a = backend.attn_paged_batch(y[:, :heads], batch, block=1)
        check_paged(a, y[:, :heads], pool, batch, 1)
        a = a.view(n, -1)
        check(o(a)[0], *om.product(exact(a), exact(o_w)))
