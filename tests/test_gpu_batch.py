"""Batched sequences on the GPU: the paged cache of ragged rows against its definition bit for bit, attention over it and
over ragged encoder rows against 64 bits within the arithmetic's bound (oracle/batch.py: attend)."""

import pytest
import torch

from oracle import batch as ob
from waveforcing_amd import _lib, backend
from waveforcing_amd.kv import CrossBatch, Fp8PagePool, Int8PagePool, PagedBatch, PagedKV

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
SCALE = 128 ** -0.5
POOLS = {"e4m3": Fp8PagePool, "int8": Int8PagePool}


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(n, heads, g, scale=1.0):
    x = torch.randn((n, heads, 128), generator=g, device=DEV) * scale
    return x.bfloat16()


def make(fmt, hkv, page, kv, new, seed, spare=2, fill=True):
    """A pool whose every page holds something, and a batch over shuffled pages of it."""
    g = gen(seed)
    counts = [-(-t // page) for t in kv]
    n = sum(counts) + spare
    pool = POOLS[fmt](n, hkv, 128, page, DEV)
    order = torch.randperm(n, generator=g, device=DEV).tolist()
    pages = [[order.pop() for _ in range(c)] for c in counts]
    if fill:
        for t in ("k", "v"):
            x = rows(n * page, hkv, g)
            x[:, :, 5] *= 9.0   # a heavy channel
            c, s = ob.quantize(x, fmt)
            getattr(pool, t + "_codes").copy_(c.view(n, page, hkv, 128))
            getattr(pool, t + "_scales").copy_(s.view(n, page, hkv).transpose(1, 2))
    return pool, PagedBatch(pool, pages, kv, new), g


def cached(pool, batch, fmt, b, which):
    return ob.cached(getattr(pool, which + "_codes"), getattr(pool, which + "_scales"), fmt, batch.pages[b],
                     batch.kv_lens[b], pool.page_tokens)


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


def check_paged(out, q, pool, batch, fmt, block, scale=SCALE):
    at = 0
    for b, (t, n) in enumerate(zip(batch.kv_lens, batch.new_lens)):
        if n:
            lim = [ob.limit(t - n + i, t, block) for i in range(n)]
            ref, bound = ob.attend(q[at:at + n], cached(pool, batch, fmt, b, "k"), cached(pool, batch, fmt, b, "v"), lim, scale)
            check(out[at:at + n], ref, bound)
        at += n


# ------------------------------------------------------------------- cache
CACHE_LENS = [([1], [1]), ([1, 0, 70, 129], [1, 0, 1, 129]), ([50, 33, 200, 777], [5, 33, 0, 64]),
              ([9] * 70, [1, 2, 0, 3, 1] * 14), ([1600, 900], [1599, 700])]


@pytest.mark.parametrize("lens", range(len(CACHE_LENS)))
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("hkv, page", [(1, 16), (12, 390), (5, 7), (2, 1)])
def test_append_and_gather(fmt, hkv, page, lens):
    kv, new = CACHE_LENS[lens]
    pool, batch, g = make(fmt, hkv, page, kv, new, 10 + lens, fill=False)
    n = sum(new)
    x = {"k": rows(n + 3, hkv, g, 2.0), "v": rows(n + 3, hkv, g, 0.01)}   # 3 padding rows
    x["k"][0, 0] = 0                                  # the smallest scale
    x["k"][n - 1, hkv - 1, 3] = float("nan")
    x["v"][n - 1, 0, 9] = float("inf")
    want = {t: (getattr(pool, t + "_codes").clone(), getattr(pool, t + "_scales").clone()) for t in x}
    pages = torch.tensor([batch.pages[b][p // page] for b, p in ob.row_positions(kv, new)], device=DEV)
    at = torch.tensor([p % page for _, p in ob.row_positions(kv, new)], device=DEV)
    for t in x:
        c, s = ob.quantize(x[t][:n], fmt)
        want[t][0][pages, at], want[t][1][pages, :, at] = c, s
    batch.append(x["k"], x["v"])
    for t in x:
        same(getattr(pool, t + "_codes"), want[t][0])
        torch.testing.assert_close(getattr(pool, t + "_scales"), want[t][1], rtol=0, atol=0, equal_nan=True)
    got = dict(zip("kv", batch.gather()))
    for t in x:
        c = want[t][0][pages, at].view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float()
        ref = (c * want[t][1][pages, :, at][..., None]).bfloat16()
        torch.testing.assert_close(got[t], ref, rtol=0, atol=0, equal_nan=True)
    assert bool(torch.isnan(got["k"][n - 1, hkv - 1]).all()) and bool(torch.isnan(got["v"][n - 1, 0]).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_strided_rows_k_only_and_whole_caches(fmt):
    pool, batch, g = make(fmt, 3, 16, [40, 21], [10, 5], 3)
    before = pool.v_codes.clone()
    qkv = rows(15, 9, g)
    batch.append(qkv[:, 3:6], None)                    # a column slice of a fused projection, K only
    same(pool.v_codes, before)
    out = torch.full((20, 6, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    batch.gather(with_v=False, out_k=out[:, 1:4])
    assert bool((out[15:] == 7).all() & (out[:, 4:] == 7).all() & (out[:, 0] == 7).all())
    c, s = ob.quantize(qkv[:, 3:6].contiguous(), fmt)
    same(out[:15, 1:4], ob.values(c, s, fmt).float().bfloat16())
    whole = PagedBatch(pool, batch.pages, batch.kv_lens, batch.kv_lens)
    k, v = whole.gather()
    for b, at in ((0, 0), (1, 40)):
        n = batch.kv_lens[b]
        same(k[at:at + n], cached(pool, batch, fmt, b, "k").float().bfloat16())
        same(v[at:at + n], cached(pool, batch, fmt, b, "v").float().bfloat16())


def test_e4m3_pages_are_the_one_sequence_pages():
    pool, batch, g = make("e4m3", 12, 390, [1000], [1000], 5, fill=False)
    other = Fp8PagePool(pool.pool_pages, 12, 128, 390, DEV)
    k, v = rows(1000, 12, g, 3.0), rows(1000, 12, g)
    batch.append(k, v)
    table = other.page_table(batch.pages[0])
    other.pack(k, v, table)
    for t in ("k_codes", "v_codes", "k_scales", "v_scales"):
        same(getattr(pool, t), getattr(other, t))
    for a, b in zip(batch.gather(), other.unpack(table, 1000)):
        same(a, b)


def test_device_lengths_and_bad_pages_stay_in_bounds():
    """Lengths and tables changed on the device: positions without a page are not written, read as zero K and V by the
    attention, and leave gathered rows as they were."""
    pool, batch, g = make("int8", 2, 16, [30, 8], [4, 8], 6)
    keep = {t: getattr(pool, t).clone() for t in ("k_codes", "k_scales")}
    batch.tables[0, 1] = pool.pool_pages              # outside the pool
    batch.kv_lens_dev[1] = 5                          # 8 rows, 5 positions: three rows before position 0
    x = rows(12, 2, g)
    batch.append(x, x)
    k, v = (torch.full((12, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    batch.gather(out_k=k, out_v=v)
    assert bool((k[:7] == 7).all()) and bool((k[7:] != 7).any())
    other = [i for i in range(pool.pool_pages) if i != batch.pages[1][0]]
    for t, c in keep.items():
        same(getattr(pool, t)[other], c[other])
    q = rows(12, 2, g)
    out = backend.attn_paged_batch(q, batch, block=1)
    zk = torch.cat([cached(pool, batch, "int8", 0, "k")[:16], torch.zeros((14, 2, 128), dtype=torch.float64, device=DEV)])
    zv = torch.cat([cached(pool, batch, "int8", 0, "v")[:16], torch.zeros((14, 2, 128), dtype=torch.float64, device=DEV)])
    check(out[:4], *ob.attend(q[:4], zk, zv, [27, 28, 29, 30], SCALE))
    assert bool((out[4:7] == 0).all())
    k1, v1 = cached(pool, batch, "int8", 1, "k")[:5], cached(pool, batch, "int8", 1, "v")[:5]
    check(out[7:], *ob.attend(q[7:], k1, v1, [1, 2, 3, 4, 5], SCALE))


# --------------------------------------------------------------- attention
ATTN_LENS = [([1], [1]), ([1, 64, 70, 129, 3], [1, 1, 0, 1, 1]), ([5, 40, 0, 200, 777, 65], [5, 33, 0, 64, 1, 2]),
             ([700, 1000], [300, 17]), ([130], [130]), ([2000, 300], [40, 299]), ([257] * 66, [1] * 66)]


@pytest.mark.parametrize("lens", range(len(ATTN_LENS)))
@pytest.mark.parametrize("block", [0, 1, 48])
@pytest.mark.parametrize("fmt, hkv, group, page", [("e4m3", 3, 1, 390), ("int8", 2, 1, 16), ("e4m3", 1, 5, 16), ("int8", 2, 4, 7),
                                                   ("e4m3", 2, 16, 64), ("int8", 1, 3, 1)])
def test_paged_attention(fmt, hkv, group, page, block, lens):
    kv, new = ATTN_LENS[lens]
    pool, batch, g = make(fmt, hkv, page, kv, new, 30 + lens)
    q = rows(sum(new), hkv * group, g)
    out = backend.attn_paged_batch(q, batch, block=block)
    check_paged(out, q, pool, batch, fmt, block)
    same(out, backend.attn_paged_batch(q, batch, block=block))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [1, 3, 20, 70, 333])
def test_long_cache_splits(fmt, new):
    """Few rows over long caches (split and joined), in one batch with short ones."""
    pool, batch, g = make(fmt, 2, 64, [9001, 100, 5000, 64 * 70], [new, min(new, 100), 0, 1], 40)
    q = rows(batch.n_new, 8, g)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, fmt, 1)


@pytest.mark.parametrize("lens", [([1], [1]), ([5, 0, 300, 64, 65], [3, 4, 0, 1, 70]), ([2000, 77], [500, 4]), ([33] * 70, [1] * 70),
                                  ([4000, 1, 0, 900], [1, 2, 2, 1]), ([512, 40], [1100, 600])])
@pytest.mark.parametrize("hkv, group", [(3, 1), (1, 6), (4, 2), (2, 16)])
def test_cross_attention(hkv, group, lens):
    t, n = lens
    g = gen(50)
    batch = CrossBatch(n, t, DEV)
    q, k, v = rows(sum(n), hkv * group, g), rows(sum(t), hkv, g), rows(sum(t), hkv, g)
    k[:, :, 7] *= 9.0
    out = backend.attn_cross_batch(q, k, v, batch)
    a = c = 0
    for i, j in zip(n, t):
        check(out[a:a + i], *ob.attend(q[a:a + i], k[c:c + j], v[c:c + j], [j] * i, SCALE))
        a, c = a + i, c + j
    same(out, backend.attn_cross_batch(q, k, v, batch))


@pytest.mark.parametrize("new", [2, 90])
def test_strides_padding_and_given_outputs(new):
    pool, batch, g = make("e4m3", 2, 48, [300, 150], [new, new], 60)
    n = batch.n_new
    wide = rows(n + 5, 9, g)
    q = wide[:, 1:5]                                   # 4 of 9 heads' columns
    out = torch.full((n + 5, 6, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    backend.attn_paged_batch(q, batch, block=1, out=out[:, :4])
    assert bool((out[n:] == 7).all()) and bool((out[:, 4:] == 7).all())
    check_paged(out[:n, :4], q[:n], pool, batch, "e4m3", 1)
    fresh = backend.attn_paged_batch(q, batch, block=1, softmax_scale=0.3)
    assert bool((fresh[n:] == 0).all())
    check_paged(fresh[:n], q[:n], pool, batch, "e4m3", 1, scale=0.3)
    kv = rows(40, 6, g)
    cb = CrossBatch([new, new], [13, 20], DEV)
    out.fill_(7.0)
    backend.attn_cross_batch(q, kv[:, 1:3], kv[:, 4:6], cb, out=out[:, :4])
    assert bool((out[n:] == 7).all()) and bool((out[:, 4:] == 7).all())
    for a, c, j in ((0, 0, 13), (new, 13, 20)):
        check(out[a:a + new, :4], *ob.attend(q[a:a + new], kv[c:c + j, 1:3], kv[c:c + j, 4:6], [j] * new, SCALE))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [1, 7, 150])
def test_nothing_unseen_reaches_a_row(fmt, new):
    """NaN and infinities behind a sequence's end, in pages of no sequence and in positions that a row's mask hides."""
    pool, batch, g = make(fmt, 2, 16, [200, 151], [new, new], 70)
    q = rows(batch.n_new, 4, g)
    clean = backend.attn_paged_batch(q, batch, block=1)
    check_paged(clean, q, pool, batch, fmt, 1)
    used = [(p, list(range(min(16, t - 16 * i)))) for ids, t in zip(batch.pages, batch.kv_lens) for i, p in enumerate(ids)]
    keep = torch.zeros((pool.pool_pages, 16), dtype=torch.bool, device=DEV)
    for p, r in used:
        keep[p, r] = True
    for t in ("k", "v"):
        codes, scales = getattr(pool, t + "_codes"), getattr(pool, t + "_scales")
        codes.masked_fill_(~keep[:, :, None, None], 0x7f)
        scales.masked_fill_(~keep[:, None, :], float("nan") if t == "k" else float("inf"))
    same(backend.attn_paged_batch(q, batch, block=1), clean)
    if new == 1:
        return
    # the last position of sequence 0: a NaN key, then a NaN value (and an e4m3 NaN code): its last row alone sees it
    page, row = batch.pages[0][199 // 16], 199 % 16
    for t in ("k", "v"):
        save = getattr(pool, t + "_scales").clone()
        getattr(pool, t + "_scales")[page, :, row] = float("nan")
        out = backend.attn_paged_batch(q, batch, block=1)
        assert bool(torch.isnan(out[new - 1]).all())
        out[new - 1] = clean[new - 1]
        same(out, clean)
        getattr(pool, t + "_scales").copy_(save)
    if fmt == "e4m3":
        pool.v_codes[page, row, 0, 17] = 0x7f
        out = backend.attn_paged_batch(q, batch, block=1)
        assert bool(torch.isnan(out[new - 1, :2, 17]).all())
        out[new - 1] = clean[new - 1]
        same(out, clean)


@pytest.mark.parametrize("new", [1, 100])
def test_extreme_scores(new):
    """Scores of +-10^4 and rows whose first keys are far below their last: exact ties, no overflow, no lost rows."""
    pool, batch, g = make("int8", 1, 64, [400], [new], 80)
    q = rows(new, 2, g, 300.0)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, "int8", 1)
    pool.k_codes.fill_(0x7f)                           # every key the same: the mean of the values
    pool.k_scales.copy_(torch.full_like(pool.k_scales, 50.0))
    q = rows(new, 2, g, 300.0)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, "int8", 1)
    zero = backend.attn_paged_batch(q, batch, block=1, softmax_scale=0.0)
    check_paged(zero, q, pool, batch, "int8", 1, scale=0.0)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [1, 100])
def test_pools_past_32_bit_offsets(fmt, new):
    """Code pools of more than 4 GiB: pages at both ends."""
    page, hkv = 1560, 40
    n = 560                                            # 560 * 1560 * 40 * 128 = 4.47e9 codes
    pool = POOLS[fmt](n, hkv, 128, page, DEV)
    batch = PagedBatch(pool, [[n - 1, 0], [n - 2]], [2000, 700], [new, new])
    g = gen(90)
    k, v, q = rows(2 * new, hkv, g), rows(2 * new, hkv, g), rows(2 * new, hkv, g)
    batch.append(k, v)
    gk, gv = batch.gather()
    for x, y in ((k, gk), (v, gv)):
        c, s = ob.quantize(x, fmt)
        same(y, ob.values(c, s, fmt).float().bfloat16())
    out = backend.attn_paged_batch(q, batch, block=1)
    check_paged(out, q, pool, batch, fmt, 1)


def test_shared_prefix_and_row_independence():
    """Two sequences over the same pages, and a row alone against the row in a batch of the same sizes."""
    pool, batch, g = make("e4m3", 2, 64, [640], [64], 100)
    two = PagedBatch(pool, [batch.pages[0], batch.pages[0]], [640, 640], [64, 64])
    q = rows(64, 4, g)
    out = backend.attn_paged_batch(torch.cat([q, q]), two, block=1)
    same(out[:64], out[64:])
    check_paged(out[:64], q, pool, batch, "e4m3", 1)


def test_streams_do_not_share_scratch():
    """Two batches' attention at once on two streams, as often as it takes to overlap; each against its own result."""
    made = [make("e4m3", 2, 64, [6000 + 64 * i], [1 + 4 * i], 110 + i) for i in range(2)]
    qs = [rows(b.n_new, 8, g) for _, b, g in made]
    want = [backend.attn_paged_batch(q, b, block=1) for q, (_, b, _) in zip(qs, made)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in made]
    got = [[], []]
    for _ in range(20):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(backend.attn_paged_batch(qs[i], made[i][1], block=1))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_captured_decode_follows_the_device_lengths(fmt):
    """One captured step (append, attention, read-back) replayed while the lengths advance on the device."""
    pool, batch, g = make(fmt, 2, 64, [250, 70, 1], [1, 1, 1], 120)
    capacity = PagedBatch(pool, batch.pages, batch.kv_lens, [1, 1, 1], max_kv=256)
    k, v, q = rows(3, 2, g), rows(3, 2, g), rows(3, 8, g)

    def step():
        capacity.append(k, v)
        return backend.attn_paged_batch(q, capacity, block=1), *capacity.gather()

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        for t in (k, v, q):
            t.copy_(rows(3, t.shape[1], g))
        lens = [250 + i, 70 + i, 1 + i]
        capacity.kv_lens_dev.copy_(torch.tensor(lens, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        eager = PagedBatch(pool, batch.pages, lens, [1, 1, 1], max_kv=256)
        got = [o.clone() for o in outs]
        for x, y in zip(got, (backend.attn_paged_batch(q, eager, block=1), *eager.gather())):
            same(x, y)
        check_paged(got[0], q, pool, eager, fmt, 1)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_batched_step_as_it_is_used(fmt):
    """Prompts, then single tokens, then idle and active streams: append, attend, attend to each prompt's text."""
    page, hkv, heads = 64, 2, 4
    pool = POOLS[fmt](40, hkv, 128, page, DEV)
    pages = [list(range(0, 8)), list(range(8, 20)), list(range(20, 24))]
    text = [77, 0, 12]
    g = gen(130)
    tk, tv = rows(sum(text), hkv, g), rows(sum(text), hkv, g)
    kv = [0, 0, 0]
    hist = [[[], []] for _ in kv]
    batch = None
    for new in ([300, 129, 1], [1, 1, 1], [1, 0, 60], [0, 250, 2]):
        kv = [t + n for t, n in zip(kv, new)]
        if batch is None:
            batch = PagedBatch(pool, pages, kv, new)
        else:
            batch.set_lens(kv, new)
        n = sum(new)
        k, v, q = rows(n, hkv, g), rows(n, hkv, g), rows(n, heads, g)
        batch.append(k, v)
        x = backend.attn_paged_batch(q, batch, block=1)
        y = backend.attn_cross_batch(x, tk, tv, CrossBatch(new, text, DEV))
        at = c = 0
        for b, m in enumerate(new):
            for i, z in enumerate((k, v)):
                hist[b][i].append(z[at:at + m])
            if m:
                kk, vv = (ob.values(*ob.quantize(torch.cat(z), fmt), fmt) for z in hist[b])
                check(x[at:at + m], *ob.attend(q[at:at + m], kk, vv, [kv[b] - m + i + 1 for i in range(m)], SCALE))
                check(y[at:at + m], *ob.attend(x[at:at + m], tk[c:c + text[b]], tv[c:c + text[b]], [text[b]] * m, SCALE))
            at, c = at + m, c + text[b]


# ------------------------------------------------- sizes, scales and contents at the kernels' edges
EDGES = [15, 16, 17, 32, 33, 48, 63, 64, 65, 127, 128, 129, 255, 256, 257]


@pytest.mark.parametrize("group", [1, 3])
@pytest.mark.parametrize("fmt", ["e4m3", "int8", "dense"])
def test_row_counts_around_the_tiles(fmt, group):
    """Sequences whose rows fill, miss and pass a tile by one, with keys that do the same, and idle ones between."""
    for new in ([n] for n in EDGES if group == 1):
        run_edges(fmt, group, new, [new[0] + 1])
    run_edges(fmt, group, EDGES, [n + 64 - n % 64 + i % 3 - 1 for i, n in enumerate(EDGES)])
    run_edges(fmt, group, [0, 3, 70, 1] * 40, [64 + i % 3 for i in range(160)] if fmt == "dense" else [80 + i % 3 for i in range(160)])


def run_edges(fmt, group, new, kv):
    if fmt == "dense":
        g = gen(140)
        batch = CrossBatch(new, kv, DEV)
        q, k, v = rows(sum(new), 2 * group, g), rows(sum(kv), 2, g), rows(sum(kv), 2, g)
        out = backend.attn_cross_batch(q, k, v, batch)
        a = c = 0
        for i, j in zip(new, kv):
            check(out[a:a + i], *ob.attend(q[a:a + i], k[c:c + j], v[c:c + j], [j] * i, SCALE))
            a, c = a + i, c + j
        return
    kv = [max(t, n) for t, n in zip(kv, new)]
    pool, batch, g = make(fmt, 2, 48, kv, new, 141)
    q = rows(sum(new), 2 * group, g)
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, fmt, 1)


@pytest.mark.parametrize("page", [16, 64, 390])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [4, 150, 300])
def test_scales_of_v_that_grow_along_the_cache(fmt, new, page):
    """Scales of V from 2^-40 (and zero) up to 2^30 and back, changing inside and between the tiles: what was summed under
    a small scale keeps its place when a large one comes, and the other way round."""
    kv = [new + 700, new + 90]
    pool, batch, g = make(fmt, 2, page, kv, [new, new], 150)
    steps = [0, 0, -40, -38, -20, -20, -20, -3, 2, 2, 9, 9, 10, 30, 30, 29, 28, 28, 27, 26, 0, -10, 5, 5, 27, 31]
    for b, t in enumerate(kv):
        for p in range(t):
            e = steps[(p // 37 + 9 * b) % len(steps)]
            s = 0.0 if p < 20 and b == 0 else 2.0 ** e * 0.013
            pool.v_scales[batch.pages[b][p // page], :, p % page] = s
    q = rows(2 * new, 4, g)
    for block in (0, 1):
        check_paged(backend.attn_paged_batch(q, batch, block=block), q, pool, batch, fmt, block)


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("page", [7, 48, 64, 390])
@pytest.mark.parametrize("new", [2, 100])
def test_pages_that_are_none_read_as_zeros(fmt, page, new):
    """Table entries outside the pool, first, in the middle and last: their keys are zero and take part."""
    pool, batch, g = make(fmt, 2, page, [1000, 500], [new, new], 160)
    n = len(batch.pages[0])
    ks, vs = [], []
    gone = {0: -1, n // 2: pool.pool_pages, n - 1: 2 ** 30}
    for i, bad in gone.items():
        batch.tables[0, i] = bad
    for which, out in (("k", ks), ("v", vs)):
        x = cached(pool, batch, fmt, 0, which)
        for i in gone:
            x[i * page:(i + 1) * page] = 0
        out.append(x)
    q = rows(2 * new, 4, g)
    out = backend.attn_paged_batch(q, batch, block=1)
    check(out[:new], *ob.attend(q[:new], ks[0], vs[0], [1000 - new + i + 1 for i in range(new)], SCALE))
    check(out[new:], *ob.attend(q[new:], cached(pool, batch, fmt, 1, "k"), cached(pool, batch, fmt, 1, "v"),
                                [500 - new + i + 1 for i in range(new)], SCALE))


@pytest.mark.parametrize("new", [1, 9, 140])
def test_other_sequences_dense_keys_do_not_reach_a_row(new):
    lens = [63, 65, 130, 1]
    g = gen(170)
    batch = CrossBatch([new] * 4, lens, DEV)
    q, k, v = rows(4 * new, 4, g), rows(sum(lens), 2, g), rows(sum(lens) + 5, 2, g)[:sum(lens)]
    clean = backend.attn_cross_batch(q, k, v, batch)
    for bad in (float("nan"), float("inf")):
        for t in (k, v):
            save = t.clone()
            t[63:128] = bad
            out = backend.attn_cross_batch(q, k, v, batch)
            for b in (0, 2, 3):
                same(out[b * new:(b + 1) * new], clean[b * new:(b + 1) * new])
            assert not bool(torch.isfinite(out[new:2 * new]).any())
            t.copy_(save)


@pytest.mark.parametrize("new", [1, 9, 40, 140])
@pytest.mark.parametrize("fmt", ["e4m3", "int8", "dense"])
def test_queries_that_are_not_finite(fmt, new):
    """A row of q with a NaN or an infinity is NaN; the others are what they were."""
    if fmt == "dense":
        g = gen(180)
        batch = CrossBatch([new], [200], DEV)
        k, v = rows(200, 2, g), rows(200, 2, g)
        attend = lambda q: backend.attn_cross_batch(q, k, v, batch)
    else:
        _, batch, g = make(fmt, 2, 64, [200], [new], 181)
        attend = lambda q: backend.attn_paged_batch(q, batch, block=0)
    q = rows(new, 4, g)
    clean = attend(q)
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = q.clone()
        x[new // 2, 1, 77] = bad
        out = attend(x)
        assert bool(torch.isnan(out[new // 2, 1]).all())
        out[new // 2, 1] = clean[new // 2, 1]
        same(out, clean)


@pytest.mark.parametrize("new", [1, 20, 140])
@pytest.mark.parametrize("fmt", ["e4m3", "int8", "dense"])
def test_scores_that_rise_and_fall_along_the_keys(fmt, new):
    """The maximum moves from tile to tile, by little, by much (past what a weight can hold) and back."""
    rise = [0.0, 0.5, 0.1, 3.0, 3.2, 9.0, 1.0, 30.0, 30.0, 25.0, 60.0, 0.0, 61.0]
    t = 64 * len(rise) + 11
    g = gen(190)
    k = rows(t, 2, g, 0.1)
    q = rows(new, 4, g, 0.1)
    q[:, :, 0] = 1.0
    for i in range(t):
        k[i, :, 0] = rise[min(i // 64, len(rise) - 1)] / SCALE
    v = rows(t, 2, g)
    if fmt == "dense":
        out = backend.attn_cross_batch(q, k, v, CrossBatch([new], [t], DEV))
        check(out, *ob.attend(q, k, v, [t] * new, SCALE))
        return
    pool, _, _ = make(fmt, 2, 64, [t], [t], 191, spare=0, fill=False)
    whole = PagedBatch(pool, [list(range(pool.pool_pages))], [t], [t])
    whole.append(k, v)
    batch = PagedBatch(pool, whole.pages, [t], [new])
    check_paged(backend.attn_paged_batch(q, batch, block=1), q, pool, batch, fmt, 1)


@pytest.mark.parametrize("new", [3, 150])
def test_dense_rows_past_32_bit_offsets(new):
    """q, k, v and out as columns of tensors whose rows are 64 K elements apart: the last sequence's begin past 2^31."""
    n = 34000                                          # 34000 * 65536 = 2.2e9 elements
    wide = torch.empty((n, 65536), dtype=torch.bfloat16, device=DEV)
    cols = lambda c, heads: wide[:, 128 * c:128 * (c + heads)].view(n, heads, 128)
    q, k, v, out = cols(0, 4), cols(8, 2), cols(12, 2), cols(16, 4)
    lens = [n - 300, 300]
    news = [n - new, new]
    g = gen(200)
    tail = [slice(n - new, n), slice(n - 300, n)]
    q[tail[0]] = rows(new, 4, g)
    for t in (k, v):
        t[tail[1]] = rows(300, 2, g)
    batch = CrossBatch([0, new], lens, DEV)
    batch.cu_q.copy_(torch.tensor([n - new, n - new, n], dtype=torch.int32))   # the first rows are no sequence's
    batch.n_q = n
    backend.attn_cross_batch(q, k, v, batch, out=out)
    check(out[tail[0]], *ob.attend(q[tail[0]], k[tail[1]], v[tail[1]], [300] * new, SCALE))


def test_captured_chunks_follow_the_device_lengths():
    """Many rows over pages and over dense keys, captured once and replayed with other lengths, tables and contents."""
    pool, batch, g = make("e4m3", 2, 64, [700, 300], [150, 90], 210)
    cross = CrossBatch([150, 90], [100, 60], DEV)
    q, k, v = rows(240, 4, g), rows(160, 2, g), rows(160, 2, g)

    def step():
        x = backend.attn_paged_batch(q, batch, block=1)
        return x, backend.attn_cross_batch(x, k, v, cross)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for new, kv, text in (([150, 90], [700, 300], [100, 60]), ([240, 0], [500, 1], [1, 0]), ([7, 130], [7, 299], [160, 0])):
        q.copy_(rows(240, 4, g))
        batch.cu_new.copy_(torch.tensor([0, new[0], sum(new)], dtype=torch.int32))
        batch.kv_lens_dev.copy_(torch.tensor(kv, dtype=torch.int32))
        cross.cu_q.copy_(torch.tensor([0, new[0], sum(new)], dtype=torch.int32))
        cross.cu_kv.copy_(torch.tensor([0, text[0], sum(text)], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        x, y = (o.clone() for o in outs)
        eager = PagedBatch(pool, batch.pages, kv, new)
        check_paged(x[:sum(new)], q[:sum(new)], pool, eager, "e4m3", 1)
        a = c = 0
        for i, j in zip(new, text):
            check(y[a:a + i], *ob.attend(x[a:a + i], k[c:c + j], v[c:c + j], [j] * i, SCALE))
            a, c = a + i, c + j


@pytest.mark.parametrize("new", [1, 20, 140])
@pytest.mark.parametrize("fmt", ["e4m3", "int8", "dense"])
def test_a_scale_of_zero_is_the_mean(fmt, new):
    """softmax_scale 0 weighs every key a row sees alike, also in tiles that end behind the last one."""
    if fmt == "dense":
        g = gen(220)
        q, k, v = rows(new, 4, g), rows(70, 2, g), rows(70, 2, g)
        out = backend.attn_cross_batch(q, k, v, CrossBatch([new], [70], DEV), softmax_scale=0.0)
        check(out, *ob.attend(q, k, v, [70] * new, 0.0))
        return
    pool, batch, g = make(fmt, 2, 48, [new + 70], [new], 221)
    q = rows(new, 4, g)
    for block in (0, 1):
        check_paged(backend.attn_paged_batch(q, batch, block=block, softmax_scale=0.0), q, pool, batch, fmt, block, scale=0.0)
