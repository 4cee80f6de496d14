"""Batched attention where values, lengths and bounds are far from the ordinary: the contract's edges, on the GPU, against
64 bits (oracle/batch.py)."""

import pytest
import torch

from oracle import batch as ob
from test_gpu_batch import DEV, SCALE, cached, check, gen, make, rows, same
from waveforcing_amd import _lib, backend
from waveforcing_amd.kv import CrossBatch, Fp8PagePool, PagedBatch

pytestmark = pytest.mark.gpu


def attend_quietly(q, k, v, loud, limits):
    """The exact output, and the bound that it has without the loud keys' values: their weights are below 2^-100 here, so
    neither they nor their roundings reach a result."""
    ref, _ = ob.attend(q, k, v, limits, SCALE)
    quiet = v.clone()
    quiet[loud] = 0
    return ref, ob.attend(q, k, quiet, limits, SCALE)[1]


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("ratio", [18, 22, 26, 40, 70])
@pytest.mark.parametrize("new", [9, 100, 300])
def test_quiet_values_among_loud_ones_keep_their_bits(fmt, ratio, new):
    """Rows whose weight is on keys with V 2^ratio below that of other keys of the same tile."""
    t = new + 150
    pool, batch, g = make(fmt, 2, 48, [t], [new], 300)
    at = torch.arange(t, device=DEV)
    loud = at % 5 == 3
    page = torch.tensor(batch.pages[0], device=DEV)[at // 48]
    k = rows(t, 2, g, 0.1)
    k[:, :, 0] = torch.where(loud, -400.0, 400.0)[:, None].bfloat16()   # scores of both kinds 2^150 apart in weight
    pool.k_codes[page, at % 48], pool.k_scales[page, :, at % 48] = ob.quantize(k, fmt)
    pool.v_scales[page, :, at % 48] *= torch.where(loud, 2.0 ** 14, 2.0 ** (14 - ratio))[:, None]
    q = rows(new, 4, g, 0.1)
    q[:, :, 0] = 1.5
    k, v = (cached(pool, batch, fmt, 0, name) for name in "kv")
    for block in (0, 1):
        limits = [ob.limit(t - new + i, t, block) for i in range(new)]
        check(backend.attn_paged_batch(q, batch, block=block), *attend_quietly(q, k, v, loud, limits))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [9, 100, 300])
def test_hidden_values_do_not_move_a_bit(fmt, new):
    """Finite values behind a row's limit, 2^10 to 2^100 above those it sees."""
    pool, batch, g = make(fmt, 2, 64, [new + 37], [new], 310)
    q = rows(new, 4, g)
    clean = backend.attn_paged_batch(q, batch, block=1)
    p = new + 36
    page, at = batch.pages[0][p // 64], p % 64
    for e in (10, 30, 100):
        pool.v_scales[page, :, at] = 2.0 ** e
        pool.k_scales[page, :, at] = 2.0
        out = backend.attn_paged_batch(q, batch, block=1)
        same(out[:-1], clean[:-1])


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [9, 100])
@pytest.mark.parametrize("scale", [1e-8, 2.0 ** -60, 2.0 ** 40])
def test_values_behind_a_tile_of_zeros(fmt, new, scale):
    """The first keys' pages are none (zero K and V); the others' scales of V are small, or large."""
    t = 128 + new + 20
    pool, batch, g = make(fmt, 2, 64, [t], [new], 320)
    batch.tables[0, :2] = -1
    pool.v_scales.copy_(scale * (1 + torch.rand(pool.v_scales.shape, generator=g, device=DEV)).bfloat16())
    q = rows(new, 4, g)
    k, v = (cached(pool, batch, fmt, 0, name) for name in "kv")
    k[:128], v[:128] = 0, 0
    limits = [t - new + i + 1 for i in range(new)]
    check(backend.attn_paged_batch(q, batch, block=1), *ob.attend(q, k, v, limits, SCALE))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new, t", [(9, 300), (100, 300), (100, 9001)])
@pytest.mark.parametrize("first, then", [(-75, 60), (60, -75), (-70, 100), (0, -126)])
def test_keys_of_any_scale_count_alike(fmt, new, t, first, then):
    """Equal scores: every seen key counts once, whatever its scale of V, and a negative one turns its value's sign."""
    pool, batch, g = make(fmt, 2, 64, [t], [new], 380)
    at = torch.arange(t, device=DEV)
    page = torch.tensor(batch.pages[0], device=DEV)[at // 64]
    e = torch.where(at < t // 2, 2.0 ** first, 2.0 ** then) * torch.where(at % 7 == 2, -0.01, 0.01)
    pool.v_scales[page, :, at % 64] = e[:, None]
    q = torch.zeros((new, 4, 128), dtype=torch.bfloat16, device=DEV)
    k, v = (cached(pool, batch, fmt, 0, name) for name in "kv")
    check(backend.attn_paged_batch(q, batch, block=1), *ob.attend(q, k, v, [t - new + i + 1 for i in range(new)], SCALE))


@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
@pytest.mark.parametrize("new", [1, 20, 140])
@pytest.mark.parametrize("fmt", ["e4m3", "int8", "dense"])
def test_infinite_queries_over_one_key(fmt, new, bad):
    """A row of q that holds an infinity is NaN, also where its every score is -inf."""
    g = gen(330)
    k = torch.zeros((new, 2, 128), dtype=torch.bfloat16, device=DEV)
    k[:, :, 3] = 1.0
    v, q = rows(new, 2, g), rows(new, 4, g)
    if fmt == "dense":
        batch = CrossBatch([new], [1], DEV)
        attend = lambda x: backend.attn_cross_batch(x, k[:1], v[:1], batch)
    else:
        pool, batch, _ = make(fmt, 2, 64, [new], [new], 331)
        batch.append(k, v)
        attend = lambda x: backend.attn_paged_batch(x, batch, block=1)
    clean = attend(q)
    for i in {0, new // 2, new - 1}:
        x = q.clone()
        x[i, 1, 3] = bad
        out = attend(x)
        assert bool(torch.isnan(out[i, 1]).all())
        out[i, 1] = clean[i, 1]
        same(out, clean)


@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("new", [1, 20, 140])
@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_a_scale_that_is_not_finite_makes_the_rows_that_see_it_nan(fmt, new, bad, which):
    """Whatever the sign of the score that an infinite scale of K gives; the rows before it keep their bits."""
    pool, batch, g = make(fmt, 2, 64, [new + 90], [new], 340)
    q = rows(new, 4, g)
    clean = backend.attn_paged_batch(q, batch, block=1)
    for p in (new + 89, 90 + new // 2, 5):
        scales = getattr(pool, which + "_scales")
        page, at = batch.pages[0][p // 64], p % 64
        save = scales[page, :, at].clone()
        scales[page, :, at] = bad
        out = backend.attn_paged_batch(q, batch, block=1)
        sees = torch.arange(90, 90 + new, device=DEV) >= p
        assert bool(torch.isnan(out[sees]).all())
        same(out[~sees], clean[~sees])
        scales[page, :, at] = save


@pytest.mark.parametrize("new", [1, 140])
def test_dense_scores_of_minus_infinity(new):
    """exp(-inf) is 0 where another key is finite, and a row all of whose scores are -inf has no mean."""
    g = gen(350)
    q, k, v = rows(new, 4, g).abs() + 0.1, rows(70, 2, g), rows(70, 2, g)
    batch = CrossBatch([new], [70], DEV)
    k[3, :, 9] = -float("inf")
    keep = [i for i in range(70) if i != 3]
    out = backend.attn_cross_batch(q, k, v, batch)
    check(out, *ob.attend(q, k[keep], v[keep], [69] * new, SCALE))
    k[:, :, 9] = -float("inf")
    assert bool(torch.isnan(backend.attn_cross_batch(q, k, v, batch)).all())


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
@pytest.mark.parametrize("new", [6, 150])
def test_rows_past_the_tensors_keep_the_others_in_place(fmt, new):
    """Device lengths that pass the tensors' rows: append, read-back and attention place the rows that there are alike."""
    pool, batch, g = make(fmt, 2, 48, [40, 2 * new + 100], [3, new], 360)
    batch.cu_new[2] = 3 + 2 * new                      # twice the rows of q, k and v
    k, v, q = rows(3 + new, 2, g), rows(3 + new, 2, g), rows(3 + new, 4, g)
    batch.append(k, v)
    gk, gv = batch.gather()
    for x, y in ((k, gk), (v, gv)):
        same(y, ob.values(*ob.quantize(x, fmt), fmt).float().bfloat16())
    first = 100                                        # position of the second sequence's first row
    page = torch.tensor(batch.pages[1], device=DEV)[torch.arange(first, first + new, device=DEV) // 48]
    at = torch.arange(first, first + new, device=DEV) % 48
    same(pool.k_codes[page, at], ob.quantize(k[3:], fmt)[0])
    for block in (1, 16):
        out = backend.attn_paged_batch(q, batch, block=block)
        t = 2 * new + 100
        check(out[3:], *ob.attend(q[3:], cached(pool, batch, fmt, 1, "k"), cached(pool, batch, fmt, 1, "v"),
                                  [ob.limit(first + i, t, block) for i in range(new)], SCALE))


@pytest.mark.parametrize("fmt", ["e4m3", "int8"])
def test_rows_before_the_first_sequence_are_nobodys(fmt):
    """A first start behind row 0: the rows before it are neither cached (where older positions lie) nor read back."""
    pool, batch, g = make(fmt, 2, 16, [30], [8], 370)
    codes, scales = pool.k_codes.clone(), pool.k_scales.clone()
    batch.cu_new[0] = 5
    k = rows(8, 2, g)
    batch.append(k, k)
    for p in range(27):                                # 27 .. 29 are the three rows'
        page, at = batch.pages[0][p // 16], p % 16
        same(pool.k_codes[page, at], codes[page, at])
        same(pool.k_scales[page, :, at], scales[page, :, at])
    out = torch.full((8, 2, 128), 7.0, dtype=torch.bfloat16, device=DEV)
    batch.gather(with_v=False, out_k=out)
    assert bool((out[:5] == 7).all())
    same(out[5:], ob.values(*ob.quantize(k[5:], fmt), fmt).float().bfloat16())


def spoil(*shapes):
    """Leaves NaN in the memory that the next new tensors of these shapes take."""
    held = [torch.full(s, float("nan"), dtype=torch.bfloat16, device=DEV) for s in shapes]
    del held


@pytest.mark.parametrize("fmt", ["e4m3", "int8", "dense"])
@pytest.mark.parametrize("new, hkv", [(1, 2), (9, 2), (40, 3), (700, 1)])
def test_rows_that_the_device_leaves_out_are_zero_in_a_new_output(fmt, new, hkv):
    """Starts on the device that own fewer rows than the tensors have, before, between (none) and behind the sequences."""
    n, heads = 3 * new, 2 * hkv
    g = gen(390)
    q = rows(n + 2, heads, g)                          # two rows behind the batch's
    if fmt == "dense":
        batch = CrossBatch([new] * 3, [50, 0, 33], DEV)
        k, v = rows(83, hkv, g), rows(83, hkv, g)
        starts, attend = batch.cu_q, lambda **kw: backend.attn_cross_batch(q, k, v, batch, **kw)
    else:
        pool, batch, _ = make(fmt, hkv, 48, [new + 60, new, new + 300], [new] * 3, 391)
        starts, attend = batch.cu_new, lambda **kw: backend.attn_paged_batch(q, batch, block=1, **kw)
    whole = attend()
    assert bool((whole[n:] == 0).all()) and bool((whole[:new] != 0).any())
    for first, last in ((0, n), (0, n - 1), (0, new), (1, n), (new // 2, new), (0, 0), (n, n)):
        starts.copy_(torch.tensor([first, max(first, min(new, last)), max(first, min(2 * new, last)), last], dtype=torch.int32))
        owned = torch.arange(n + 2, device=DEV)
        owned = (owned >= first) & (owned < last)
        spoil((n + 2, heads, 128))
        out = attend()
        assert bool(torch.isfinite(out).all()) and bool((out[~owned] == 0).all())
        given = torch.full_like(out, 7.0)
        same(attend(out=given)[owned], out[owned])
        assert bool((given[~owned] == 7).all())
        if fmt != "dense":
            spoil((n, hkv, 128), (n, hkv, 128))
            gk, gv = batch.gather()
            assert bool((gk[~owned[:n]] == 0).all()) and bool((gv[~owned[:n]] == 0).all())
            half = torch.full_like(gk, 7.0)
            spoil((n, hkv, 128))
            _, other = batch.gather(out_k=half)
            same(other, gv)
            assert bool((half[~owned[:n]] == 7).all())
            same(half[owned[:n]], gk[owned[:n]])


@pytest.mark.parametrize("new", [8, 200])
def test_replays_with_fewer_rows_hold_none_of_the_rows_before(new):
    pool, batch, g = make("int8", 2, 64, [new + 300, new + 10], [new, new], 400)
    cross = CrossBatch([new, new], [70, 20], DEV)
    q, k, v = rows(2 * new, 4, g), rows(90, 2, g), rows(90, 2, g)

    def step():
        x = backend.attn_paged_batch(q, batch, block=1)
        return (x, backend.attn_cross_batch(q, k, v, cross), *batch.gather())

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for a, b in ((new, new), (new, 1), (2, 0), (0, 5), (new, new)):
        for t in (batch.cu_new, cross.cu_q):
            t.copy_(torch.tensor([0, a, a + b], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        for x, y in zip(outs, want):
            assert bool((x[a + b:] == 0).all())
            same(x, y)


def test_a_new_output_without_sequences_is_refused_at_the_entry():
    x = torch.zeros((4, 2, 128), dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="rows without a sequence"):
        _lib.call("wf_attn_cross_batch_fresh", x.data_ptr(), 4, 2, 2, 128, 256, x.data_ptr(), x.data_ptr(), 4, 256, None, None, 0, 4,
                  4, 1.0, x.data_ptr(), 256, None, 0, None)
    assert PagedBatch(Fp8PagePool(1, 2, 128, 16, DEV), [], []).gather()[0].shape == (0, 2, 128)


@pytest.mark.parametrize("new", [2, 100])
@pytest.mark.parametrize("shift", [1, 4])
def test_dense_rows_at_any_address(new, shift):
    """Contiguous rows that begin in the middle of a 16-byte word are copied, not refused."""
    g = gen(410)

    def at_shift(x):
        flat = torch.empty(x.numel() + shift, dtype=x.dtype, device=DEV)
        y = flat[shift:].view(x.shape)
        y.copy_(x)
        assert y.data_ptr() % 16 and y.is_contiguous()
        return y

    pool, batch, _ = make("int8", 2, 16, [new + 30], [new], 411)
    other, same_pages, _ = make("int8", 2, 16, [new + 30], [new], 411)
    q, k, v = rows(new, 4, g), rows(new, 2, g), rows(new, 2, g)
    batch.append(k, v)
    same_pages.append(at_shift(k), at_shift(v))
    same(pool.k_codes, other.k_codes)
    same(pool.v_scales, other.v_scales)
    same(backend.attn_paged_batch(at_shift(q), batch, block=1), backend.attn_paged_batch(q, batch, block=1))
    cross = CrossBatch([new], [new], DEV)
    same(backend.attn_cross_batch(at_shift(q), at_shift(k), v, cross), backend.attn_cross_batch(q, k, v, cross))
