"""Batched sequences, host side: descriptors, refusals and their messages (no GPU)."""

import pytest
import torch

from oracle import batch as ob
from waveforcing_amd import _lib, backend
from waveforcing_amd.kv import CrossBatch, Fp8PagePool, Int8PagePool, PagedBatch, PagedKV


def pool(cls=Fp8PagePool, pages=6, heads=2, page=16):
    return cls(pages, heads, 128, page, "cpu")


def test_descriptor_arrays():
    b = PagedBatch(pool(), [[4, 1], [], [3]], [20, 0, 16], [3, 0, 16])
    assert b.cu_new.tolist() == [0, 3, 3, 19] and b.kv_lens_dev.tolist() == [20, 0, 16]
    assert b.tables.tolist() == [[4, 1], [-1, -1], [3, -1]]
    assert (b.n_new, b.max_new, b.max_kv) == (19, 16, 20)
    b.set_lens([21, 0, 16], [1, 0, 0], max_kv=32)
    assert b.cu_new.tolist() == [0, 1, 1, 1] and b.kv_lens_dev.tolist() == [21, 0, 16] and b.max_kv == 32
    assert PagedBatch(pool(), [[0], [1]], [5, 6]).new_lens == [1, 1]
    c = CrossBatch([2, 0, 3], [7, 1, 0], "cpu")
    assert c.cu_q.tolist() == [0, 2, 2, 5] and c.cu_kv.tolist() == [0, 7, 8, 8] and (c.max_q, c.max_kv) == (3, 7)


@pytest.mark.parametrize("pages, kv, new, error, text", [
    ([[6]], [1], [1], RuntimeError, "outside pool"),
    ([[-1]], [1], [1], ValueError, "page id"),
    ([[0]], [17], [1], RuntimeError, "cannot hold 17"),
    ([[0]], [3], [4], ValueError, "4 new rows among 3"),
    ([[0]], [-1], [0], ValueError, "kv_lens"),
    ([[0]], [1], [-1], ValueError, "new_lens"),
    ([[0], [1]], [1], [1], ValueError, "2 page lists, 1 kv_lens"),
    ([[0]], [1, 2], None, ValueError, "1 page lists, 2 kv_lens"),
])
def test_descriptor_refusals(pages, kv, new, error, text):
    with pytest.raises(error, match=text):
        PagedBatch(pool(), pages, kv, new)


def test_bounds_and_cross_refusals():
    with pytest.raises(ValueError, match="max_kv=4 is below"):
        PagedBatch(pool(), [[0]], [5], max_kv=4)
    b = PagedBatch(pool(), [[0]], [5])
    with pytest.raises(RuntimeError, match="cannot hold 17"):
        b.set_lens([17])
    with pytest.raises(ValueError, match="1 q_lens and 2 kv_lens"):
        CrossBatch([1], [1, 2], "cpu")
    with pytest.raises(ValueError, match="kv_lens holds -3"):
        CrossBatch([1], [-3], "cpu")


def test_rows_written_twice_are_refused():
    x = torch.zeros((2, 2, 128), dtype=torch.bfloat16)
    for pages, kv, new in (([[0], [0]], [1, 2], [1, 1]),          # two sequences write one page
                           ([[0, 1], [2, 1]], [20, 20], [1, 0]),  # one writes what the other reads
                           ([[3, 3]], [20], [2])):                # one page twice in a sequence
        with pytest.raises(RuntimeError, match="would be written but is used 2 times"):
            PagedBatch(pool(), pages, kv, new).append(x, x)


def test_tensor_refusals():
    b = PagedBatch(pool(), [[0]], [5], [3])
    x = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="has 2 rows, the batch 3"):
        b.append(x[:2], None)
    with pytest.raises(ValueError, match="heads/dim"):
        b.append(x[:, :1], None)
    with pytest.raises(ValueError, match="bfloat16"):
        b.append(x.float(), None)
    with pytest.raises(ValueError, match="dense heads"):
        b.gather(out_k=torch.zeros((3, 2, 256), dtype=torch.bfloat16)[..., ::2])
    with pytest.raises(ValueError, match="query heads"):
        backend.attn_paged_batch(torch.zeros((3, 3, 128), dtype=torch.bfloat16), b)
    with pytest.raises(ValueError, match="q has 2 rows"):
        backend.attn_paged_batch(x[:2], b)
    with pytest.raises(ValueError, match="q must be bf16"):
        backend.attn_paged_batch(x.half(), b)
    with pytest.raises(ValueError, match="block=-1"):
        backend.attn_paged_batch(x, b, block=-1)
    with pytest.raises(ValueError, match="out must be"):
        backend.attn_paged_batch(x, b, out=torch.zeros((2, 2, 128), dtype=torch.bfloat16))
    with pytest.raises(TypeError, match="PagedBatch"):
        backend.attn_paged_batch(x, None)
    c = CrossBatch([3], [4], "cpu")
    k = torch.zeros((4, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="hold the batch's 4 rows"):
        backend.attn_cross_batch(x, k[:3], k[:3], c)
    with pytest.raises(ValueError, match="must match"):
        backend.attn_cross_batch(x, k, k[:, :1], c)
    with pytest.raises(ValueError, match="do not group"):
        backend.attn_cross_batch(torch.zeros((3, 3, 128), dtype=torch.bfloat16), k, k, c)
    with pytest.raises(TypeError, match="CrossBatch"):
        backend.attn_cross_batch(x, k, k, b)


def test_int8_pages_are_refused_by_the_one_sequence_forms():
    p = pool(Int8PagePool)
    x = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    for call in (lambda: p.pack(x, x, p.page_table([0])), lambda: p.unpack(p.page_table([0]), 3),
                 lambda: p.pack_k_norm_rope(x.view(3, 256), None, p.page_table([0]), x[0, 0], 1e-6, None)):
        with pytest.raises(TypeError, match="PagedBatch"):
            call()
    with pytest.raises(TypeError, match="e4m3 pages"):
        backend.attn_paged_fp8(x, PagedKV(p, p.page_table([0]), 3))


# every entry point's checks come before it touches the device
APPEND = dict(k=16, v=32, rows=4, heads=2, dim=128, ld=256, fmt=0, cu=48, lens=64, seqs=1, tab=80, ldt=1, page=16, kc=96,
              vc=112, ks=128, vs=144, pages=4, stream=None)
PAGED = dict(q=16, rows=4, heads=4, kv_heads=2, dim=128, ldq=512, fmt=0, kc=32, vc=48, ks=64, vs=80, pages=4, page=16, cu=96,
             lens=112, seqs=1, tab=128, ldt=1, max_new=4, max_kv=16, block=0, scale=0.1, out=144, ldo=512, ws=None, wsb=0,
             stream=None)
CROSS = dict(q=16, rows=4, heads=4, kv_heads=2, dim=128, ldq=512, k=32, v=48, kv_rows=8, ldkv=256, cu_q=64, cu_kv=80, seqs=1,
             max_q=4, max_kv=8, scale=0.1, out=96, ldo=512, ws=None, wsb=0, stream=None)


@pytest.mark.parametrize("entry, args, change, text", [
    ("wf_kv_batch_append", APPEND, dict(dim=64), "head_dim=64"),
    ("wf_kv_batch_append", APPEND, dict(rows=-1), "negative"),
    ("wf_kv_batch_append", APPEND, dict(fmt=2), "unknown cache format 2"),
    ("wf_kv_batch_append", APPEND, dict(page=0), "page_tokens=0"),
    ("wf_kv_batch_append", APPEND, dict(ld=248), "row stride 248"),
    ("wf_kv_batch_append", APPEND, dict(ld=260), "row stride 260"),
    ("wf_kv_batch_append", APPEND, dict(k=18), "16-byte aligned"),
    ("wf_kv_batch_append", APPEND, dict(k=None), "null K"),
    ("wf_kv_batch_append", APPEND, dict(vc=None), "V given without V pool"),
    ("wf_kv_batch_append", APPEND, dict(cu=None), "null row starts"),
    ("wf_kv_batch_append", APPEND, dict(tab=None), "null page tables"),
    ("wf_kv_batch_append", APPEND, dict(rows=1 << 31), "reaches 2"),
    ("wf_kv_batch_append", APPEND, dict(pages=1 << 30), "rows or more"),
    ("wf_attn_paged_batch", PAGED, dict(heads=3), "do not group"),
    ("wf_attn_paged_batch", PAGED, dict(kv_heads=0), "negative or zero"),
    ("wf_attn_paged_batch", PAGED, dict(dim=64), "head_dim=64"),
    ("wf_attn_paged_batch", PAGED, dict(block=-1), "block=-1"),
    ("wf_attn_paged_batch", PAGED, dict(scale=float("nan")), "softmax_scale"),
    ("wf_attn_paged_batch", PAGED, dict(scale=-1.0), "softmax_scale"),
    ("wf_attn_paged_batch", PAGED, dict(ldq=504), "ldq/ldo"),
    ("wf_attn_paged_batch", PAGED, dict(q=24), "16-byte"),
    ("wf_attn_paged_batch", PAGED, dict(ks=None), "null pointer"),
    ("wf_attn_paged_batch", PAGED, dict(max_kv=-1), "bad bound"),
    ("wf_attn_paged_batch", PAGED, dict(rows=1 << 30), "reaches 2"),
    ("wf_attn_cross_batch", CROSS, dict(kv_rows=-1), "key rows"),
    ("wf_attn_cross_batch", CROSS, dict(ldkv=128), "ldkv=128"),
    ("wf_attn_cross_batch", CROSS, dict(k=40), "16-byte"),
    ("wf_attn_cross_batch", CROSS, dict(v=None), "null pointer"),
])
def test_entry_point_refusals(entry, args, change, text):
    with pytest.raises(RuntimeError, match=text):
        _lib.call(entry, *{**args, **change}.values())


def test_empty_calls_return():
    _lib.call("wf_kv_batch_append", *{**APPEND, "rows": 0, "k": None, "cu": None}.values())
    _lib.call("wf_attn_paged_batch", *{**PAGED, "rows": 0}.values())
    _lib.call("wf_attn_cross_batch", *{**CROSS, "seqs": 0}.values())


def test_oracle_positions_and_limits():
    assert ob.row_positions([5, 0, 2], [2, 0, 2]) == [(0, 3), (0, 4), (2, 0), (2, 1)]
    assert [ob.limit(p, 10, 4) for p in (0, 3, 4, 9)] == [4, 4, 8, 10]
    assert [ob.limit(p, 10, 0) for p in (0, 9)] == [10, 10] and ob.limit(6, 10, 1) == 7


@pytest.mark.parametrize("fmt, half", [("int8", 0.5 / 127), ("e4m3", 2.0 ** -4)])
def test_oracle_quantization_is_half_a_step(fmt, half):
    x = torch.randn((50, 3, 128), generator=torch.Generator().manual_seed(1)).bfloat16()
    c, s = ob.quantize(x, fmt)
    err = (ob.values(c, s, fmt) - x.double()).abs()
    # int8: half a step of the row's maximum; e4m3: 2^-4 of the value, or half the smallest step 2^-9 s; the e4m3
    # scale is itself rounded to bf16 (2^-8), which clips the maximum by at most that
    # int8's quotient is rounded to fp32 first (at most 127 2^-24 of a step) and its scale too (2^-24 of it): half a step
    # times 1 + 254 2^-24 + 2 2^-24 < 1 + 2^-15
    top = x.double().abs().amax(-1, keepdim=True)
    lim = half * top * (1 + 2.0 ** -15) if fmt == "int8" else (half + 2.0 ** -8) * x.double().abs() + s.double()[..., None] * 2.0 ** -10
    assert bool((err <= lim).all())


def workspace(*sizes):
    import ctypes

    n = ctypes.c_int64(-1)
    _lib.call("wf_attn_batch_workspace", *sizes, ctypes.addressof(n))
    return n.value


def test_workspace_query():
    """No scratch where nothing is split; a single long sequence takes some, of whole (row, split) records."""
    assert workspace(0, 8, 8, 0, 0, 0) == 0 and workspace(64, 8, 8, 64, 1, 100) == 0
    one = workspace(1, 12, 12, 1, 1, 30000)
    assert one > 0 and one % (130 * 4) == 0
    for sizes in ((1 << 62, 1, 1, 1, 1, 1), (1 << 20, 1 << 20, 1, 1, 1, 1), (1, 1, 1, 1 << 40, 1, 1), (1, 1, 1, 1, 1, 1 << 40)):
        with pytest.raises(RuntimeError, match="2\\^31"):
            workspace(*sizes)
    assert workspace(1, 1, 1, 1, 1 << 62, 1) == 0    # a bound of the rows past the rows is the rows
    for sizes in ((-1, 1, 1, 1, 1, 1), (1, 0, 1, 1, 1, 1), (1, 1, 1, -1, 1, 1), (1, 1, 1, 1, 1, -1)):
        with pytest.raises(RuntimeError, match="negative or zero"):
            workspace(*sizes)
    with pytest.raises(RuntimeError, match="group"):
        workspace(1, 3, 2, 1, 1, 1)


def test_one_long_sequence_does_not_split_the_many_short_ones_finely():
    """The pieces of a sequence shrink in number as the other sequences' surplus ones grow."""
    record = 16 * 130 * 4 * 8                          # a split of a tile of 16 rows of each of 8 key heads
    pieces = [workspace(n, 40, 8, n, 1, 131072) // record // (n * 5 // 16 + n) for n in (1, 64, 256, 1024)]
    assert pieces == sorted(pieces, reverse=True) and pieces[0] == 64 and 1 < pieces[-1] <= 8
    with pytest.raises(RuntimeError, match="too many"):   # a grid of 2^32 threads
        _lib.call("wf_attn_cross_batch", 16, 1 << 19, 512, 512, 128, 512 * 128, 16, 16, 1, 512 * 128, 16, 16, 1 << 19, 1, 1,
                  1.0, 16, 512 * 128, 16, 1 << 40, None)
