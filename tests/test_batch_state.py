"""Batched sequences, host side: what a batch keeps over refused calls and new lengths (no GPU)."""

import ctypes

import pytest
import torch

from waveforcing_amd import _lib, backend
from waveforcing_amd.kv import CrossBatch, Fp8PagePool, Int8PagePool, PagedBatch


def pool(cls=Fp8PagePool):
    return cls(6, 2, 128, 16, "cpu")


def state(b):
    return (b.kv_lens, b.new_lens, b.n_new, b.max_new, b.max_kv, b.cu_new.tolist(), b.kv_lens_dev.tolist(),
            b.tables.tolist())


@pytest.mark.parametrize("kv, new, most, error", [
    ([20, 9], [9, 1], 4, ValueError),                       # a bound below the lengths
    ([20, 9], [9], None, ValueError),                       # one length short
    ([33, 9], [9, 1], None, RuntimeError),                  # past the pages
    ([20, 9], [21, 1], None, ValueError),                   # more new rows than positions
    ([20, -1], [9, 1], None, ValueError),
    ([20, 9], [9, (1 << 31) - 1024], None, ValueError),
    ([20, "x"], [9, 1], None, ValueError),
])
def test_refused_lengths_leave_the_batch_as_it_was(kv, new, most, error):
    b = PagedBatch(pool(), [[4, 1], [3]], [5, 7], [1, 2], max_kv=40)
    before = state(b)
    with pytest.raises(error):
        b.set_lens(kv, new, max_kv=most)
    assert state(b) == before
    b.set_lens([20, 9], [9, 1], max_kv=32)
    assert state(b) == ([20, 9], [9, 1], 10, 9, 32, [0, 9, 10], [20, 9], [[4, 1], [3, -1]])


def test_a_given_bound_stays():
    b = PagedBatch(pool(), [[4, 1], [3]], [5, 7], max_kv=32)
    b.set_lens([6, 8])
    assert b.max_kv == 32
    b.set_lens([7, 9], max_kv=20)
    assert b.max_kv == 20
    b.set_lens([25, 9])                                     # past the bound
    assert b.max_kv == 25
    b.set_lens([8, 10])
    assert b.max_kv == 20
    b = PagedBatch(pool(), [[4, 1], [3]], [5, 7])           # none given: the longest
    b.set_lens([9, 8])
    assert b.max_kv == 9
    b.set_lens([1, 8])
    assert b.max_kv == 8
    assert PagedBatch(pool(), [], []).max_kv == 0


def test_a_view_reads_pages_in_their_own_format():
    for cls, other in ((Fp8PagePool, Int8PagePool), (Int8PagePool, Fp8PagePool)):
        p = pool(cls)
        view = cls.view_of(p, 2, 3)
        assert (view.format, view.pool_pages) == (p.format, 3) and view.k_codes.data_ptr() == p.k_codes[2].data_ptr()
        with pytest.raises(TypeError, match="another code format"):
            other.view_of(p, 2, 3)


def workspace(*sizes):
    n = ctypes.c_int64(-1)
    _lib.call("wf_attn_batch_workspace", *sizes, ctypes.addressof(n))
    return n.value


def test_workspace_of_sizes_that_no_call_takes_is_refused():
    """Sizes whose product passes 64 bits: refused as the attention refuses them, not wrapped around."""
    most = (1 << 31) - 1
    for sizes in ((1, 1 << 30, 1 << 30, most, 1, most), (1, 1 << 20, 1 << 20, 1 << 20, 1, 1 << 30),
                  (1 << 15, 1 << 15, 1 << 15, 1 << 19, 1, most)):
        with pytest.raises(RuntimeError, match="too many"):
            workspace(*sizes)
    assert workspace(0, most, most, most, 1, most) == 0     # no rows: a call that returns at once


@pytest.mark.parametrize("scale", [2.5e38, 2.9e38, float("inf")])
def test_a_scale_that_overflows_in_base_2_is_refused(scale):
    args = (16, 4, 4, 2, 128, 512, 32, 48, 8, 256, 64, 80, 1, 4, 8, scale, 96, 512, None, 0, None)
    with pytest.raises(RuntimeError, match="softmax_scale"):
        _lib.call("wf_attn_cross_batch", *args)


@pytest.mark.parametrize("heads", [1 << 16, 1 << 24, 1 << 25])
def test_rows_of_heads_past_32_bit_offsets_are_refused(heads):
    """Elements are placed in a row by 32-bit numbers; the entry points take fewer heads than would pass them."""
    ld = 128 * heads
    with pytest.raises(RuntimeError, match="2\\^16 or more"):
        _lib.call("wf_kv_batch_append", 16, 32, 1, heads, 128, ld, 0, 48, 64, 1, 80, 1, 1, 96, 112, 128, 144, 1, None)
    with pytest.raises(RuntimeError, match="2\\^16 or more"):
        _lib.call("wf_kv_batch_gather", 96, 112, 128, 144, 1, 0, 1, 48, 64, 1, 80, 1, 1, heads, 128, 16, 32, ld, None)
    if heads >= 1 << 24:
        with pytest.raises(RuntimeError, match="2\\^24 or more"):
            _lib.call("wf_attn_cross_batch", 16, 1, heads, 1, 128, ld, 32, 48, 8, 256, 64, 80, 1, 1, 8, 0.1, 96, ld, None, 0, None)


def test_tensors_on_the_cpu_are_refused_by_name():
    b, c = PagedBatch(pool(), [[0]], [5], [3]), CrossBatch([3], [3], "cpu")
    x = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    for name, run in (("wf_kv_batch_append", lambda: b.append(x, x)), ("wf_kv_batch_gather", lambda: b.gather()),
                      ("wf_attn_paged_batch", lambda: backend.attn_paged_batch(x, b)),
                      ("wf_attn_cross_batch", lambda: backend.attn_cross_batch(x, x, x, c))):
        with pytest.raises(ValueError, match=f"{name}.*on cpu"):
            run()
