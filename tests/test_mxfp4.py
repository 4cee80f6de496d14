"""MXFP4 rows, linears and pages on the host: the definition's properties, layouts, and every refusal (no GPU)."""

import pytest
import torch
import torch.nn as nn

from oracle import mxfp4 as om
from waveforcing_amd import _lib, mxfp4


def every_bf16():
    return torch.arange(65536, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)


def test_oracle_scale_is_the_smallest_power_of_two_and_no_value_is_far():
    x = every_bf16()
    x = x[torch.isfinite(x)]
    block = torch.zeros((len(x), 32), dtype=torch.bfloat16)
    block[:, 5] = x
    codes, scales = om.quantize(block)
    s = torch.exp2(scales[:, 0].double() - 127)
    a = x.double().abs()
    free = (scales[:, 0] > 2) & (scales[:, 0] < 252)
    assert bool((a < 7 * s)[scales[:, 0] < 252].all()) and bool((a >= 3.5 * s)[free].all())
    v = om.values(codes, scales)[:, 5]
    step = torch.where(a < 2 * s, 0.5, torch.where(a < 4 * s, 1.0, 2.0)) * s
    assert bool(((v - x.double()).abs() <= step / 2)[scales[:, 0] < 252].all())
    assert bool((om.values(codes, scales)[:, [0, 31]] == 0).all())


def test_oracle_ties_signs_and_nonfinite_blocks():
    x = torch.tensor([6.0, -0.25, 0.25, 0.75, 1.25, 1.75, -2.5, 3.5, 5.0, -0.0, 0.2578125, 4.96875] + [0.0] * 20).bfloat16()[None]
    codes, scales = om.quantize(x)
    assert scales.tolist() == [[127]]
    assert codes[0, :12].tolist() == [7, 8, 0, 2, 2, 4, 12, 6, 6, 8, 1, 6]
    x[0, 3] = float("inf")
    codes, scales = om.quantize(x)
    assert scales.tolist() == [[255]] and not codes.any() and torch.isnan(om.values(codes, scales)).all()


def test_panels_round_trip():
    g = torch.Generator().manual_seed(1)
    for rows, blocks in ((1, 1), (3, 5), (16, 4), (17, 12), (130, 7), (0, 3)):
        c = torch.randint(0, 256, (rows, 16 * blocks), generator=g, dtype=torch.int64).to(torch.uint8)
        s = torch.randint(0, 256, (rows, blocks), generator=g, dtype=torch.int64).to(torch.uint8)
        q = mxfp4.from_rows(c, s)
        want = om.panels(c, s)
        assert torch.equal(q.codes, want[0]) and torch.equal(q.scales, want[1]) and q[2:] == (rows, 32 * blocks)
        back = mxfp4.to_rows(q)
        assert torch.equal(back[0], c) and torch.equal(back[1], s)
    for c, s in ((torch.zeros((2, 16)), torch.zeros((2, 1))), (torch.zeros(16, dtype=torch.uint8), torch.zeros((1, 1), dtype=torch.uint8))):
        with pytest.raises(ValueError, match="expected uint8"):
            mxfp4.from_rows(c, s)
    for shape_c, shape_s in (((2, 16), (2, 2)), ((2, 24), (2, 1)), ((2, 16), (3, 1))):
        with pytest.raises(ValueError, match="do not go with"):
            mxfp4.from_rows(torch.zeros(shape_c, dtype=torch.uint8), torch.zeros(shape_s, dtype=torch.uint8))


def test_python_refusals():
    bf = torch.zeros((4, 64), dtype=torch.bfloat16)
    for bad, text in ((bf.float(), "bf16"), (bf[0], "bf16"), (bf[:, :40], "not a multiple of 32")):
        with pytest.raises(ValueError, match=text):
            mxfp4.quant_mxfp4(bad)
    with pytest.raises(ValueError, match="on a GPU"):
        mxfp4.quant_mxfp4(bf)
    q = mxfp4.from_rows(torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8))
    with pytest.raises(ValueError, match="on a GPU"):
        mxfp4.dequant_mxfp4(*q)
    for bad, text in ((q._replace(rows=17), "q's codes must be"), (q._replace(k=160), "q's codes must be"), (q._replace(k=48), "not a multiple"),
                      (q._replace(rows=-1), "-1 rows"), (q._replace(scales=q.scales[:, :, :8]), "q's scales must be"),
                      (q._replace(codes=q.codes.float()), "q's codes must be"),
                      (q._replace(codes=torch.zeros(1025, dtype=torch.uint8)[1:].view(1, 1, 4, 16, 16)), "16-byte aligned")):
        with pytest.raises(ValueError, match=text):
            mxfp4.dequant_mxfp4(*bad)
    for out in (torch.zeros((4, 64)), bf[:, :32], torch.zeros((4, 68), dtype=torch.bfloat16)[:, :64], bf.t()):
        with pytest.raises(ValueError, match="out must be bf16"):
            mxfp4.dequant_mxfp4(*q, out=out)
    wide = mxfp4.from_rows(torch.zeros((4, 64), dtype=torch.uint8), torch.zeros((4, 4), dtype=torch.uint8))
    with pytest.raises(ValueError, match="a has rows of 64 values"):
        mxfp4.gemm_mxfp4(q, wide)
    with pytest.raises(ValueError, match="bias must be"):
        mxfp4.gemm_mxfp4(q, q, bias=torch.zeros(4))
    with pytest.raises(ValueError, match="on a GPU"):
        mxfp4.gemm_mxfp4(q, q)
    with pytest.raises(ValueError, match="move the weight to a GPU"):
        mxfp4.WaveMxfp4Linear(bf, None)
    for n, k in ((6, 32), (4, 0)):
        with pytest.raises(ValueError, match="unsupported linear shape"):
            mxfp4.WaveMxfp4Linear.from_quantized(mxfp4.from_rows(torch.zeros((n, k // 2), dtype=torch.uint8), torch.zeros((n, k // 32), dtype=torch.uint8)))
    linear = mxfp4.WaveMxfp4Linear.from_quantized(q, torch.zeros(4))
    assert linear.bias.dtype == torch.bfloat16 and linear.in_features == 64 and linear.weight_rows == q
    with pytest.raises(ValueError, match="input width 32"):
        linear(torch.zeros((1, 32), dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="on a GPU"):
        linear(bf)
    with pytest.raises(ValueError, match="bias has shape"):
        mxfp4.WaveMxfp4Linear.from_quantized(q, torch.zeros(5))


def test_swap_refuses_what_the_others_refuse():
    with pytest.raises(ValueError, match="no .blocks"):
        mxfp4.quantize_transformer_mxfp4(nn.Linear(2, 2))


@pytest.mark.parametrize("args, text", [
    ((16, -1, 32, 32, 16, 16, None), "bad sizes"),
    ((16, 1, 64, 32, 16, 16, None), "bad sizes"),
    ((16, 1, 48, 48, 16, 16, None), "multiple of 32"),
    ((16, 1 << 28, 32, 32, 16, 16, None), "too large"),
    ((16, 1, 1 << 28, 1 << 28, 16, 16, None), "too large"),
    ((16, 1 << 20, 1 << 20, 1 << 20, 16, 16, None), "too large"),
    ((None, 1, 32, 32, 16, 16, None), "null pointer"),
    ((8, 1, 32, 32, 16, 16, None), "16-byte aligned"),
    ((16, 1, 32, 36, 16, 16, None), "16-byte aligned"),
    ((16, 1, 32, 32, 16, 8, None), "16-byte aligned"),
])
def test_quant_refusals(args, text):
    with pytest.raises(RuntimeError, match=text):
        _lib.call("wf_mxfp4_quant", *args)
    x, rows, k, ld, codes, scales, st = args
    with pytest.raises(RuntimeError, match=text):
        _lib.call("wf_mxfp4_dequant", codes, scales, rows, k, x, ld, st)


@pytest.mark.parametrize("change, text", [
    (dict(m=-1), "bad sizes"), (dict(ldy=4), "bad sizes"), (dict(k=48), "multiple of 32"), (dict(k=0), "multiple of 32|bad sizes"),
    (dict(n=6), "multiples of 4"), (dict(ldy=10), "multiples of 4"), (dict(a=None), "null pointer"), (dict(w=None), "null pointer"),
    (dict(y=None), "null pointer"), (dict(w_scales=None), "null pointer"), (dict(w=24), "aligned"), (dict(a=24), "aligned"),
    (dict(y=4), "aligned"), (dict(bias=4), "aligned"), (dict(flags=2), "unknown flags"), (dict(m=1 << 27, k=64), "2 GiB"),
    (dict(n=1 << 27, ldy=1 << 27, k=64), "2 GiB"), (dict(m=1 << 24, n=1 << 24, ldy=1 << 24, k=32), "too large"),
])
def test_product_refusals(change, text):
    d = dict(a=16, a_scales=16, w=16, w_scales=16, m=20, n=8, k=32, bias=None, y=16, ldy=8, flags=0)
    d.update(change)
    with pytest.raises(RuntimeError, match=text):
        _lib.call("wf_gemm_mxfp4", d["a"], d["a_scales"], d["w"], d["w_scales"], d["m"], d["n"], d["k"], d["bias"], d["y"], d["ldy"],
                  d["flags"], None)
    if "a" in change:
        d["x"] = d["a"]
        text = "null pointer|aligned"
    with pytest.raises(RuntimeError, match=text):
        _lib.call("wf_mxfp4_linear", d.get("x", 16), d["m"], d["k"], max(d["k"], 64) if "a" not in change else 36, d["w"], d["w_scales"],
                  d["bias"], d["n"], d["y"], d["ldy"], d["flags"], 16, 16, None)


def test_linear_needs_a_workspace_above_the_fused_rows():
    with pytest.raises(RuntimeError, match="null workspace"):
        _lib.call("wf_mxfp4_linear", 16, 17, 32, 32, 16, 16, None, 8, 16, 8, 0, None, 16, None)
    with pytest.raises(RuntimeError, match="workspaces must be"):
        _lib.call("wf_mxfp4_linear", 16, 17, 32, 32, 16, 16, None, 8, 16, 8, 0, 16, 8, None)
    for fn, args in (("wf_gemm_mxfp4", (None, None, None, None, 0, 8, 32, None, None, 8, 0, None)),
                     ("wf_mxfp4_linear", (None, 0, 32, 32, None, None, None, 8, None, 8, 0, None, None, None)),
                     ("wf_mxfp4_quant", (None, 0, 32, 32, None, None, None))):
        _lib.call(fn, *args)   # nothing to do


# the scale rule of csrc/mxfp4_codec.hpp, from the bits
def test_scale_byte_from_the_bits_is_the_definition():
    x = every_bf16()[:0x7f80]
    bits = torch.arange(0x7f80)
    byte = (((bits + 0x20) >> 7) - 2).clamp(2, 252)
    block = torch.zeros((len(x), 32), dtype=torch.bfloat16)
    block[:, 0] = x
    assert torch.equal(om.quantize(block)[1][:, 0].long(), byte)


# -------------------------------------------------------------------- pages
def test_page_pools():
    from waveforcing_amd.kv import Fp8PagePool, Int8PagePool, Mxfp4PagePool

    pool = Mxfp4PagePool(3, 2, 128, 16, "cpu")
    assert pool.k_codes.shape == (3, 16, 2, 64) and pool.v_scales.shape == (3, 2, 16, 4) and pool.v_scales.dtype == torch.uint8
    assert pool.nbytes == Mxfp4PagePool.bytes_for(3, 2, 128, 16)
    for call in (pool.pack, pool.unpack, pool.pack_k_norm_rope):
        with pytest.raises(TypeError, match="MXFP4 pages"):
            call()
    for other in (Fp8PagePool, Int8PagePool):
        with pytest.raises(TypeError, match="another code format"):
            other.view_of(pool, 0, 1)
        with pytest.raises(TypeError, match="another code format"):
            Mxfp4PagePool.view_of(other(3, 2, 128, 16, "cpu"), 0, 1)
    assert Mxfp4PagePool.view_of(pool, 1, 2).k_scales.data_ptr() == pool.k_scales[1].data_ptr()


def test_one_sequence_attention_refuses_the_pages():
    from waveforcing_amd import backend
    from waveforcing_amd.kv import Mxfp4PagePool, PagedKV

    pool = Mxfp4PagePool(3, 2, 128, 64, "cpu")
    with pytest.raises(Exception, match="e4m3"):
        backend.attn_paged_fp8(torch.zeros((1, 2, 128), dtype=torch.bfloat16), PagedKV(pool, pool.page_table([0]), 1))


def test_unknown_formats_are_refused():
    for fmt in (-1, 2, 3, 5):
        with pytest.raises(RuntimeError, match="unknown cache format"):
            _lib.call("wf_kv_batch_append", 16, 16, 1, 2, 128, 256, fmt, 16, 16, 1, 16, 1, 16, 16, 16, 16, 16, 4, None)
