"""MXFP4 rows and linears on the GPU: codes and scales bit for bit, products against 64 bits within the arithmetic's bound
(oracle/mxfp4.py: product)."""

import pytest
import torch
import torch.nn as nn

from oracle import mxfp4 as om
from waveforcing_amd import mxfp4

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def rows(m, k, g, scale=1.0):
    x = torch.randn((m, k), generator=g, device=DEV) * scale
    x[:, torch.rand((k,), generator=g, device=DEV) < 0.02] *= 20
    return x.bfloat16()


def same(x, y):
    assert x.shape == y.shape and x.dtype == y.dtype
    assert torch.equal(x, y), f"{int((x != y).sum())} of {x.numel()} differ"


def check(out, ref, bound):
    out = out.double()
    assert bool((torch.isnan(out) == torch.isnan(ref)).all())
    off = ((out - ref).abs() - bound).nan_to_num(0)
    assert float(off.max()) <= 0, f"off by {float((out - ref).abs().nan_to_num(0).max()):.3g}, over the bound by {float(off.max()):.3g}"


def exact(x):
    return om.values(*om.quantize(x))


# ------------------------------------------------------------------- rows
@pytest.mark.parametrize("m, k", [(1, 32), (2, 64), (5, 96), (3, 128), (4, 160), (16, 512), (3, 544), (17, 1568), (65, 2080), (301, 4128)])
def test_rows_and_back(m, k):
    g = gen(m + k)
    wide = rows(m, k + 24, g)
    x = wide[:, 8:8 + k]                     # rows with a stride of their own, 16 bytes into them
    x[0] = 0
    x[m - 1, k - 1] = float("nan")
    x[m // 2, 3] = float("-inf")
    q = mxfp4.quant_mxfp4(x)
    c, s = om.quantize(x)
    for got, want in zip(q, om.panels(om.pack(c), s)):
        same(got, want)
    assert q[2:] == (m, k)
    for got, want in zip(mxfp4.to_rows(q), (om.pack(c), s)):
        same(got, want)
    out = torch.full((m, k + 16), 7.0, dtype=torch.bfloat16, device=DEV)
    mxfp4.dequant_mxfp4(*q, out=out[:, 8:8 + k])
    assert bool((out[:, :8] == 7).all()) and bool((out[:, 8 + k:] == 7).all())
    want = om.values(c, s).float().bfloat16()
    torch.testing.assert_close(out[:, 8:8 + k], want, rtol=0, atol=0, equal_nan=True)
    torch.testing.assert_close(mxfp4.dequant_mxfp4(*q), want, rtol=0, atol=0, equal_nan=True)


def test_every_bf16_under_every_neighbouring_maximum():
    """Each bf16 as its block's largest value, and as another's neighbour at 1, 1.75, 3.49 and 100 times it."""
    x = torch.arange(65536, dtype=torch.int32, device=DEV).to(torch.int16).view(torch.bfloat16)
    block = torch.zeros((65536, 5 * 32), dtype=torch.bfloat16, device=DEV)
    for i, f in enumerate((0, 1, 1.75, 3.49, 100)):
        block[:, 32 * i + 9] = x
        block[:, 32 * i + 20] = (x.float() * -f).bfloat16()
    codes, scales = mxfp4.to_rows(mxfp4.quant_mxfp4(block))
    c, s = om.quantize(block)
    same(scales, s)
    same(codes, om.pack(c))


def test_every_code_and_scale_byte_reads_back():
    codes = torch.arange(256, dtype=torch.int64, device=DEV).to(torch.uint8)[:, None].expand(256, 16 * 256).contiguous()
    s = torch.arange(256, dtype=torch.int64, device=DEV).to(torch.uint8)[None].expand(256, 256).contiguous()
    got = mxfp4.dequant_mxfp4(*mxfp4.from_rows(codes, s))
    want = om.values(om.unpack(codes), s).float().bfloat16()
    torch.testing.assert_close(got, want, rtol=0, atol=0, equal_nan=True)


def test_unaligned_and_transposed_rows_are_copied_and_empty_ones_pass():
    g = gen(5)
    x = rows(7, 65 * 32 + 1, g)[:, 1:]
    same(mxfp4.quant_mxfp4(x)[0], mxfp4.quant_mxfp4(x.clone())[0])
    t = rows(64, 40, g).t()
    same(mxfp4.quant_mxfp4(t)[0], mxfp4.quant_mxfp4(t.contiguous())[0])
    empty = mxfp4.quant_mxfp4(x[:0])
    assert empty.codes.shape == (0, 17, 4, 16, 16) and mxfp4.dequant_mxfp4(*empty).shape == (0, 2080)


# --------------------------------------------------------------- products
ROWS = [1, 2, 7, 15, 16, 17, 31, 32, 33, 48, 49, 63, 64, 65, 100, 127, 128, 129, 200, 257, 300, 520]


@pytest.mark.parametrize("k, n", [(32, 4), (96, 36), (128, 64), (160, 260), (544, 132), (1568, 2212), (2080, 516), (256, 1028)])
def test_linear_at_every_row_count(k, n):
    g = gen(k + n)
    w, b = rows(n, k, g, 0.05), rows(1, n, g)[0].contiguous()
    for i, m in enumerate(ROWS):
        x = rows(m, k, g)
        bias, gelu = (b if i % 3 else None), i % 2 == 1
        linear = mxfp4.WaveMxfp4Linear(w, bias, gelu=gelu)
        y, none = linear(x)
        assert none is None
        check(y, *om.product(exact(x), exact(w), bias, gelu))
        same(y, mxfp4.gemm_mxfp4(mxfp4.quant_mxfp4(x), linear.weight_rows, linear.bias, gelu))
        same(y, linear(x)[0])


@pytest.mark.parametrize("m, k, n", [(1, 1536, 4608), (16, 5120, 13824), (3, 13824, 5120), (40, 8960, 1536), (64, 5120, 5120),
                                     (390, 1536, 8960), (1560, 1536, 1536), (1100, 1568, 8196), (4680, 1536, 4608), (2000, 5120, 5120),
                                     (4680, 1536, 8960), (1560, 5120, 13824), (4680, 5120, 5120), (4681, 2592, 5124), (2570, 800, 7172)])
def test_linear_at_the_presets_sizes(m, k, n):
    g = gen(m + k + n)
    x, w, b = rows(m, k, g), rows(n, k, g, 0.02), rows(1, n, g)[0].contiguous()
    linear = mxfp4.WaveMxfp4Linear(w, b)
    check(linear(x)[0], *om.product(exact(x), exact(w), b))


@pytest.mark.parametrize("m", [3, 16, 40, 64, 100, 300, 700])
def test_strides_shapes_and_given_outputs(m):
    g = gen(m)
    k, n = 416, 196
    w = rows(n, k, g, 0.05)
    linear = mxfp4.WaveMxfp4Linear(w, None)
    wide = rows(m, k + 40, g)
    x = wide[:, 16:16 + k]
    y = linear(x)[0]
    check(y, *om.product(exact(x.contiguous()), exact(w)))
    same(linear(x.reshape(1, m, k))[0][0], y)
    same(linear(rows(2 * m, k, gen(m))[::2][:m].clone())[0], linear(rows(2 * m, k, gen(m))[::2])[0])
    out = torch.full((m + 2, n + 12), 7.0, dtype=torch.bfloat16, device=DEV)
    q = mxfp4.quant_mxfp4(x)
    for lo in (4, 8):                        # rows of 8-byte and of 16-byte alignment
        out.fill_(7.0)
        got = mxfp4.gemm_mxfp4(q, linear.weight_rows, out=out[1:m + 1, lo:lo + n])
        same(got, y)
        out[1:m + 1, lo:lo + n] = 7
        assert bool((out == 7).all())
    assert linear(x[:0])[0].shape == (0, n)


def test_bias_out_of_a_larger_tensor_and_a_module_cast_to_another_type():
    g = gen(8)
    w, b = rows(100, 96, g, 0.1), rows(1, 131, g)[0]
    for m in (3, 40, 200):
        x = rows(m, 96, g)
        for at in (0, 1, 3, 31):             # 2, 6 and 62 bytes into its storage too
            check(mxfp4.WaveMxfp4Linear(w, b[at:at + 100])(x)[0], *om.product(exact(x), exact(w), b[at:at + 100]))
        cast = mxfp4.WaveMxfp4Linear(w, b[:100]).float()
        with pytest.raises(ValueError, match="bias has become torch.float32"):
            cast(x)
        same(cast.bfloat16()(x)[0], mxfp4.WaveMxfp4Linear(w, b[:100])(x)[0])


@pytest.mark.parametrize("m", [1, 16, 33, 64, 130, 600])
def test_nonfinite_rows_stay_by_themselves(m):
    g = gen(m)
    k, n = 352, 300
    x, w = rows(m, k, g), rows(n, k, g, 0.05)
    clean = mxfp4.WaveMxfp4Linear(w, None)(x)[0]
    bad, wbad = x.clone(), w.clone()
    bad[m - 1, k - 1] = float("inf")
    y = mxfp4.WaveMxfp4Linear(w, None)(bad)[0]
    assert bool(torch.isnan(y[m - 1]).all())
    same(y[:m - 1], clean[:m - 1])
    wbad[n - 1, 0] = float("nan")
    y = mxfp4.WaveMxfp4Linear(wbad, None)(x)[0]
    assert bool(torch.isnan(y[:, n - 1]).all())
    same(y[:, :n - 1], clean[:, :n - 1])


@pytest.mark.parametrize("m", [4, 50, 200])
def test_ranges_of_the_scales(m):
    """Rows and weights at the ends of bf16: products far apart, sums that stay finite, values below the smallest scale."""
    g = gen(m)
    k, n = 256, 64
    x, w = rows(m, k, g), rows(n, k, g)
    e = torch.arange(m, device=DEV) % 4
    x = (x.float() * torch.tensor([2.0 ** -130, 2.0 ** -60, 1.0, 2.0 ** 60], device=DEV)[e][:, None]).bfloat16()
    w[:, 128:] = (w[:, 128:].float() * 2.0 ** -40).bfloat16()
    check(mxfp4.WaveMxfp4Linear(w, None)(x)[0], *om.product(exact(x), exact(w)))


@pytest.mark.parametrize("m", [2, 30, 200])
def test_padding_rows_of_panels_reach_nothing(m):
    """Whatever stands in a panel's rows and values past the last: NaN scales and codes of other rows."""
    g = gen(m)
    k, n = 416, 36                           # 14 values blocks of 16, 4 rows of the last panel
    x, w = rows(m, k, g), rows(n, k, g, 0.05)
    a, b = mxfp4.quant_mxfp4(x), mxfp4.quant_mxfp4(w)
    want = mxfp4.gemm_mxfp4(a, b)
    for q in (a, b):
        last = q.rows - 16 * (q.codes.shape[0] - 1)
        q.codes[-1, :, :, last:] = 0x77
        q.scales[-1, :, last:] = 255
    same(mxfp4.gemm_mxfp4(a, b), want)
    same(mxfp4.dequant_mxfp4(*a), exact(x).float().bfloat16())


def test_captured_linear_replays_and_two_streams():
    g = gen(9)
    w = rows(516, 544, g, 0.05)
    linear = mxfp4.WaveMxfp4Linear(w, None, gelu=True)
    xs = [rows(m, 544, g) for m in (5, 40, 200)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        for x in xs:
            linear(x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [linear(x)[0] for x in xs]
    for _ in range(3):
        for x in xs:
            x.copy_(rows(*x.shape, g))
        graph.replay()
        torch.cuda.synchronize()
        for x, o in zip(xs, outs):
            same(o, linear(x)[0])
    want = [linear(x)[0] for x in xs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(10):
        for st in streams:
            with torch.cuda.stream(st):
                got.append([linear(x)[0] for x in xs])
    torch.cuda.synchronize()
    for ys in got:
        for y, z in zip(ys, want):
            same(y, z)


def test_a_transformers_blocks_swapped():
    class Block(nn.Module):
        def __init__(self):
            super().__init__()
            self.proj = nn.Linear(64, 64)
            self.ffn = nn.Module()
            self.ffn.fc_in, self.ffn.act, self.ffn.fc_out = nn.Linear(64, 160), nn.GELU(approximate="tanh"), nn.Linear(160, 64)

    model = nn.Module()
    model.blocks = nn.ModuleList([Block() for _ in range(2)]).to(DEV).to(torch.bfloat16)
    w = model.blocks[0].ffn.fc_in.weight.detach().clone()
    b = model.blocks[0].ffn.fc_in.bias.detach().clone()
    assert mxfp4.quantize_transformer_mxfp4(model) == 4
    assert mxfp4.quantize_transformer_mxfp4(model) == 0
    ffn = model.blocks[0].ffn
    assert isinstance(ffn.act, nn.Identity) and ffn.fc_in.gelu and not ffn.fc_out.gelu
    x = rows(20, 64, gen(2))
    check(ffn.fc_in(x)[0], *om.product(exact(x), exact(w), b, True))
    assert mxfp4.quantize_transformer_mxfp4(model, scope="all") == 2
