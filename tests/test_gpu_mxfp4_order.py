"""The MXFP4 linear equals quantization and product bit for bit where the order of its sums shows: blocks of one row many
binades apart, at every form of the few-rows kernel."""

import pytest
import torch

from waveforcing_amd import mxfp4

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def spread(m, k, g, binades):
    """bf16 rows whose blocks of 32 differ by a normal number of binades: their sums are not exact in fp32."""
    x = torch.randn((m, k // 32, 32), generator=g, device=DEV)
    e = torch.randn((m, k // 32, 1), generator=g, device=DEV) * binades
    return (x * torch.exp2(e)).reshape(m, k).bfloat16()


@pytest.mark.parametrize("n", [1536, 5120, 8188, 8192, 13824])
def test_linear_is_quantization_and_product(n):
    k = 5120
    g = torch.Generator(device=DEV).manual_seed(n)
    w = mxfp4.quant_mxfp4(spread(n, k, g, 4))
    bias = torch.randn((n,), generator=g, device=DEV).bfloat16()
    linear = mxfp4.WaveMxfp4Linear.from_quantized(w, bias)
    for m in (1, 4, 5, 8, 9, 12, 16, 17, 40):
        for binades in (4, 6):
            x = spread(m, k, g, binades)
            y, z = linear(x)[0], mxfp4.gemm_mxfp4(mxfp4.quant_mxfp4(x), w, bias)
            assert torch.equal(y, z), f"m={m}: {int((y != z).sum())} of {y.numel()} differ"
