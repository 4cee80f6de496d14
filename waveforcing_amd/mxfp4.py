"""Microscaled 4-bit floating point (MXFP4) rows and linears on the HIP kernels.

Blocks of 32 consecutive values hold e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) under a power of two
(E8M0): 17 bytes for 32 values.  The matrix cores take codes and scales as they are, at twice the rate of 8-bit operands,
and a linear's weight is read in half the bytes of an 8-bit one.  The 4-bit counterpart of the W8A8 linears of
``waveforcing_amd.fp8`` (wave_rt/runtime/fp8.py:21-61; the reference has no 4-bit form), with the same interfaces:
``WaveMxfp4Linear.forward(x) -> (y, None)`` and an in-place module swap over ``transformer.blocks``.

Scales are laid out for the kernels: uint8 ``[ceil(k / 128), rows4, 4]`` with ``rows4`` the rows rounded up to 4, byte b of
(g, r) belonging to values ``128 g + 32 b .. + 31`` of row r.  :func:`scales_to_rows` and :func:`scales_from_rows` convert
to and from one row of ``k / 32`` bytes for every row, the layout in which MX checkpoints hold them.
"""

from __future__ import annotations

import torch
import torch.nn as nn

from . import _lib
from .fp8 import _resolve_scope, _swap_block_linears
from .kv import dense

BLOCK = 32


def _scales_shape(rows: int, k: int) -> tuple[int, int, int]:
    return -(-k // 128), -(-rows // 4) * 4, 4


def _rows(x: torch.Tensor, name: str) -> torch.Tensor:
    """bf16 rows [R, K] (K % 32 == 0) on a GPU, as the kernels read them; a copy if their strides or address do not allow it."""
    if x.dim() != 2 or x.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bf16 [rows, k], got {tuple(x.shape)} {x.dtype}")
    if x.shape[1] % BLOCK:
        raise ValueError(f"{name} has rows of {x.shape[1]} values: not a multiple of {BLOCK}")
    rows, k = x.shape
    if rows and k and (x.stride(1) != 1 or x.data_ptr() % 16 or (rows > 1 and (x.stride(0) % 8 or x.stride(0) < k))):
        x = dense(x)
    return x


def _ld(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _operand(codes: torch.Tensor, scales: torch.Tensor, name: str) -> tuple[int, int]:
    """(rows, k) of codes and scales as :func:`quant_mxfp4` returns them."""
    if codes.dim() != 2 or codes.dtype != torch.uint8 or not codes.is_contiguous() or codes.shape[1] % 16:
        raise ValueError(f"{name} codes must be contiguous uint8 [rows, k / 2] with k % 32 == 0, got {tuple(codes.shape)} {codes.dtype}")
    rows, k = codes.shape[0], 2 * codes.shape[1]
    if tuple(scales.shape) != _scales_shape(rows, k) or scales.dtype != torch.uint8 or not scales.is_contiguous():
        raise ValueError(f"{name} scales must be contiguous uint8 {_scales_shape(rows, k)}, got {tuple(scales.shape)} {scales.dtype}")
    if scales.device != codes.device:
        raise ValueError(f"{name} codes are on {codes.device}, its scales on {scales.device}")
    if codes.numel() and (codes.data_ptr() % 16 or scales.data_ptr() % 16):
        raise ValueError(f"{name} codes and scales must be 16-byte aligned")
    return rows, k


def _output(out: torch.Tensor | None, rows: int, cols: int, device, align: int) -> torch.Tensor:
    """A new bf16 [rows, cols], or the given one if the kernels can write it (row stride a multiple of ``align``)."""
    if out is None:
        return torch.empty((rows, cols), dtype=torch.bfloat16, device=device)
    if (tuple(out.shape) != (rows, cols) or out.dtype != torch.bfloat16 or out.device != device
            or (out.numel() and (out.stride(1) != 1 or out.data_ptr() % (2 * align)
                                 or (rows > 1 and (out.stride(0) % align or out.stride(0) < cols))))):
        raise ValueError(f"out must be bf16 [{rows}, {cols}] on {device} with dense rows whose stride {align} divides")
    return out


def quant_mxfp4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes uint8 [R, K / 2], scales uint8 [ceil(K / 128), R4, 4]) of bf16 rows [R, K], K % 32 == 0 (wf_mxfp4_quant).

    Per block, s is the smallest power of two with max|x| < 7 s (2^-125 to 2^125), a code the nearest e2m1 number to x / s,
    an even code on a tie, at most 6.  A block that holds a NaN or an infinity reads back as NaN."""
    x = _rows(x, "x")
    R, K = x.shape
    codes = torch.empty((R, K // 2), dtype=torch.uint8, device=x.device)
    scales = torch.empty(_scales_shape(R, K), dtype=torch.uint8, device=x.device)
    _lib.call_on(x.device, "wf_mxfp4_quant", x.data_ptr(), R, K, _ld(x), codes.data_ptr(), scales.data_ptr())
    return codes, scales


def dequant_mxfp4(codes: torch.Tensor, scales: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of codes and scales as bf16 [R, K], exact (wf_mxfp4_dequant)."""
    R, K = _operand(codes, scales, "the")
    out = _output(out, R, K, codes.device, 8)
    _lib.call_on(codes.device, "wf_mxfp4_dequant", codes.data_ptr(), scales.data_ptr(), R, K, out.data_ptr(), _ld(out))
    return out


def scales_to_rows(scales: torch.Tensor, rows: int, k: int) -> torch.Tensor:
    """Scales of :func:`quant_mxfp4` as E8M0 bytes [rows, k / 32]."""
    if tuple(scales.shape) != _scales_shape(rows, k) or k % BLOCK:
        raise ValueError(f"scales of {rows} rows of {k} values have shape {_scales_shape(rows, k)}, got {tuple(scales.shape)}")
    return scales.transpose(0, 1).flatten(1)[:rows, :k // BLOCK].contiguous()


def scales_from_rows(scales: torch.Tensor) -> torch.Tensor:
    """E8M0 bytes [rows, k / 32] in the kernels' layout."""
    if scales.dim() != 2 or scales.dtype != torch.uint8:
        raise ValueError(f"expected uint8 [rows, k / 32], got {tuple(scales.shape)} {scales.dtype}")
    rows, blocks = scales.shape
    g, rows4, _ = _scales_shape(rows, BLOCK * blocks)
    out = torch.zeros((rows4, 4 * g), dtype=torch.uint8, device=scales.device)
    out[:rows, :blocks] = scales
    return out.view(rows4, g, 4).transpose(0, 1).contiguous()


def _bias(bias: torch.Tensor | None, n: int, device) -> torch.Tensor | None:
    if bias is not None and (tuple(bias.shape) != (n,) or bias.dtype != torch.bfloat16 or bias.device != device
                             or not bias.is_contiguous() or bias.data_ptr() % 8):
        raise ValueError(f"bias must be contiguous bf16 [{n}] on {device}")
    return bias


def gemm_mxfp4(a_codes: torch.Tensor, a_scales: torch.Tensor, w_codes: torch.Tensor, w_scales: torch.Tensor,
               bias: torch.Tensor | None = None, gelu: bool = False, out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [M, N] = act(a [M, K] x w [N, K]^T + bias) of two operands of :func:`quant_mxfp4` (wf_gemm_mxfp4): fp32 sums,
    act GELU(tanh) with ``gelu``, rounded once.  N must be a multiple of 4."""
    M, K = _operand(a_codes, a_scales, "a")
    N, kw = _operand(w_codes, w_scales, "w")
    if kw != K or w_codes.device != a_codes.device:
        raise ValueError(f"a has rows of {K} values on {a_codes.device}, w of {kw} on {w_codes.device}")
    out = _output(out, M, N, a_codes.device, 4)
    _lib.call_on(a_codes.device, "wf_gemm_mxfp4", a_codes.data_ptr(), a_scales.data_ptr(), w_codes.data_ptr(), w_scales.data_ptr(),
                 M, N, K, _lib.ptr(_bias(bias, N, a_codes.device)), out.data_ptr(), _ld(out), _lib.GEMM_GELU_TANH if gelu else 0)
    return out


class WaveMxfp4Linear(nn.Module):
    """4-bit linear (weights and activations MXFP4) with the reference linear's return contract ``(y, None)``.

    The weight is quantized once at construction, activations at every call (up to 16 rows inside the product's kernel, one
    launch); ``gelu`` folds GELU(tanh) into the result."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, gelu: bool = False) -> None:
        super().__init__()
        if weight.dim() != 2:
            raise ValueError("weight must be 2-D [out, in]")
        if not weight.is_cuda:
            raise ValueError("WaveMxfp4Linear quantizes on the GPU; move the weight to a GPU first")
        self._take(*quant_mxfp4(self._checked(weight).detach().to(torch.bfloat16)), bias, gelu)

    @staticmethod
    def _checked(weight: torch.Tensor) -> torch.Tensor:
        n, k = weight.shape
        if k % BLOCK or n % 4 or not k:
            raise ValueError(f"unsupported linear shape {tuple(weight.shape)} (in % {BLOCK}, out % 4 required)")
        return weight

    @classmethod
    def from_codes(cls, codes: torch.Tensor, scales: torch.Tensor, bias: torch.Tensor | None = None,
                   gelu: bool = False) -> "WaveMxfp4Linear":
        """A linear of a weight that is quantized already: codes uint8 [out, in / 2] and scales as :func:`quant_mxfp4` returns
        them, or E8M0 bytes [out, in / 32]."""
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        if scales.dim() == 2:
            scales = scales_from_rows(scales)
        n, k = _operand(codes, scales, "weight")
        cls._checked(codes.new_empty((n, k), device="meta"))
        self._take(codes, scales, bias, gelu)
        return self

    def _take(self, codes, scales, bias, gelu) -> None:
        self.out_dtype = torch.bfloat16
        self.out_features, self.in_features = codes.shape[0], 2 * codes.shape[1]
        self.register_buffer("w_codes", codes)
        self.register_buffer("w_scales", scales)
        if bias is not None:
            bias = bias.detach().to(device=codes.device, dtype=torch.bfloat16).contiguous()
            if tuple(bias.shape) != (self.out_features,):
                raise ValueError(f"bias has shape {tuple(bias.shape)}, the weight {self.out_features} rows")
            self.register_buffer("bias", bias)
        else:
            self.bias = None
        self.gelu = gelu

    def _raw(self, x2: torch.Tensor) -> torch.Tensor:
        if x2.dim() != 2 or x2.shape[1] != self.in_features:
            raise ValueError(f"input width {x2.shape[-1]} != in_features {self.in_features}")
        if x2.device != self.w_codes.device:
            raise ValueError(f"x is on {x2.device}, the weight on {self.w_codes.device}")
        x2 = _rows(x2, "x")
        M, K = x2.shape
        y = torch.empty((M, self.out_features), dtype=torch.bfloat16, device=x2.device)
        codes = scales = None
        if M > _lib.MXFP4_FUSED_ROWS:
            codes = torch.empty((M, K // 2), dtype=torch.uint8, device=x2.device)
            scales = torch.empty(_scales_shape(M, K), dtype=torch.uint8, device=x2.device)
        _lib.call_on(x2.device, "wf_mxfp4_linear", x2.data_ptr(), M, K, _ld(x2), self.w_codes.data_ptr(), self.w_scales.data_ptr(),
                     _lib.ptr(self.bias), self.out_features, y.data_ptr(), self.out_features,
                     _lib.GEMM_GELU_TANH if self.gelu else 0, _lib.ptr(codes), _lib.ptr(scales))
        return y

    def forward(self, x: torch.Tensor):
        shape = x.shape
        y = self._raw(x.reshape(-1, shape[-1]))
        return y.reshape(*shape[:-1], self.out_features), None


def quantize_transformer_mxfp4(transformer: nn.Module, verbose: bool = False, scope: str | None = None,
                               fuse_gelu: bool = True) -> int:
    """Replace selected block linears in place with WaveMxfp4Linear; return the count.

    Selection and errors follow wave_rt/runtime/fp8.py:93-137.  With ``fuse_gelu`` a block whose ``ffn.act`` is
    ``nn.GELU(approximate='tanh')`` gets the activation folded into fc_in (``ffn.act`` becomes Identity)."""

    def make(parent, leaf, w, b):
        act = getattr(parent, "act", None)
        gelu = fuse_gelu and leaf == "fc_in" and isinstance(act, nn.GELU) and act.approximate == "tanh"
        linear = WaveMxfp4Linear(w, b, gelu=gelu)
        if gelu:
            setattr(parent, "act", nn.Identity())
        return linear

    scope = _resolve_scope(scope)
    n = _swap_block_linears(transformer, scope, make)
    if verbose:
        print(f"[wave-mxfp4] quantized {n} linears to MXFP4 (scope={scope})", flush=True)
    return n
