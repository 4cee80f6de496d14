"""Microscaled 4-bit floating point (MXFP4) rows and linears on the HIP kernels.

Blocks of 32 consecutive values hold e2m1 codes (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives) under a power of two
(E8M0): 17 bytes for 32 values.  The matrix cores take codes and scales as they are, at twice the rate of 8-bit operands,
and a linear's weight is read in half the bytes of an 8-bit one.  The 4-bit counterpart of the W8A8 linears of
``waveforcing_amd.fp8`` (wave_rt/runtime/fp8.py:21-61; the reference has no 4-bit form), with the same interfaces:
``WaveMxfp4Linear.forward(x) -> (y, None)`` and an in-place module swap over ``transformer.blocks``.

Quantized rows are laid out for the kernels, in panels of 16 rows by 128 values that a wave's matrix instruction takes as they
lie in memory (:class:`Mxfp4Rows`); :func:`to_rows` and :func:`from_rows` convert to and from codes and scales row by row, as MX
checkpoints hold them.
"""

from __future__ import annotations

from typing import NamedTuple

import torch
import torch.nn as nn

from . import _lib
from .fp8 import _resolve_scope, _swap_block_linears
from .kv import dense

BLOCK = 32


class Mxfp4Rows(NamedTuple):
    """``rows`` quantized rows of ``k`` values, as :func:`quant_mxfp4` returns them; P = ceil(rows / 16), G = ceil(k / 128).

    codes uint8 [P, G, 4, 16, 16]: byte j of (p, g, b, r) holds the values 128 g + 32 b + 2 j (low half) and the next (high
    half) of row 16 p + r; scales uint8 [P, G, 16, 4]: byte b of (p, g, r) is the E8M0 byte of the values 128 g + 32 b .. + 31
    of that row.  Both are zero where there is no such row or value; the product relies on that of values past k, not of rows."""

    codes: torch.Tensor
    scales: torch.Tensor
    rows: int
    k: int


def _shapes(rows: int, k: int) -> tuple[tuple, tuple]:
    p, g = -(-rows // 16), -(-k // 128)
    return (p, g, 4, 16, 16), (p, g, 16, 4)


def _rows(x: torch.Tensor, name: str) -> tuple[torch.Tensor, int, int, int]:
    """(rows, R, K, row stride) of bf16 rows [R, K] (K % 32 == 0), as the kernels read them; a copy if their strides or address
    do not allow it."""
    if x.dim() != 2 or x.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be bf16 [rows, k], got {tuple(x.shape)} {x.dtype}")
    rows, k = x.shape
    if k % BLOCK:
        raise ValueError(f"{name} has rows of {k} values: not a multiple of {BLOCK}")
    ld, dense_values = x.stride()
    if rows <= 1:
        ld = k   # (one row has no stride)
    if rows and k and (dense_values != 1 or x.data_ptr() % 16 or ld % 8 or not k <= ld < 1 << 26):
        return dense(x), rows, k, k
    return x, rows, k, ld


def _ld(x: torch.Tensor) -> int:
    return x.stride(0) if x.shape[0] > 1 else x.shape[1]


def _operand(q: Mxfp4Rows, name: str) -> Mxfp4Rows:
    """q if its tensors are those of its rows and k."""
    codes, scales, rows, k = q
    if rows < 0 or k < 0 or k % BLOCK:
        raise ValueError(f"{name} has {rows} rows of {k} values: not a multiple of {BLOCK}")
    shape_c, shape_s = _shapes(rows, k)
    for what, t, shape in ("codes", codes, shape_c), ("scales", scales, shape_s):
        if t.shape != shape or t.dtype != torch.uint8 or not t.is_contiguous():
            raise ValueError(f"{name}'s {what} must be contiguous uint8 {shape} for {rows} rows of {k} values, got {tuple(t.shape)} {t.dtype}")
        if t.data_ptr() % 16:   # (0 where nothing is there)
            raise ValueError(f"{name}'s {what} must be 16-byte aligned")
    if scales.device != codes.device:
        raise ValueError(f"{name}'s codes are on {codes.device}, its scales on {scales.device}")
    return q


def _output(out: torch.Tensor | None, rows: int, cols: int, device, align: int) -> torch.Tensor:
    """A new bf16 [rows, cols], or the given one if the kernels can write it (row stride a multiple of ``align``)."""
    if out is None:
        return torch.empty((rows, cols), dtype=torch.bfloat16, device=device)
    if (tuple(out.shape) != (rows, cols) or out.dtype != torch.bfloat16 or out.device != device
            or (out.numel() and (out.stride(1) != 1 or out.data_ptr() % (2 * align)
                                 or (rows > 1 and (out.stride(0) % align or out.stride(0) < cols))))):
        raise ValueError(f"out must be bf16 [{rows}, {cols}] on {device} with dense rows whose stride {align} divides")
    return out


def quant_mxfp4(x: torch.Tensor) -> Mxfp4Rows:
    """bf16 rows [R, K], K % 32 == 0, quantized (wf_mxfp4_quant).

    Per block, s is the smallest power of two with max|x| < 7 s (2^-125 to 2^125), a code the nearest e2m1 number to x / s,
    an even code on a tie, at most 6.  A block that holds a NaN or an infinity reads back as NaN."""
    x, R, K, ld = _rows(x, "x")
    shape_c, shape_s = _shapes(R, K)
    device = x.device
    codes, scales = x.new_empty(shape_c, dtype=torch.uint8), x.new_empty(shape_s, dtype=torch.uint8)
    _lib.call_on(device, "wf_mxfp4_quant", x.data_ptr(), R, K, ld, codes.data_ptr(), scales.data_ptr())
    return Mxfp4Rows(codes, scales, R, K)


def dequant_mxfp4(codes: torch.Tensor, scales: torch.Tensor, rows: int, k: int, out: torch.Tensor | None = None) -> torch.Tensor:
    """The values of quantized rows (the fields of :class:`Mxfp4Rows`) as bf16 [rows, k], exact (wf_mxfp4_dequant)."""
    _operand(Mxfp4Rows(codes, scales, rows, k), "q")
    out = _output(out, rows, k, codes.device, 8)
    _lib.call_on(codes.device, "wf_mxfp4_dequant", codes.data_ptr(), scales.data_ptr(), rows, k, out.data_ptr(), _ld(out))
    return out


def to_rows(q: Mxfp4Rows) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes [rows, k / 2], E8M0 bytes [rows, k / 32]) of quantized rows."""
    codes, scales, rows, k = _operand(q, "q")
    codes = codes.permute(0, 3, 1, 2, 4).flatten(2).flatten(0, 1)
    scales = scales.transpose(1, 2).flatten(2).flatten(0, 1)
    return codes[:rows, :k // 2].contiguous(), scales[:rows, :k // BLOCK].contiguous()


def from_rows(codes: torch.Tensor, scales: torch.Tensor) -> Mxfp4Rows:
    """Codes uint8 [rows, k / 2] (the even value of a pair low) and E8M0 bytes uint8 [rows, k / 32] in the kernels' layout."""
    if codes.dim() != 2 or scales.dim() != 2 or codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"expected uint8 codes [rows, k / 2] and scales [rows, k / 32], got {tuple(codes.shape)} {codes.dtype} and "
                         f"{tuple(scales.shape)} {scales.dtype}")
    rows, k = codes.shape[0], 2 * codes.shape[1]
    if k % BLOCK or tuple(scales.shape) != (rows, k // BLOCK) or scales.device != codes.device:
        raise ValueError(f"codes of {rows} rows of {k} values on {codes.device} do not go with scales {tuple(scales.shape)} on {scales.device}")
    (p, g, *_), _ = _shapes(rows, k)
    wide_c, wide_s = codes.new_zeros((16 * p, 64 * g)), scales.new_zeros((16 * p, 4 * g))
    wide_c[:rows, :k // 2], wide_s[:rows, :k // BLOCK] = codes, scales
    return Mxfp4Rows(wide_c.view(p, 16, g, 4, 16).permute(0, 2, 3, 1, 4).contiguous(), wide_s.view(p, 16, g, 4).transpose(1, 2).contiguous(),
                     rows, k)


def _bias(bias: torch.Tensor | None, n: int, device) -> torch.Tensor | None:
    if bias is not None and (tuple(bias.shape) != (n,) or bias.dtype != torch.bfloat16 or bias.device != device
                             or not bias.is_contiguous() or bias.data_ptr() % 8):
        raise ValueError(f"bias must be contiguous bf16 [{n}] on {device}")
    return bias


def gemm_mxfp4(a: Mxfp4Rows, w: Mxfp4Rows, bias: torch.Tensor | None = None, gelu: bool = False,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """bf16 [M, N] = act(a [M, K] x w [N, K]^T + bias) of two quantized operands (wf_gemm_mxfp4): fp32 sums, act GELU(tanh)
    with ``gelu``, rounded once.  N must be a multiple of 4."""
    device = _operand(a, "a").codes.device
    if _operand(w, "w").k != a.k or w.codes.device != device:
        raise ValueError(f"a has rows of {a.k} values on {device}, w of {w.k} on {w.codes.device}")
    out = _output(out, a.rows, w.rows, device, 4)
    _lib.call_on(device, "wf_gemm_mxfp4", a.codes.data_ptr(), a.scales.data_ptr(), w.codes.data_ptr(), w.scales.data_ptr(), a.rows,
                 w.rows, a.k, _lib.ptr(_bias(bias, w.rows, device)), out.data_ptr(), _ld(out), _lib.GEMM_GELU_TANH if gelu else 0)
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
        n, k = weight.shape
        self._check_shape(n, k)
        self._take(quant_mxfp4(weight.detach().to(torch.bfloat16)), bias, gelu)

    @staticmethod
    def _check_shape(n: int, k: int) -> None:
        if k % BLOCK or n % 4 or not k:
            raise ValueError(f"unsupported linear shape {(n, k)} (in % {BLOCK}, out % 4 required)")

    @classmethod
    def from_quantized(cls, weight: Mxfp4Rows, bias: torch.Tensor | None = None, gelu: bool = False) -> "WaveMxfp4Linear":
        """A linear of a weight that is quantized already (:func:`quant_mxfp4`, or :func:`from_rows` of a checkpoint's)."""
        self = cls.__new__(cls)
        nn.Module.__init__(self)
        _operand(weight, "weight")
        cls._check_shape(weight.rows, weight.k)
        self._take(weight, bias, gelu)
        return self

    def _take(self, weight: Mxfp4Rows, bias, gelu) -> None:
        self.out_dtype = torch.bfloat16
        self.out_features, self.in_features = weight.rows, weight.k
        self.register_buffer("w_codes", weight.codes)
        self.register_buffer("w_scales", weight.scales)
        if bias is not None:
            bias = bias.detach().to(device=weight.codes.device, dtype=torch.bfloat16).contiguous()
            if tuple(bias.shape) != (self.out_features,):
                raise ValueError(f"bias has shape {tuple(bias.shape)}, the weight {self.out_features} rows")
            self.register_buffer("bias", bias.clone() if bias.data_ptr() % 8 else bias)   # (a view of a larger tensor: the kernels read 8 bytes)
        else:
            self.bias = None
        self.gelu = gelu

    @property
    def weight_rows(self) -> Mxfp4Rows:
        """The quantized weight."""
        return Mxfp4Rows(self.w_codes, self.w_scales, self.out_features, self.in_features)

    def _raw(self, x2: torch.Tensor) -> torch.Tensor:
        x2, M, K, ld = _rows(x2, "x")
        n, buffers = self.out_features, self._buffers   # (their own dict: a module's attributes cost a search each)
        w, bias, device = buffers["w_codes"], buffers.get("bias"), x2.device
        if K != self.in_features:
            raise ValueError(f"input width {K} != in_features {self.in_features}")
        if device != w.device:
            raise ValueError(f"x is on {device}, the weight on {w.device}")
        if bias is not None and bias.dtype != torch.bfloat16:
            raise ValueError(f"the bias has become {bias.dtype}: keep the module in bf16")
        y = torch.empty((M, n), dtype=torch.bfloat16, device=device)
        codes = scales = None
        if M > _lib.MXFP4_FUSED_ROWS:   # one workspace: the quantized rows' codes, then their scales
            panels = -(-M // 16) * -(-K // 128)
            ws = torch.empty((1088 * panels,), dtype=torch.uint8, device=device)
            codes = ws.data_ptr()
            scales = codes + 1024 * panels
        _lib.call_on(device, "wf_mxfp4_linear", x2.data_ptr(), M, K, ld, w.data_ptr(), buffers["w_scales"].data_ptr(),
                     None if bias is None else bias.data_ptr(), n, y.data_ptr(), n, _lib.GEMM_GELU_TANH if self.gelu else 0, codes, scales)
        return y

    def forward(self, x: torch.Tensor):
        if x.dim() == 2:
            return self._raw(x), None
        shape = x.shape
        return self._raw(x.reshape(-1, shape[-1])).view(*shape[:-1], self.out_features), None


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
