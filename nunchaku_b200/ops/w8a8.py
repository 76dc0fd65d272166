"""The 8-bit path: 16-bit rows -> int8 codes with one scale per token (optionally behind a residual addition and an RMSNorm), and
the int8 GEMM with a scale per token and per output channel.

Counterparts in the reference: ``quantize_w8a8_act`` and ``gemm_w8a8`` (src/kernels/zgemm/gemm_w8a8.cu), there with 16-bit scales.
Forward only, as the rest of the package.
"""
from __future__ import annotations

import torch

from .. import _lib
from ..utils import HALF_DTYPES, dtype_code, launch


def _rows(name: str, t: torch.Tensor, cols: int) -> tuple[int, int]:
    """(number of rows, row stride) of ``t`` [..., cols] as a 2-D matrix; raises when its rows have no common stride."""
    if t.is_contiguous():
        return t.numel() // cols, cols
    if t.stride(-1) == 1 or cols == 1:
        rows, stride = 1, None
        for size, st in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
            if size == 1:
                continue
            if stride is None:
                stride = st
            elif st != stride * rows:
                break
            rows *= size
        else:
            stride = cols if stride is None else stride
            if stride >= cols and stride % 8 == 0:
                return rows, stride
    raise ValueError(f"{name} must be rows of contiguous columns, one row stride (a multiple of 8 elements) apart")


def _check_half(name: str, t: torch.Tensor, like: torch.Tensor | None = None) -> None:
    if not t.is_cuda or t.dtype not in HALF_DTYPES:
        raise ValueError(f"{name} must be a CUDA bf16 / fp16 tensor (this library has no CPU path)")
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError(f"{name} must have x's dtype and device")


def _quantize(x, weight, residual, eps):
    _check_half("x", x)
    shape = x.shape
    cols = shape[-1] if shape else 0
    n = x.numel()
    if n == 0 or cols % 16 or cols > 2**30:
        raise ValueError("x must be [..., C] with at least one row and C a positive multiple of 16 (up to 16384)")
    dev = x.device
    if x.is_contiguous():
        rows, x_stride = n // cols, cols
        codes = torch.empty_like(x, dtype=torch.int8)
    else:
        rows, x_stride = _rows("x", x, cols)
        codes = torch.empty(shape, dtype=torch.int8, device=dev)
    scales = torch.empty_strided((rows,), (1,), dtype=torch.float32, device=dev)
    if len(shape) != 2:
        scales = scales.view(shape[:-1])
    hidden = None
    hidden_ptr = res_ptr = weight_ptr = res_stride = 0
    if weight is not None:
        _check_half("weight", weight, x)
        if weight.shape != (cols,) or not weight.is_contiguous():
            raise ValueError("weight must be a contiguous [C]")
        weight_ptr = weight.data_ptr()
    if residual is not None:
        _check_half("residual", residual, x)
        if residual.shape != shape:
            raise ValueError("residual must have x's shape")
        res_stride = cols if residual.is_contiguous() else _rows("residual", residual, cols)[1]
        hidden = torch.empty_like(x, memory_format=torch.contiguous_format)
        res_ptr, hidden_ptr = residual.data_ptr(), hidden.data_ptr()
    launch(_lib.load().svdq_quantize_w8a8,
           _lib.pack_quantize_w8a8(x.data_ptr(), res_ptr, weight_ptr, codes.data_ptr(), scales.data_ptr(), hidden_ptr, rows, x_stride, res_stride,
                                 cols, eps, dtype_code(x.dtype)), dev)
    return codes, scales, hidden


def quantize_w8a8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Symmetric 8-bit codes of bf16 / fp16 ``x`` [..., C] with one scale per row: ``scale = max|x| / 127``, ``code = rint(x / scale)``.
    Returns (codes int8 like x, scales fp32 [...]).  For activations (one scale per token) and for weights [N, K] (one per output
    channel) alike.  C: a multiple of 16 up to 16384; the rows of x may be strided.  A row of zeros has scale 0; a row with a NaN or an
    infinity has scale NaN (and codes 0)."""
    codes, scales, _ = _quantize(x, None, None, 0.0)
    return codes, scales


def rms_norm_quantize_w8a8(x: torch.Tensor, weight: torch.Tensor, residual: torch.Tensor | None = None,
                           eps: float = 1e-6) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """``quantize_w8a8(rms_norm(x + residual) * weight)`` in one pass: h = x (+ residual), y = h / sqrt(mean(h^2) + eps) * weight.

    x, residual: bf16 or fp16 [..., C] (rows may be strided), weight [C] of the same dtype.  Returns (codes int8 like x, scales fp32
    [...], hidden): hidden = x + residual rounded to x's dtype (the residual stream; fp16 saturates), None without a residual.  The norm
    works on the fp32 sum.  eps: at least 1e-30.  A row whose sum of squares is not finite has scale NaN (and codes 0)."""
    if weight is None:
        raise ValueError("weight is required (quantize_w8a8 is the form without the norm)")
    if not eps >= 1e-30:
        raise ValueError("eps must be at least 1e-30")
    return _quantize(x, weight, residual, eps)


def dequantize_w8a8(codes: torch.Tensor, scales: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values codes stand for: ``codes * scales[..., None]`` rounded once to ``out_dtype`` (bf16 or fp16), for int8 ``codes`` [..., C]
    (C a multiple of 16) and fp32 ``scales`` [...], both contiguous."""
    if not codes.is_cuda or codes.dtype != torch.int8 or not codes.is_contiguous():
        raise ValueError("codes must be a contiguous CUDA int8 tensor")
    if scales.dtype != torch.float32 or scales.device != codes.device or not scales.is_contiguous():
        raise ValueError("scales must be a contiguous fp32 tensor on codes' device")
    cols = codes.shape[-1] if codes.dim() else 0
    if codes.numel() == 0 or cols % 16 or cols > 2**30 or scales.shape != codes.shape[:-1]:
        raise ValueError("codes must be [..., C] with at least one row and C a positive multiple of 16, scales [...]")
    code = dtype_code(out_dtype)
    out = torch.empty_like(codes, dtype=out_dtype)
    launch(_lib.load().svdq_dequantize_w8a8,
           _lib.pack_dequantize_w8a8(codes.data_ptr(), scales.data_ptr(), out.data_ptr(), codes.numel() // cols, cols, code), codes.device)
    return out


def gemm_w8a8(act: torch.Tensor, wgt: torch.Tensor, ascales: torch.Tensor, wscales: torch.Tensor, bias: torch.Tensor | None = None,
              out: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``(act @ wgt.T) * ascales[:, None] * wscales (+ bias)`` for int8 ``act`` [..., K] and ``wgt`` [N, K], fp32 ``ascales`` [...] (one
    per token) and ``wscales`` [N].  The integer sum is exact; scales and bias are applied in fp32 with one rounding to the output's type.

    K: a multiple of 16 up to 131056; N: a multiple of 8; 1 to 2**30 rows.  ``out`` [..., N] bf16 / fp16 may be rows of a
    wider buffer (unit column stride, one row stride that is a multiple of 8); by default a new tensor of ``out_dtype`` (bias's dtype,
    else bf16)."""
    dev = act.device
    if not act.is_cuda or act.dtype != torch.int8 or wgt.dtype != torch.int8 or not act.is_contiguous() or not wgt.is_contiguous():
        raise ValueError("act and wgt must be contiguous CUDA int8 tensors")
    if ascales.dtype != torch.float32 or wscales.dtype != torch.float32 or not ascales.is_contiguous() or not wscales.is_contiguous():
        raise ValueError("ascales and wscales must be contiguous fp32 tensors")
    if wgt.device != dev or ascales.device != dev or wscales.device != dev:
        raise ValueError("all tensors must be on act's device")
    shape = act.shape
    if wgt.dim() != 2 or not shape or shape[-1] != wgt.shape[1] or act.numel() == 0:
        raise ValueError("act must be [..., K] with at least one row and wgt [N, K]")
    N, K = wgt.shape
    lead = shape[:-1]
    if ascales.shape != lead or wscales.shape != (N,):
        raise ValueError("ascales must be act's shape without K and wscales [N]")
    if out is not None:
        if out.shape != (*lead, N) or out.device != dev or (out_dtype is not None and out.dtype != out_dtype):
            raise ValueError("out must be [..., N] on act's device (of out_dtype, where that is given)")
        dtype = out.dtype
    else:
        dtype = out_dtype if out_dtype is not None else bias.dtype if bias is not None else torch.bfloat16
    code = dtype_code(dtype)
    if bias is not None and (bias.shape != (N,) or bias.dtype != dtype or not bias.is_contiguous() or bias.device != dev):
        raise ValueError("bias must be a contiguous [N] of the output's dtype on act's device")
    rows = act.numel() // K
    if max(rows, N, K) > 2**30:
        raise ValueError("gemm_w8a8: at most 2**30 rows and columns")
    if out is None:
        out = torch.empty_strided((rows, N), (N, 1), dtype=dtype, device=dev)
        if len(shape) != 2:
            out = out.view(*lead, N)
        stride = N
    else:
        stride = _rows("out", out, N)[1]
    launch(_lib.load().svdq_gemm_w8a8,
           _lib.pack_gemm_w8a8(act.data_ptr(), wgt.data_ptr(), ascales.data_ptr(), wscales.data_ptr(), 0 if bias is None else bias.data_ptr(),
                             out.data_ptr(), stride, rows, N, K, code), dev)
    return out
