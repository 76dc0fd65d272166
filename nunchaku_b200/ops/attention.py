"""Softmax attention for 128-wide heads on the tcgen05 kernel of ``csrc/attention.cu``.

Mirrors ``nunchaku::ops::attention_fp16`` (nunchaku/csrc/ops.h:112-118, kernel src/kernels/zgemm/attention.cu:10-96; called
from nunchaku/models/attention_processors/flux.py:160-185).
"""
from __future__ import annotations

import ctypes

import torch

from .. import _lib
from ..utils import HALF_DTYPES, dtype_code, launch, on_device, stream_ptr

HEAD_DIM = 128


def _strides(name: str, t: torch.Tensor) -> tuple[int, int, int]:
    if t.dim() != 4 or t.shape[3] != HEAD_DIM or t.stride(3) != 1:
        raise ValueError(f"{name} must be [batch, heads, tokens, {HEAD_DIM}] (any strides, the last dimension contiguous)")
    s = [t.stride(0), t.stride(1), t.stride(2)]
    if t.shape[0] == 1:
        s[0] = 0
    if any(x % 8 for x in s) or t.data_ptr() % 16:
        raise ValueError(f"{name}: strides must be multiples of 8 elements and the data 16-byte aligned")
    return tuple(s)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, out: torch.Tensor | None = None,
              scale: float | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` per (batch, head).

    q: [B, H, Tq, 128]; k, v: [B, H, Tkv, 128], bf16 or fp16, as views with any (batch, head, token) strides: the reference's
    packed head-major tensors and token-major ``x.view(B, T, H, 128).transpose(1, 2)`` views are both taken as they are.
    out: [B, Tq, H*128] (default: a new tensor) or a [B, H, Tq, 128] view of one.  scale defaults to 128 ** -0.5."""
    for n, t in (("q", q), ("k", k), ("v", v)):
        if not t.is_cuda or t.dtype not in HALF_DTYPES or t.dtype != q.dtype:
            raise ValueError(f"{n} must be a CUDA bf16 / fp16 tensor of q's dtype")
    B, H, Tq, _ = q.shape
    if k.shape != v.shape or k.shape[0] != B or k.shape[1] != H:
        raise ValueError("k and v must be [batch, heads, tokens_kv, 128] with q's batch and heads")
    ret = out
    if out is None:
        ret = out = torch.empty(B, Tq, H * HEAD_DIM, dtype=q.dtype, device=q.device)
    if out.dim() == 3:
        if out.shape != (B, Tq, H * HEAD_DIM) or out.stride(2) != 1:
            raise ValueError("out must be [batch, tokens_q, heads*128] with unit channel stride")
        out = out.unflatten(2, (H, HEAD_DIM)).transpose(1, 2)
    if out.shape != q.shape or out.dtype != q.dtype or not out.is_cuda:
        raise ValueError("out must match q's shape (as [B, H, Tq, 128]) and dtype")
    args = _lib.AttentionArgs(q=q.data_ptr(), k=k.data_ptr(), v=v.data_ptr(), out=out.data_ptr(),
                              q_stride=(ctypes.c_int64 * 3)(*_strides("q", q)), k_stride=(ctypes.c_int64 * 3)(*_strides("k", k)),
                              v_stride=(ctypes.c_int64 * 3)(*_strides("v", v)), o_stride=(ctypes.c_int64 * 3)(*_strides("out", out)),
                              batch=B, heads=H, q_len=Tq, kv_len=k.shape[2], head_dim=HEAD_DIM,
                              scale=float(HEAD_DIM ** -0.5 if scale is None else scale), dtype=dtype_code(q.dtype))
    with on_device(q.device):
        _lib.check(_lib.load().svdq_attention(ctypes.byref(args), stream_ptr(q.device)))
    return ret


def attention_fp16(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, o: torch.Tensor, scale: float) -> None:
    """The reference's call (nunchaku/csrc/ops.h:112-118): q, k, v packed [B, H, T, 128], o [B, Tq, H*128], written in place.
    The reference takes fp16 inputs with a bf16 or fp16 output; here all four share one 16-bit type."""
    attention(q, k, v, out=o, scale=scale)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_lens: torch.Tensor | None = None,
                    mask: torch.Tensor | None = None, kv_offsets: torch.Tensor | None = None, out: torch.Tensor | None = None,
                    scale: float | None = None) -> torch.Tensor:
    """``softmax(scale * q k^T) v`` of queries over an encoder's states of another length (``MultiHeadCrossAttention``,
    src/SanaModel.cpp:138-190), over the states that exist for each sample.

    q: [B, H, Tq, D]; k, v: [B, Hk, T, D] views with any (batch, head, token) strides (multiples of 8 elements; batch and head may be
    expanded), bf16 or fp16, D a multiple of 8 up to 128, H a multiple of Hk (query head h reads stored head h // (H // Hk)).
    Which states exist, at most one of: ``kv_lens`` int32 [B] (the first so many of each sample), ``mask`` bool [B, T] (those that are
    True; T up to 32768), ``kv_offsets`` int32 [B + 1] (k and v are then packed [total, Hk, D], sample b owning rows
    ``kv_offsets[b]:kv_offsets[b + 1]``); all on q's device, read there (lengths outside 0..T are clamped).  None: all T.  A sample without
    states gets zeros; states that do not exist may hold anything, NaN included.  With k and v longer than 2**22, Tq * H / Hk is at most
    2**20 - 16.
    out: [B, Tq, H*D] (default: a new tensor) or a [B, H, Tq, D] view of one.  scale defaults to D ** -0.5 and must be positive."""
    dtype, dev = q.dtype, q.device
    if not q.is_cuda or dtype not in HALF_DTYPES:
        raise ValueError("q must be a CUDA bf16 / fp16 tensor (this library has no CPU path)")
    if k.dtype != dtype or v.dtype != dtype or k.device != dev or v.device != dev:
        raise ValueError("k and v must have q's dtype and device")
    if q.dim() != 4:
        raise ValueError("q must be [batch, heads, tokens, D]")
    B, H, Tq, D = q.shape
    if (kv_lens is not None) + (mask is not None) + (kv_offsets is not None) > 1:
        raise ValueError("at most one of kv_lens, mask and kv_offsets")
    if k.shape != v.shape:
        raise ValueError("k and v must have the same shape")
    lens_ptr = off_ptr = mask_ptr = mask_stride = 0
    if kv_offsets is not None:
        if k.dim() != 3 or k.shape[2] != D:
            raise ValueError("with kv_offsets, k and v are packed [total, kv_heads, D]")
        T, Hk = k.shape[0], k.shape[1]
        kst, vst = k.stride(), v.stride()
        ks, vs = (0, kst[1], kst[0]), (0, vst[1], vst[0])
        if kv_offsets.dtype != torch.int32 or kv_offsets.device != dev or kv_offsets.shape != (B + 1,) or not kv_offsets.is_contiguous():
            raise ValueError("kv_offsets must be a contiguous int32 [batch + 1] on q's device")
        off_ptr = kv_offsets.data_ptr()
    else:
        if k.dim() != 4 or k.shape[0] != B or k.shape[3] != D:
            raise ValueError("k and v must be [batch, kv_heads, tokens, D] with q's batch and D")
        Hk, T = k.shape[1], k.shape[2]
        kst, vst = k.stride(), v.stride()
        ks, vs = kst[:3], vst[:3]
        if kv_lens is not None:
            if kv_lens.dtype != torch.int32 or kv_lens.device != dev or kv_lens.shape != (B,) or not kv_lens.is_contiguous():
                raise ValueError("kv_lens must be a contiguous int32 [batch] on q's device")
            lens_ptr = kv_lens.data_ptr()
        elif mask is not None:
            if mask.dtype != torch.bool or mask.device != dev or mask.shape != (B, T) or (mask.stride(1) != 1 and T > 1):
                raise ValueError("mask must be bool [batch, tokens] on q's device with unit token stride")
            mask_ptr, mask_stride = mask.data_ptr(), mask.stride(0)
    qs = q.stride()
    if qs[3] != 1 or kst[-1] != 1 or vst[-1] != 1:
        raise ValueError("the last dimension of q, k and v must be contiguous")
    if min(B, H, Tq, D, Hk, T) == 0:
        raise ValueError("cross_attention: empty tensors (where no sample has states, k and v still need one row, of any content)")
    if max(B, H, Tq, T, D) > 2**30:
        raise ValueError("cross_attention: at most 2**30 samples, heads and tokens")
    ret = out
    if out is None:
        C = H * D
        ret = torch.empty_strided((B, Tq, C), (Tq * C, C, 1), dtype=dtype, device=dev)
        os = (Tq * C, D, C)
    else:
        if out.dtype != dtype or out.device != dev:
            raise ValueError("out must have q's dtype and device")
        if out.dim() == 3:
            if out.shape != (B, Tq, H * D) or out.stride(2) != 1:
                raise ValueError("out must be [batch, tokens_q, heads*D] with unit channel stride")
            os = (out.stride(0), D, out.stride(1))
        else:
            if out.shape != q.shape or out.stride(3) != 1:
                raise ValueError("out must be [batch, tokens_q, heads*D] or [batch, heads, tokens_q, D]")
            os = out.stride()[:3]
    args = _lib.pack_cross_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), ret.data_ptr(), *qs[:3], *ks, *vs, *os, lens_ptr, off_ptr, mask_ptr, mask_stride,
                                   B, H, Hk, Tq, T, D, float(D ** -0.5 if scale is None else scale), dtype_code(dtype))
    launch(_lib.load().svdq_cross_attention, args, dev)
    return ret
