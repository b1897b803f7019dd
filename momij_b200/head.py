"""4-bit projections and logits (include/momij_moe.h): ``qmm4`` for a few tokens
against a matrix of 4-bit codes with group scales (the vocabulary projection, or
attention's projections), and ``process_logits`` for penalties, biases and
grammar masks before sampling.

Counterparts in momij: SeedlessMetal.swift:2598-2716, QuantProj.swift,
LogitsProcessor.swift, XGrammarGuide.swift.  Errors surface as
:class:`momij_b200.moe.SeedlessError`; arguments of a wrong type, shape or device
raise ``TypeError`` / ``ValueError``.
"""
from __future__ import annotations

import ctypes

import torch

from .attn import _ints, _keep, _on, _raw_stream
from .moe import DTYPE_BF16, DTYPE_F16, _check, lib

DTYPE_F32 = 2

_vp, _i, _ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong
lib.momij_qmm4.argtypes = [_vp, _ll, _vp, _vp, _vp, _vp, _ll] + [_i] * 5 + [_vp]
lib.momij_process_logits.argtypes = ([_vp, _ll, _i, _vp, _i, _i, _vp, _vp, _i] + [_vp] * 6 + [_i, _vp, _ll, _vp])

_CODES = {torch.bfloat16: DTYPE_BF16, torch.float16: DTYPE_F16, torch.float32: DTYPE_F32}


def qmm4(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *, gs: int = 64,
         out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """``out`` [M, N] = x [M, K] times the transpose of the 4-bit matrix ``w`` int32/uint32
    [N, K/8] (code k of a word at bits 4k .. 4k+3) with ``scales``, ``biases`` [N, K/gs].
    Rows of ``x`` and ``out`` may be strided."""
    dev = x.device
    index = _on(dev, w, scales, biases, out)
    M, K = x.shape
    N = w.shape[0]
    dt = x.dtype
    if dt != torch.bfloat16 and dt != torch.float16:
        raise TypeError(f"activations must be bf16 or fp16, got {dt}")
    if scales.dtype != dt or biases.dtype != dt:
        raise TypeError("scales and biases have the activations' dtype")
    if w.dtype != torch.int32 and w.dtype != torch.uint32:
        raise TypeError("codes are packed in 32-bit words")
    if x.stride(1) != 1 and K > 1:
        raise ValueError("rows of x must be contiguous")
    if (tuple(w.shape) != (N, K // 8) or tuple(scales.shape) != (N, K // gs) or scales.shape != biases.shape
            or not (w.is_contiguous() and scales.is_contiguous() and biases.is_contiguous())):
        raise ValueError("w is [N, K/8], scales and biases [N, K/gs], contiguous")
    if out is None:
        out = torch.empty(M, N, dtype=dt, device=dev)
        _keep(out, stream)
    elif tuple(out.shape) != (M, N) or out.dtype != dt or (N > 1 and out.stride(1) != 1):
        raise ValueError("out is [M, N] of the activations' dtype with contiguous rows")
    _check(lib.momij_qmm4(x.data_ptr(), x.stride(0) if M > 1 else K, w.data_ptr(), scales.data_ptr(), biases.data_ptr(),
                          out.data_ptr(), out.stride(0) if M > 1 else N, M, K, N, gs, _CODES[dt], _raw_stream(stream, index)),
           "qmm4")
    return out


def _rows(t: torch.Tensor | None, name: str, B: int) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.float32 or tuple(t.shape) != (B,) or not t.is_contiguous():
        raise ValueError(f"{name} is a contiguous float32 tensor [{B}]")
    return t.data_ptr()


def process_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, cu_history: torch.Tensor | None = None,
                   repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, cu_bias: torch.Tensor | None = None,
                   allowed: torch.Tensor | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """fp32 [B, V]: ``logits`` with penalties over each row's ``history`` (ids of all rows,
    offsets ``cu_history`` [B+1]), the biases of ``bias_ids`` / ``cu_bias`` and -inf where
    ``allowed`` (int32 [B, ceil(V/32)], bit v%32 of word v//32) has a zero bit.
    ``out`` may be ``logits`` itself where that is fp32."""
    dev = logits.device
    index = _on(dev, history, cu_history, repetition, presence, frequency, bias_ids, bias, cu_bias, allowed, out)
    B, V = logits.shape
    if logits.dtype not in _CODES:
        raise TypeError(f"logits are bf16, fp16 or fp32, got {logits.dtype}")
    if logits.stride(1) != 1 and V > 1:
        raise ValueError("rows of the logits must be contiguous")
    if (history is None) != (cu_history is None):
        raise ValueError("history and cu_history go together")
    if (bias_ids is None) != (cu_bias is None) or (bias_ids is None) != (bias is None):
        raise ValueError("bias_ids, bias and cu_bias go together")
    nh = 0 if history is None else history.numel()
    nb = 0 if bias_ids is None else bias_ids.numel()
    if allowed is not None and (allowed.dtype != torch.int32 or tuple(allowed.shape) != (B, (V + 31) // 32)
                                or (allowed.shape[1] > 1 and allowed.stride(1) != 1)):
        raise ValueError("allowed is int32 [B, ceil(V/32)] with contiguous rows")
    if out is None:
        out = torch.empty(B, V, dtype=torch.float32, device=dev)
        _keep(out, stream)
    elif tuple(out.shape) != (B, V) or out.dtype != torch.float32 or not out.is_contiguous():
        raise ValueError("out is a contiguous float32 [B, V] tensor")
    _check(lib.momij_process_logits(
        logits.data_ptr(), logits.stride(0) if B > 1 else V, _CODES[logits.dtype], out.data_ptr(), B, V,
        _ints(history, "history", (nh,)), _ints(cu_history, "cu_history", (B + 1,)), nh, _rows(repetition, "repetition", B),
        _rows(presence, "presence", B), _rows(frequency, "frequency", B), _ints(bias_ids, "bias_ids", (nb,)),
        _rows(bias, "bias", nb), _ints(cu_bias, "cu_bias", (B + 1,)), nb, None if allowed is None else allowed.data_ptr(),
        (allowed.stride(0) if B > 1 else allowed.shape[1]) if allowed is not None else 0, _raw_stream(stream, index)),
        "processLogits")
    return out
