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

import torch

from .attn import _on, _ops


def qmm4(x: torch.Tensor, w: torch.Tensor, scales: torch.Tensor, biases: torch.Tensor, *, gs: int = 64,
         out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """``out`` [M, N] = x [M, K] times the transpose of the 4-bit matrix ``w`` int32/uint32
    [N, K/8] (code k of a word at bits 4k .. 4k+3) with ``scales``, ``biases`` [N, K/gs].
    Rows of ``x`` and ``out`` may be strided."""
    if stream is not None:
        return _on(stream, qmm4, x, w, scales, biases, gs=gs, out=out)
    return _ops.qmm4(x, w, scales, biases, gs, out)


def process_logits(logits: torch.Tensor, *, history: torch.Tensor | None = None, cu_history: torch.Tensor | None = None,
                   repetition: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, bias_ids: torch.Tensor | None = None,
                   bias: torch.Tensor | None = None, cu_bias: torch.Tensor | None = None,
                   allowed: torch.Tensor | None = None, out: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """fp32 [B, V]: ``logits`` with penalties over each row's ``history`` (ids of all rows,
    offsets ``cu_history`` [B+1]), the biases of ``bias_ids`` / ``cu_bias`` and -inf where
    ``allowed`` (int32 [B, ceil(V/32)], bit v%32 of word v//32) has a zero bit.
    ``out`` may be ``logits`` itself where that is fp32."""
    if stream is not None:
        return _on(stream, process_logits, logits, history=history, cu_history=cu_history, repetition=repetition, presence=presence,
                   frequency=frequency, bias_ids=bias_ids, bias=bias, cu_bias=cu_bias, allowed=allowed, out=out)
    return _ops.logits(logits, history, cu_history, repetition, presence, frequency, bias_ids, bias, cu_bias, allowed, out)
