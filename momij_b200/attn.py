"""The attention half of a layer on an 8-bit paged cache (include/momij_moe.h):
head norms with rotation and append, attention over the cache, cache values.

A cache is pages of 64 tokens with one scale per page and kv head for K and one
for V; ``block_table[b, i]`` names the page of tokens ``64 i .. 64 i + 63`` of
sequence ``b``, and ``lens[b]`` counts its tokens *including* the ones that a call
appends or queries, so one pair of tensors serves every call of a step:

    cache = attn.new_kv_cache(n_pages, n_kv_heads, head_dim)
    rope = attn.rope_table(max_positions, rot_dim, theta)
    ws = attn.new_workspace(max_tokens, n_heads, head_dim)
    q = attn.qk_norm_rope_append(qkv, cache, block_table, lens, n_heads=Hq, q_weight=qw,
                                 k_weight=kw, eps=eps, rope=rope, workspace=ws)
    o = attn.attention(q, cache, block_table, lens, window=512, workspace=ws)
    moe.synchronize(workspace=ws)     # raises on a page, length or position out of range

Counterparts in momij: SeedlessMetal.swift:2794-3004, MapleFused.swift:260-325,
MapleAttention.swift, QuantProj.swift:24-172 (16-bit there).  Errors surface as
:class:`momij_b200.moe.SeedlessError`; arguments of a wrong type, shape or device
raise ``TypeError`` / ``ValueError`` before anything is enqueued.
"""
from __future__ import annotations

import ctypes
import importlib.machinery
import importlib.util
import os
from dataclasses import dataclass

import torch

from . import moe
from .moe import _check, lib

PAGE = 64  # MOMIJ_KV_PAGE
HEADER_BYTES = 256

lib.momij_attention_workspace_size.argtypes = [ctypes.c_int, ctypes.c_int]
lib.momij_attention_workspace_size.restype = ctypes.c_size_t


def _load_ops():
    """csrc/bind.cpp's module, given the addresses of this process's library."""
    path = os.path.join(moe.HERE, "lib", "_momij_ops.so")
    if not os.path.exists(path):
        raise ImportError(f"{path} is missing: build it with `python -m momij_b200.build`")
    loader = importlib.machinery.ExtensionFileLoader("_momij_ops", path)
    ops = importlib.util.module_from_spec(importlib.util.spec_from_loader("_momij_ops", loader))
    loader.exec_module(ops)
    ops.bind(_check, *(ctypes.cast(f, ctypes.c_void_p).value for f in (
        lib.momij_qk_norm_rope_append, lib.momij_cache_read, lib.momij_attention, lib.momij_qmm4, lib.momij_process_logits)))
    return ops


_ops = _load_ops()


@dataclass(frozen=True)
class KVCache:
    """Codes and scales of a paged cache (the layout of include/momij_moe.h):
    ``k`` uint8 [pages, Hkv, 64, D], ``v`` uint8 [pages, Hkv, D, 64], fp32 scales [pages, Hkv]."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    def __post_init__(self):
        P, H, page, D = self.k.shape
        if page != PAGE or tuple(self.v.shape) != (P, H, D, PAGE):
            raise ValueError(f"k is [pages, Hkv, {PAGE}, D] and v [pages, Hkv, D, {PAGE}]")
        if tuple(self.k_scale.shape) != (P, H) or tuple(self.v_scale.shape) != (P, H):
            raise ValueError("scales are [pages, Hkv]")
        if self.k.dtype != torch.uint8 or self.v.dtype != torch.uint8:
            raise TypeError("codes are uint8")
        if self.k_scale.dtype != torch.float32 or self.v_scale.dtype != torch.float32:
            raise TypeError("scales are float32")
        for t in (self.k, self.v, self.k_scale, self.v_scale):
            if not t.is_cuda or t.device != self.k.device:
                raise ValueError("a cache lies on one CUDA device")
            if not t.is_contiguous():
                raise ValueError("cache tensors must be contiguous")


def new_kv_cache(n_pages: int, n_kv_heads: int, head_dim: int, device=None) -> KVCache:
    """An empty cache (zero scales)."""
    dev = device or "cuda"
    return KVCache(torch.full((n_pages, n_kv_heads, PAGE, head_dim), 128, dtype=torch.uint8, device=dev),
                   torch.full((n_pages, n_kv_heads, head_dim, PAGE), 128, dtype=torch.uint8, device=dev),
                   torch.zeros(n_pages, n_kv_heads, device=dev), torch.zeros(n_pages, n_kv_heads, device=dev))


def rope_table(positions: int, rot_dim: int, theta: float = 10_000.0, device=None) -> torch.Tensor:
    """[positions, rot_dim] fp32: cosines, then sines, of position * theta^(-2i/rot_dim),
    computed in 64 bits (an fp32 angle is off by 2^-24 of the position)."""
    half = rot_dim // 2
    angle = (torch.arange(positions, dtype=torch.float64)[:, None]
             * theta ** (-torch.arange(half, dtype=torch.float64) / half))
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device or "cuda")


def workspace_size(n_tokens: int, n_heads: int) -> int:
    return int(lib.momij_attention_workspace_size(n_tokens, n_heads))


def new_workspace(n_tokens: int, n_heads: int, head_dim: int = 128, device=None) -> torch.Tensor:
    """Zero-filled workspace for calls of up to ``n_tokens`` query tokens (the
    kernels keep it reusable; one per stream)."""
    return torch.zeros(max(workspace_size(n_tokens, n_heads), HEADER_BYTES), dtype=torch.uint8, device=device or "cuda")


def _on(stream, call, *args, **kwargs):
    """A call with a stream of the caller's current: what it allocates and fills is
    ordered with the kernel, and results are held until the stream that was current is
    done with them, too.  (The operators check for None themselves, and give their
    arguments one by one: a closure over them, or a call more, is 5 % of a small
    operator's time.)"""
    before = torch.cuda.current_stream()
    if not isinstance(stream, torch.cuda.Stream):  # a handle; 0 is the default stream's
        stream = torch.cuda.ExternalStream(int(stream)) if int(stream) else torch.cuda.default_stream()
    with torch.cuda.stream(stream):
        out = call(*args, **kwargs)
    for t in out if isinstance(out, tuple) else (out,):
        t.record_stream(before)
    return out


def qk_norm_rope_append(qkv: torch.Tensor, cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, *, n_heads: int,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                        rope: torch.Tensor | None = None, interleaved: bool = False, cu_q: torch.Tensor | None = None,
                        max_q: int = 0, q_out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                        stream=None) -> torch.Tensor:
    """Norms queries and keys per head, rotates them by position and appends keys
    and values to the cache (momij_qk_norm_rope_append).  ``qkv`` [T, (Hq + 2 Hkv) D]
    (rows may be strided); returns the queries [T, Hq, D]."""
    if stream is not None:
        return _on(stream, qk_norm_rope_append, qkv, cache, block_table, lens, n_heads=n_heads, q_weight=q_weight, k_weight=k_weight,
                   eps=eps, rope=rope, interleaved=interleaved, cu_q=cu_q, max_q=max_q, q_out=q_out, workspace=workspace)
    return _ops.append(qkv, cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, lens, n_heads, q_weight, k_weight, eps,
                       rope, interleaved, cu_q, max_q, q_out, workspace)


def cache_read(cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, *, count: int, first: torch.Tensor | None = None,
               dtype=torch.bfloat16, workspace: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of ``count`` tokens per sequence from ``first[b]`` on (default 0),
    [B, count, Hkv, D]; zeros at and past ``lens[b]``."""
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"values are bf16 or fp16, not {dtype}")
    if stream is not None:
        return _on(stream, cache_read, cache, block_table, lens, count=count, first=first, dtype=dtype, workspace=workspace)
    return _ops.read(cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, lens, first, count, dtype == torch.float16, workspace)


def attention(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, *, scale: float | None = None,
              window: int = 0, cu_q: torch.Tensor | None = None, max_q: int = 0, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal attention of the new tokens' queries ``q`` [T, Hq, D] over the cache
    (momij_attention); ``scale`` defaults to D^-1/2, ``window`` 0 means all positions.
    Token rows of ``q`` and ``out`` may be strided.  Without a workspace the call makes
    one of its own, and nothing reports a page or length out of range."""
    if stream is not None:
        return _on(stream, attention, q, cache, block_table, lens, scale=scale, window=window, cu_q=cu_q, max_q=max_q, out=out,
                   workspace=workspace)
    if workspace is None:  # (with one, the call itself looks at q)
        if not isinstance(q, torch.Tensor):
            raise TypeError("q is a tensor")
        if q.dim() != 3:
            raise ValueError("q is [T, Hq, D]")
        workspace = new_workspace(q.shape[0], q.shape[1], device=q.device)
    return _ops.attention(q, cache.k, cache.v, cache.k_scale, cache.v_scale, block_table, lens, scale, window, cu_q, max_q, out, workspace)
