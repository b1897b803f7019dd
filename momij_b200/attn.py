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
from dataclasses import dataclass

import torch

from . import moe
from .moe import _check, _dtype_code, lib

PAGE = 64  # MOMIJ_KV_PAGE
HEADER_BYTES = 256

_vp, _i, _f, _sz, _ll = ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t, ctypes.c_longlong
lib.momij_qk_norm_rope_append.argtypes = ([_vp, _ll, _vp, _vp, _vp, _f, _vp, _i, _i, _i] + [_vp] * 4 + [_i, _vp, _i, _vp, _vp]
                                          + [_i] * 7 + [_vp, _sz, _vp])
lib.momij_cache_read.argtypes = [_vp] * 4 + [_i, _vp, _i, _vp, _vp, _i, _vp, _vp] + [_i] * 4 + [_vp, _sz, _vp]
lib.momij_attention_workspace_size.argtypes = [_i, _i]
lib.momij_attention_workspace_size.restype = _sz
lib.momij_attention.argtypes = ([_vp, _ll, _vp, _ll] + [_vp] * 4 + [_i, _vp, _i, _vp, _vp] + [_i] * 6 + [_f, _i, _i]
                                + [_vp, _sz, _vp])


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
        ptrs = (self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr())
        object.__setattr__(self, "_ptrs", ptrs)
        object.__setattr__(self, "_dims", (P, H, D, self.k.device))


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


def _on(device: torch.device, *tensors) -> int:
    """Refuses tensors on another device than the current one; its index."""
    cur = torch.cuda.current_device()
    if device.index != cur:
        raise ValueError(f"tensors on {device}, current device cuda:{cur}")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"tensors on {t.device} and {device}")
    return cur


def _raw_stream(stream, index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(index) if stream is None else moe._stream(stream)


def _ints(t: torch.Tensor | None, name: str, shape) -> int | None:
    if t is None:
        return None
    if t.dtype != torch.int32:
        raise TypeError(f"{name} is int32")
    if tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{name} is a contiguous tensor of shape {shape}")
    return t.data_ptr()


def _table(block_table: torch.Tensor, B: int) -> int:
    if block_table.dtype != torch.int32:
        raise TypeError("block_table is int32")
    if block_table.dim() != 2 or block_table.shape[0] != B or not block_table.is_contiguous():
        raise ValueError("block_table is a contiguous [B, columns] tensor")
    return block_table.data_ptr()


def _keep(t: torch.Tensor, stream) -> None:
    """A tensor allocated here and used on a stream given by the caller stays
    allocated until that stream is done with it."""
    if isinstance(stream, torch.cuda.Stream):
        t.record_stream(stream)


def qk_norm_rope_append(qkv: torch.Tensor, cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, *, n_heads: int,
                        q_weight: torch.Tensor | None = None, k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                        rope: torch.Tensor | None = None, interleaved: bool = False, cu_q: torch.Tensor | None = None,
                        max_q: int = 0, q_out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                        stream=None) -> torch.Tensor:
    """Norms queries and keys per head, rotates them by position and appends keys
    and values to the cache (momij_qk_norm_rope_append).  ``qkv`` [T, (Hq + 2 Hkv) D]
    (rows may be strided); returns the queries [T, Hq, D]."""
    P, Hkv, D, dev = cache._dims
    index = _on(dev, qkv, block_table, lens, q_weight, k_weight, rope, cu_q, q_out, workspace)
    T, width = qkv.shape
    B = lens.shape[0]
    if width != (n_heads + 2 * Hkv) * D or (T > 1 and qkv.stride(0) < width) or qkv.stride(1) != 1:
        raise ValueError(f"qkv is [T, {(n_heads + 2 * Hkv) * D}] with contiguous rows")
    for w in (q_weight, k_weight):
        if w is not None and (w.dtype != qkv.dtype or tuple(w.shape) != (D,) or not w.is_contiguous()):
            raise ValueError(f"norm weights are contiguous [{D}] of the activations' dtype")
    rows = rot = 0
    if rope is not None:
        rows, rot = rope.shape
        if rope.dtype != torch.float32 or not rope.is_contiguous():
            raise ValueError("rope is a contiguous float32 table")
    if q_out is None:
        q_out = torch.empty(T, n_heads, D, dtype=qkv.dtype, device=dev)
        _keep(q_out, stream)
    elif tuple(q_out.shape) != (T, n_heads, D) or q_out.dtype != qkv.dtype or not q_out.is_contiguous():
        raise ValueError("q_out is a contiguous [T, Hq, D] tensor of the activations' dtype")
    k, v, ks, vs = cache._ptrs
    _check(lib.momij_qk_norm_rope_append(
        qkv.data_ptr(), qkv.stride(0) if T > 1 else width, q_out.data_ptr(), None if q_weight is None else q_weight.data_ptr(),
        None if k_weight is None else k_weight.data_ptr(), eps, None if rope is None else rope.data_ptr(), rows, rot,
        interleaved, k, v, ks, vs, P, _table(block_table, B), block_table.shape[1], _ints(lens, "lens", (B,)),
        _ints(cu_q, "cu_q", (B + 1,)), T, B, max_q, n_heads, Hkv, D, _dtype_code(qkv),
        None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.nbytes,
        _raw_stream(stream, index)), "qkNormRopeAppend")
    return q_out


def cache_read(cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, *, count: int, first: torch.Tensor | None = None,
               dtype=torch.bfloat16, workspace: torch.Tensor | None = None, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of ``count`` tokens per sequence from ``first[b]`` on (default 0),
    [B, count, Hkv, D]; zeros at and past ``lens[b]``."""
    P, Hkv, D, dev = cache._dims
    index = _on(dev, block_table, lens, first, workspace)
    B = lens.shape[0]
    k_out = torch.empty(B, count, Hkv, D, dtype=dtype, device=dev)
    v_out = torch.empty(B, count, Hkv, D, dtype=dtype, device=dev)
    _keep(k_out, stream)
    _keep(v_out, stream)
    k, v, ks, vs = cache._ptrs
    _check(lib.momij_cache_read(
        k, v, ks, vs, P, _table(block_table, B), block_table.shape[1], _ints(lens, "lens", (B,)), _ints(first, "first", (B,)),
        count, k_out.data_ptr(), v_out.data_ptr(), B, Hkv, D, _dtype_code(k_out),
        None if workspace is None else workspace.data_ptr(), 0 if workspace is None else workspace.nbytes,
        _raw_stream(stream, index)), "cacheRead")
    return k_out, v_out


def attention(q: torch.Tensor, cache: KVCache, block_table: torch.Tensor, lens: torch.Tensor, *, scale: float | None = None,
              window: int = 0, cu_q: torch.Tensor | None = None, max_q: int = 0, out: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None, stream=None) -> torch.Tensor:
    """Causal attention of the new tokens' queries ``q`` [T, Hq, D] over the cache
    (momij_attention); ``scale`` defaults to D^-1/2, ``window`` 0 means all positions.
    Token rows of ``q`` and ``out`` may be strided."""
    P, Hkv, D, dev = cache._dims
    index = _on(dev, q, block_table, lens, cu_q, out, workspace)
    T, Hq, d = q.shape
    B = lens.shape[0]
    if d != D or q.stride(2) != 1 or (Hq > 1 and q.stride(1) != D):
        raise ValueError(f"q is [T, Hq, {D}] with contiguous rows")
    if out is None:
        out = torch.empty(T, Hq, D, dtype=q.dtype, device=dev)
        _keep(out, stream)
    elif tuple(out.shape) != (T, Hq, D) or out.dtype != q.dtype or out.stride(2) != 1 or (Hq > 1 and out.stride(1) != D):
        raise ValueError("out is [T, Hq, D] of q's dtype with contiguous rows")
    if workspace is None:
        workspace = new_workspace(T, Hq, D, dev)
        _keep(workspace, stream)
    k, v, ks, vs = cache._ptrs
    _check(lib.momij_attention(
        q.data_ptr(), q.stride(0) if T > 1 else Hq * D, out.data_ptr(), out.stride(0) if T > 1 else Hq * D, k, v, ks, vs, P,
        _table(block_table, B), block_table.shape[1], _ints(lens, "lens", (B,)), _ints(cu_q, "cu_q", (B + 1,)), T, B, max_q,
        Hq, Hkv, D, D ** -0.5 if scale is None else scale, window, _dtype_code(q), workspace.data_ptr(), workspace.nbytes,
        _raw_stream(stream, index)), "attention")
    return out
