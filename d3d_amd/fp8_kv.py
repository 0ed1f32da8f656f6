"""The 8-bit paged KV cache: appends into it and block attention over it.

Keys and values are e4m3 codes with one power-of-two scale for each block of
tokens and KV head, half the bytes of the bf16 cache for every attention call
to read.  The functions are those of :mod:`d3d_amd.attention` and
:mod:`d3d_amd.layers` under the same names, with an :class:`Fp8KV` in the place
of ``k_cache`` and ``v_cache``:

* ``kv_append``                -- the KV store of
                                  serving/vendor/ssd/layers/attention.py:21-22
* ``qk_rope_append``           -- q/k norm, rotation and the store
* ``flash_attn_with_kvcache``, ``draft_block_attn``, ``packed_block_attn``

The reference's cache is bf16; there is no counterpart to this one in it.
All tensors live on one HIP device; there is no CPU path.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from functools import lru_cache
from typing import Optional

import torch

from . import _lib
from .layers import Product, SplitProduct

HEAD_DIM = 128
CODE = torch.float8_e4m3fn
SCALE = torch.float8_e8m0fnu
_SCALE = 1.0 / math.sqrt(HEAD_DIM)
_NO_WORKSPACE = 256  # bytes asked for where one range per request leaves nothing to merge


@dataclass(frozen=True, eq=False)
class Fp8KV:
    """One layer's 8-bit paged cache: codes ``k``, ``v`` [num_pages, Hkv,
    page_size, 128] e4m3 and scales ``k_scale``, ``v_scale`` [num_pages, Hkv,
    page_size / block] e8m0; an entry stands for code * scale.

    ``block`` (tokens that share a scale) is a power of two in 16 .. 256 that
    divides the page size.  Zero bytes are a valid empty cache, and pages can
    be used again without clearing: writing a block's first slot starts it
    anew.  Growing a scale moves codes by their exponents only, so appending
    token by token loses nothing that quantising the block at once keeps
    (while the codes stay normal: entries within 2^-14 of the block's largest).
    """
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor
    v_scale: torch.Tensor

    def __post_init__(self):
        for t, s in ((self.k, self.k_scale), (self.v, self.v_scale)):
            if t.ndim != 4 or t.shape != self.k.shape or t.shape[3] != HEAD_DIM:
                raise ValueError(f"expected k/v [num_pages, Hkv, page_size, {HEAD_DIM}] of equal shape")
            if t.dtype != CODE or s.dtype != SCALE:
                raise ValueError("expected float8_e4m3fn codes and float8_e8m0fnu scales")
            if s.ndim != 3 or s.shape != self.k_scale.shape or s.shape[:2] != t.shape[:2]:
                raise ValueError("expected k_scale/v_scale [num_pages, Hkv, page_size / block] of equal shape")
            if not (t.is_contiguous() and s.is_contiguous()):
                raise ValueError("codes and scales must be contiguous")
            if t.data_ptr() % 16:
                raise ValueError("codes must be 16-byte aligned")
        n = self.k_scale.shape[2]
        block = self.page_size // n if n and self.page_size % n == 0 else 0
        if not 16 <= block <= 256 or block & (block - 1):
            raise ValueError("a scale must cover a power of two of tokens in 16 .. 256 that divides the page size")
        if not self.num_pages or not self.kv_heads:
            raise ValueError("a cache needs at least one page and one KV head")
        if any(t.device != self.k.device for t in (self.v, self.k_scale, self.v_scale)):
            raise ValueError("codes and scales must be on one device")
        object.__setattr__(self, "_index", self.k.get_device())
        object.__setattr__(self, "_device", self.k.device)
        object.__setattr__(self, "_dims", tuple(self.k.shape[:3]))
        object.__setattr__(self, "block", block)

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, device, *, block: int = 16) -> "Fp8KV":
        """An empty cache (all zero)."""
        if block < 1 or page_size % block:
            raise ValueError("the block must divide the page size")
        codes = (num_pages, kv_heads, page_size, HEAD_DIM)
        scales = (num_pages, kv_heads, page_size // block)
        return cls(*(torch.zeros(codes, dtype=torch.uint8, device=device).view(CODE) for _ in range(2)),
                   *(torch.zeros(scales, dtype=torch.uint8, device=device).view(SCALE) for _ in range(2)))

    @property
    def num_pages(self) -> int:
        return self.k.shape[0]

    @property
    def kv_heads(self) -> int:
        return self.k.shape[1]

    @property
    def page_size(self) -> int:
        return self.k.shape[2]

    def _ptrs(self):
        return self.k.data_ptr(), self.v.data_ptr(), self.k_scale.data_ptr(), self.v_scale.data_ptr()

    def dequantize(self):
        """The values the cache stands for: bf16 (k, v) [num_pages,
        page_size, Hkv, 128], the bf16 cache's layout (exact)."""
        P, H, ps, D = self.k.shape
        return tuple((c.float().view(P, H, ps // self.block, self.block, D) * s.float()[..., None, None])
                     .view(P, H, ps, D).transpose(1, 2).contiguous().to(torch.bfloat16)
                     for c, s in ((self.k, self.k_scale), (self.v, self.v_scale)))


def _check_device(cache: Fp8KV, *tensors: Optional[torch.Tensor]) -> torch.device:
    """The cache's HIP device, which every given tensor must be on."""
    index = cache._index
    if index < 0:
        _lib.require_device(cache.k, *tensors)  # raises, naming the devices
    for t in tensors:
        if t is not None and t.get_device() != index:
            _lib.require_device(cache.k, *tensors)
    return cache._device


def _rows(x: torch.Tensor, n: int, heads: int, name: str) -> torch.Tensor:
    """x as [n, heads, 128] bf16 whose rows are contiguous and 8-byte aligned (a
    slice of a fused qkv product stays as it is)."""
    if x.dtype is not torch.bfloat16:
        x = x.to(torch.bfloat16)
    if x.shape != (n, heads, HEAD_DIM):
        if x.numel() != n * heads * HEAD_DIM:
            raise ValueError(f"{name} must hold [tokens, {heads}, {HEAD_DIM}] entries")
        x = x.reshape(n, heads, HEAD_DIM)
    step, inner, one = x.stride()
    if inner != HEAD_DIM or one != 1 or step % 4 or x.data_ptr() % 8:
        x = x.clone(memory_format=torch.contiguous_format)  # contiguous() keeps an odd address, or one row's stride
    return x


def kv_append(k: torch.Tensor, v: torch.Tensor, cache: Fp8KV, slot_mapping: torch.Tensor) -> None:
    """Quantise new keys/values into the cache by flat slot index.

    ``k``/``v`` [N, Hkv, 128] (or [N, Hkv * 128]) bf16, ``slot_mapping`` [N]
    int; slot = page_id * page_size + offset.  Slots outside the cache are
    skipped; of tokens with the same slot the last one counts.  A block whose
    first slot is written starts anew (its other slots become 0 unless written
    too); otherwise its scale grows as the new entries need and the entries it
    holds move to it.
    """
    dev = _check_device(cache, k, v, slot_mapping)
    n = slot_mapping.numel()
    P, H, ps = cache._dims
    k, v = _rows(k, n, H, "k"), _rows(v, n, H, "v")
    if slot_mapping.dtype is not torch.int64 or not slot_mapping.is_contiguous():
        slot_mapping = slot_mapping.to(torch.int64).contiguous()
    st = _lib.load().d3d_kv_append_fp8(k.data_ptr(), v.data_ptr(), k.stride(0), v.stride(0), *cache._ptrs(),
                                       slot_mapping.data_ptr(), n, H, HEAD_DIM, ps, cache.block, P,
                                       _lib.stream_ptr(dev))
    if st:
        _lib.check(st, "d3d_kv_append_fp8")


def qk_rope_append(qkv: Product, positions: torch.Tensor, q_norm: torch.Tensor, k_norm: torch.Tensor,
                   inv_freq: torch.Tensor, cache: Fp8KV, slot_mapping: torch.Tensor, heads: int, kv_heads: int,
                   eps: float, *, q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Normalise and rotate q and k, store k and v in the cache; returns q [T, Hq, 128].

    ``qkv`` [T, (Hq + 2 Hkv) * 128] bf16, or a SplitProduct of
    ``layers.project``; ``positions`` and ``slot_mapping`` [T] int64.  Norm and
    rotation run in fp32 for q, with one rounding to bf16 at the end, and in
    64 bits for k, whose result is rounded to its code, for the target and the
    draft alike; the store is ``kv_append``'s.
    """
    split = qkv if isinstance(qkv, SplitProduct) else None
    src = split.parts if split is not None else qkv
    dev = _check_device(cache, src, positions, q_norm, k_norm, inv_freq, slot_mapping, q_out)
    P, H, ps = cache._dims
    if heads < 1 or kv_heads != H:
        raise ValueError("the cache's KV heads do not match the model's")
    width = (heads + 2 * kv_heads) * HEAD_DIM
    if src.dtype is not (torch.bfloat16 if split is None else torch.float32) or not src.is_contiguous():
        raise ValueError("qkv must be contiguous bf16 (split partials contiguous fp32)")
    if src.shape[-1] != width:
        raise ValueError("qkv row width must be (heads + 2 kv_heads) * head_dim")
    T = src.shape[1] if split is not None else src.numel() // width
    long, bf16 = torch.int64, torch.bfloat16
    if positions.dtype is not long or positions.numel() != T or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int64 with one entry per token")
    if slot_mapping.dtype is not long or slot_mapping.numel() != T or not slot_mapping.is_contiguous():
        raise ValueError("slot_mapping must be contiguous int64 with one entry per token")
    if q_norm.dtype is not bf16 or q_norm.numel() != HEAD_DIM or not q_norm.is_contiguous():
        raise ValueError(f"q_norm must be contiguous bf16 [{HEAD_DIM}]")
    if k_norm.dtype is not bf16 or k_norm.numel() != HEAD_DIM or not k_norm.is_contiguous():
        raise ValueError(f"k_norm must be contiguous bf16 [{HEAD_DIM}]")
    if inv_freq.dtype is not torch.float32 or inv_freq.numel() != HEAD_DIM // 2 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous fp32 [head_dim / 2]")
    if q_out is None:
        q_out = torch.empty(T, heads, HEAD_DIM, dtype=torch.bfloat16, device=dev)
    elif q_out.dtype is not torch.bfloat16 or q_out.numel() != T * heads * HEAD_DIM or not q_out.is_contiguous():
        raise ValueError("q_out must be contiguous bf16 [T, heads, head_dim]")
    lib = _lib.load()
    call, head = ((lib.d3d_qk_rope_append_fp8, (src.data_ptr(),)) if split is None else
                  (lib.d3d_qk_rope_append_fp8_parts, (src.data_ptr(), split.splits)))
    st = call(*head, positions.data_ptr(), q_norm.data_ptr(), k_norm.data_ptr(), inv_freq.data_ptr(), q_out.data_ptr(),
              *cache._ptrs(), slot_mapping.data_ptr(), T, heads, kv_heads, HEAD_DIM, eps, ps, cache.block, P,
              _lib.stream_ptr(dev))
    if st:
        _lib.check(st, "d3d_qk_rope_append_fp8")
    return q_out


@lru_cache(maxsize=4096)
def _workspace_bytes(B: int, Q: int, Hq: int, Hkv: int, page_size: int, max_context: int) -> int:
    return _lib.load().d3d_attn_fp8_workspace_bytes(B, Q, Hq, Hkv, HEAD_DIM, page_size, max_context)


def _attn(fn_name: str, q, cache: Fp8KV, lens, block_table, softmax_scale, max_seqlen_k, out, vis=None):
    dev = _check_device(cache, q, lens, block_table, vis, out)
    if q.ndim != 4:
        raise ValueError("expected q [B, Q, Hq, D]")
    B, Q, Hq, D = q.shape
    P, H, ps = cache._dims
    if D != HEAD_DIM or Hq % H:
        raise ValueError("q and cache head shapes are incompatible")
    rows, max_pages = block_table.shape if block_table.ndim == 2 else (-1, 0)
    if rows != B:
        raise ValueError("expected block_table [B, max_pages]")
    if lens.numel() != B:
        raise ValueError("expected one context length per request")
    if max_seqlen_k is None:
        max_seqlen_k = max_pages * ps  # an upper bound that needs no host read
    else:
        max_seqlen_k = int(max_seqlen_k)
        if max_seqlen_k > max_pages * ps:
            raise ValueError("max_seqlen_k exceeds the block table's capacity")
    q_ptr = q.data_ptr()
    if q.dtype is not torch.bfloat16 or not q.is_contiguous() or q_ptr % 16:
        q = q.to(torch.bfloat16).contiguous()
        if q.data_ptr() % 16:
            q = q.clone()
        q_ptr = q.data_ptr()
    if block_table.dtype is not torch.int32 or not block_table.is_contiguous():
        block_table = block_table.to(torch.int32).contiguous()
    if lens.dtype is not torch.int32 or not lens.is_contiguous():
        lens = lens.to(torch.int32).contiguous()
    if out is None:
        out = torch.empty_like(q)
    elif out.dtype is not torch.bfloat16 or out.shape != q.shape or not out.is_contiguous():
        raise ValueError("out must be contiguous bf16 of q's shape")
    ws_ptr, ws_bytes = None, _workspace_bytes(B, Q, Hq, H, ps, max_seqlen_k)
    if ws_bytes > _NO_WORKSPACE:
        ws = _lib.workspace(dev, "attn_fp8", ws_bytes)
        ws_ptr = ws.data_ptr()
    st = getattr(_lib.load(), fn_name)(
        q_ptr, *cache._ptrs(), block_table.data_ptr(), lens.data_ptr(), *(() if vis is None else (vis.data_ptr(),)),
        out.data_ptr(), B, Q, Hq, H, D, ps, cache.block, max_pages, P,
        _SCALE if softmax_scale is None else softmax_scale, max_seqlen_k, ws_ptr, ws_bytes, _lib.stream_ptr(dev))
    if st:
        _lib.check(st, fn_name)
    return out


def flash_attn_with_kvcache(q: torch.Tensor, cache: Fp8KV, cache_seqlens: torch.Tensor, block_table: torch.Tensor, *,
                            causal: bool = True, softmax_scale: Optional[float] = None,
                            max_seqlen_k: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Paged attention of a block of Q queries per request; returns [B, Q, Hq, 128] bf16.

    With ``causal=True`` query i sees keys j <= cache_seqlens[b] - Q + i; with
    ``causal=False`` every key j < cache_seqlens[b].  ``max_seqlen_k``
    (optional) bounds cache_seqlens and sizes the context split; it defaults
    to the block table's capacity; ``softmax_scale`` is positive and finite.
    Rows that see no key are 0.
    """
    name = "d3d_verify_attn_paged_fp8" if causal else "d3d_draft_block_attn_fp8"
    return _attn(name, q, cache, cache_seqlens, block_table, softmax_scale, max_seqlen_k, out)


def draft_block_attn(q: torch.Tensor, cache: Fp8KV, context_lens: torch.Tensor, block_table: torch.Tensor, *,
                     softmax_scale: Optional[float] = None, max_seqlen_k: Optional[int] = None,
                     out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Draft block attention: prefix plus a bidirectional block (recovery mask)."""
    return _attn("d3d_draft_block_attn_fp8", q, cache, context_lens, block_table, softmax_scale, max_seqlen_k, out)


def packed_block_attn(q: torch.Tensor, cache: Fp8KV, context_lens: torch.Tensor, block_table: torch.Tensor,
                      q_visibility: torch.Tensor, *, softmax_scale: Optional[float] = None,
                      max_seqlen_k: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Packed multi-branch draft attention; ``q_visibility`` [Q, 3] int32 as
    :func:`d3d_amd.attention.packed_visibility` gives it, on the device."""
    if q.ndim != 4 or q_visibility.shape != (q.shape[1], 3) or q_visibility.dtype != torch.int32:
        raise ValueError("q_visibility must be int32 [Q, 3]")
    return _attn("d3d_packed_block_attn_fp8", q, cache, context_lens, block_table, softmax_scale, max_seqlen_k, out,
                 vis=q_visibility.contiguous())
