"""The 4-bit KV cache: the store that writes it and the decode attention that
reads it (csrc/kv4_cache.cu; the reference's cache, nanovllm/layers/attention.py,
is BF16 only).

K and V are held as 4-bit codes with one BF16 scale per 32 channels: 144 bytes
per token and KV head where the BF16 cache has 512.  A group's scale is
bf16(absmax / 7) (1 for an all-zero group), a value's code is
round-half-even(x / scale) in [-7, 7]; a value reads back as code * scale.  The
byte order within a page is described in include/nv4.h.  A group that holds an
infinity or NaN reads back as NaN.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from nanovllm import _native

HEAD_DIM = 128
PAGE_TOKENS = 256
GROUP_CHANNELS = 32


class Kv4Cache(NamedTuple):
    """One layer's cache: codes uint8 [pages, kv_heads, 256, 64] and scales BF16
    [pages, kv_heads, 256, 4], for K and for V."""
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor


def alloc_kv4_cache(num_pages: int, num_kv_heads: int, device) -> Kv4Cache:
    """An empty cache (its contents are undefined until a slot is stored)."""
    if num_pages < 1 or num_kv_heads < 1:
        raise ValueError("Expected at least one page and one KV head")

    def pair():
        return (torch.empty((num_pages, num_kv_heads, PAGE_TOKENS, HEAD_DIM // 2), dtype=torch.uint8, device=device),
                torch.empty((num_pages, num_kv_heads, PAGE_TOKENS, HEAD_DIM // GROUP_CHANNELS), dtype=torch.bfloat16,
                            device=device))
    return Kv4Cache(*pair(), *pair())


def page_bytes(num_kv_heads: int) -> int:
    """Bytes of one page of one layer."""
    return 2 * num_kv_heads * PAGE_TOKENS * (HEAD_DIM // 2 + HEAD_DIM // GROUP_CHANNELS * 2)


def _check_cache(cache: Kv4Cache) -> int:
    """Number of KV heads of a well-formed cache."""
    codes = cache.k_codes.shape
    if len(codes) != 4 or codes[0] < 1 or codes[1] < 1 or codes[2:] != (PAGE_TOKENS, HEAD_DIM // 2):
        raise ValueError("Expected codes[pages,Hkv,256,64]")
    scales = codes[:3] + (HEAD_DIM // GROUP_CHANNELS,)
    if cache.v_codes.shape != codes or cache.k_scales.shape != scales or cache.v_scales.shape != scales:
        raise ValueError("Expected K and V codes[pages,Hkv,256,64] and scales[pages,Hkv,256,4]")
    if cache.k_codes.dtype != torch.uint8 or cache.v_codes.dtype != torch.uint8:
        raise TypeError("Codes must be UINT8")
    if cache.k_scales.dtype != torch.bfloat16 or cache.v_scales.dtype != torch.bfloat16:
        raise TypeError("Cache scales must be BF16")
    return codes[1]


def qk_norm_rope_store_kv4(qkv, q_weight, k_weight, cos_sin, positions, slot_mapping, cache: Kv4Cache | None, *,
                           num_heads: int, num_kv_heads: int, eps: float, q_out=None, return_values: bool = False):
    """RMSNorm of the q and k heads, rotary embedding, K and V quantised into the
    cache rows ``slot_mapping`` (page * 256 + offset, each at most once; negative:
    stores nothing).

    ``qkv`` BF16 [T, (num_heads + 2 * num_kv_heads) * 128] (q | k | v),
    ``q_weight`` / ``k_weight`` BF16 [128], ``cos_sin`` FP32 [max_position, 128]
    (cos, then sin), ``positions`` INT64 [T], ``slot_mapping`` INT32 [T].  Returns
    q [T, num_heads, 128] in BF16, with ``return_values`` (q, k, v) where k and v
    [T, num_kv_heads, 128] are the values that the cache holds for the tokens,
    in BF16: attention over them gives what a later read of the cache gives.
    ``slot_mapping`` and ``cache`` may both be None: nothing is stored then.
    """
    if num_heads < 1 or num_kv_heads < 1:
        raise ValueError("Expected at least one query head and one KV head")
    if qkv.ndim != 2 or qkv.dtype != torch.bfloat16 or qkv.shape[0] < 1 \
            or qkv.shape[1] != (num_heads + 2 * num_kv_heads) * HEAD_DIM:
        raise ValueError("Expected BF16 qkv[T,(Hq+2Hkv)*128], T>0")
    t = qkv.shape[0]
    if q_weight.shape != (HEAD_DIM,) or k_weight.shape != (HEAD_DIM,) or q_weight.dtype != torch.bfloat16 \
            or k_weight.dtype != torch.bfloat16:
        raise ValueError("Expected BF16 q_weight[128] and k_weight[128]")
    if cos_sin.ndim != 2 or cos_sin.shape[0] < 1 or cos_sin.shape[1] != HEAD_DIM or cos_sin.dtype != torch.float32:
        raise ValueError("Expected FP32 cos_sin[max_position,128]")
    if positions.shape != (t,) or positions.dtype != torch.int64:
        raise ValueError("Expected INT64 positions[T]")
    if (slot_mapping is None) != (cache is None):
        raise ValueError("slot_mapping and cache go together")
    if slot_mapping is not None and (slot_mapping.shape != (t,) or slot_mapping.dtype != torch.int32):
        raise ValueError("Expected INT32 slot_mapping[T]")
    if cache is not None and _check_cache(cache) != num_kv_heads:
        raise ValueError("The cache has another number of KV heads")
    if q_out is None:
        q_out = qkv.new_empty((t, num_heads, HEAD_DIM))
    elif q_out.shape != (t, num_heads, HEAD_DIM) or q_out.dtype != torch.bfloat16:
        raise ValueError("Expected BF16 q_out[T,Hq,128]")
    if not _native.on_one_device(qkv.get_device(), qkv, q_weight, k_weight, cos_sin, positions, slot_mapping, q_out,
                                 *(cache or ())):
        raise ValueError("All tensors must be contiguous on one CUDA device")
    k_out = v_out = None
    if return_values:
        k_out = qkv.new_empty((t, num_kv_heads, HEAD_DIM))
        v_out = qkv.new_empty((t, num_kv_heads, HEAD_DIM))
    _native.qk_norm_rope_store_kv4(qkv, q_weight, k_weight, cos_sin, positions, slot_mapping, q_out, k_out, v_out,
                                   *(cache or (None,) * 4), num_heads, num_kv_heads, eps)
    return (q_out, k_out, v_out) if return_values else q_out


def kv4_attention_workspace(batch: int, num_heads: int, max_pages: int, device) -> torch.Tensor:
    """Scratch of ``paged_decode_attention_kv4`` for up to this batch and table
    width; calls that may overlap (other streams) need one each."""
    nbytes = _native.paged_attention_kv4_workspace_bytes(batch, num_heads, max_pages)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def paged_decode_attention_kv4(q, cache: Kv4Cache, block_tables, context_lens, *, scale: float, out=None,
                               workspace=None):
    """Attention of one query token per sequence over the 4-bit cache.

    ``q`` BF16 [B, Hq, 128] (Hq a multiple of the cache's KV heads, at most 8
    times as many), ``block_tables`` INT32 [B, max_pages], ``context_lens`` INT32
    [B] (0: a padding row, whose output is zero).  ``workspace`` comes from
    ``kv4_attention_workspace``; without it one is taken from torch's allocator.
    Returns ``out`` BF16 [B, Hq, 128].
    """
    if q.ndim != 3 or q.dtype != torch.bfloat16 or q.shape[0] < 1 or q.shape[2] != HEAD_DIM:
        raise ValueError("Expected BF16 q[B,Hq,128], B>0")
    b, hq, _ = q.shape
    hkv = _check_cache(cache)
    if hq < hkv or hq % hkv or hq // hkv > 8:
        raise ValueError("Expected query heads to be 1 to 8 times the KV heads")
    if block_tables.ndim != 2 or block_tables.shape[0] != b or block_tables.shape[1] < 1 \
            or block_tables.dtype != torch.int32:
        raise ValueError("Expected INT32 block_tables[B,max_pages]")
    if context_lens.shape != (b,) or context_lens.dtype != torch.int32:
        raise ValueError("Expected INT32 context_lens[B]")
    if not scale > 0:
        raise ValueError("scale must be positive")
    if out is None:
        out = q.new_empty(q.shape)
    elif out.shape != q.shape or out.dtype != torch.bfloat16:
        raise ValueError("Expected BF16 out[B,Hq,128]")
    if workspace is None:
        nbytes = _native.paged_attention_kv4_workspace_bytes(b, hq, block_tables.shape[1])
        workspace = q.new_empty(nbytes, dtype=torch.uint8)
    if not _native.on_one_device(q.get_device(), q, block_tables, context_lens, out, workspace, *cache):
        raise ValueError("All tensors must be contiguous on one CUDA device")
    _native.paged_decode_attention_kv4(q, *cache, block_tables, context_lens, out, workspace, scale)
    return out
