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
_NO_CACHE = (None,) * 4


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
    rounded to BF16 (each by up to 2^-8 of itself; the decode attention reads them
    unrounded).
    ``slot_mapping`` and ``cache`` may both be None: nothing is stored then.
    """
    return _native.serving().store(qkv, q_weight, k_weight, cos_sin, positions, slot_mapping, *(cache or _NO_CACHE),
                                   num_heads, num_kv_heads, eps, q_out, return_values)


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
    return _native.serving().attention(q, *cache, block_tables, context_lens, out, workspace, scale)
