"""Operators of requests that share cached tokens, over the paged BF16 cache
(csrc/paged_attention.cu, csrc/paged_attention_tc.cu): the append that writes it, the attention of prompts over
what their requests have cached already, and the decode attention of a batch whose
requests share a prefix.  (The reference calls flash-attn over its block tables,
nanovllm/layers/attention.py:59-75, which reads a shared prefix once per request.)

The cache is that of the model runner: BF16 [pages, 256, kv_heads, 128] for K and for
V, token t of a request in page ``block_tables[request, t // 256]`` at row ``t % 256``.
Requests share a prefix by naming the same pages; ``step_tables.build_step_tables``
makes the tables, slots and positions.  Outputs carry no gradient.
"""
from __future__ import annotations

import torch

from nanovllm import _native

HEAD_DIM = 128
PAGE_TOKENS = 256


def append_kv(q, k, v, cos_sin, positions, slot_mapping, k_cache, v_cache, *, q_weight=None, k_weight=None,
              eps: float = 1e-6, q_out=None):
    """Keys and values written to the cache rows ``slot_mapping`` (page * 256 + offset,
    each at most once; negative: stores nothing), the rotation applied on the way.

    ``q`` BF16 [T, Hq, 128] (or None), ``k`` and ``v`` BF16 [T, Hkv, 128], each with a
    token's heads contiguous and any distance between tokens (a multiple of 8
    channels): separate projections or views of a fused one.  With ``q_weight`` /
    ``k_weight`` BF16 [128] that side is RMS-normalised first.  ``cos_sin`` FP32
    [max_position, R] (cos, then sin): of the first R channels (a multiple of 16)
    c and c + R/2 are rotated.  ``positions`` INT64 [T], ``slot_mapping`` INT32 [T].
    Everything is FP32 with one rounding at the end (``qk_norm_rope_store`` of the
    engine rounds three times, as the reference does).  Returns ``q_out`` [T, Hq,
    128] (may be a contiguous ``q`` itself), None without ``q``.
    """
    return _native.serving().append_kv(q, k, v, cos_sin, positions, slot_mapping, k_cache, v_cache, q_weight, k_weight,
                                       eps, q_out)


def prefill_attention_workspace(num_tokens: int, batch: int, num_heads: int, num_kv_heads: int, device) -> torch.Tensor:
    """Scratch of ``paged_prefill_attention`` for up to so many tokens and requests (up to
    43 MB, and 40 bytes for every request and every block of up to 128 query rows of a KV
    head); calls that may overlap (other streams, graphs) need one each."""
    nbytes = _native.paged_prefill_attention_workspace_bytes(num_tokens, batch, num_heads, num_kv_heads)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def paged_prefill_attention(q, k_cache, v_cache, block_tables, context_lens, query_starts, *, scale: float, out=None,
                            workspace=None):
    """Attention of the new tokens of several requests, each over the tokens its
    request has in the cache, the new ones included (causal).

    ``q`` BF16 [T, Hq, 128] (Hq 1 to 16 times the KV heads), ``block_tables`` INT32
    [B, max_pages], ``context_lens`` INT32 [B], ``query_starts`` INT32 [B + 1], not
    falling: rows ``query_starts[b]`` to ``query_starts[b + 1] - 1`` are the last
    tokens of request b's context.  A row that sees no token gets zeros; rows of no
    request are left as they are.  What the cache holds behind a request's last token
    may be anything, its own tokens' values must be finite.  Probabilities are rounded to
    BF16 once.  Returns ``out`` BF16 [T, Hq, 128] (32-byte aligned; over no input).
    """
    return _native.serving().prefill_attention(q, k_cache, v_cache, block_tables, context_lens, query_starts, out,
                                               workspace, scale)


def shared_prefix_workspace(batch: int, groups: int, num_heads: int, num_kv_heads: int, device) -> torch.Tensor:
    """Scratch of ``shared_prefix_attention`` for up to so many requests and groups (43 MB,
    4160 bytes for every request and query head, and less than 100 for every request and
    group); calls that may overlap (other streams, graphs) need one each."""
    nbytes = _native.shared_prefix_attention_workspace_bytes(batch, groups, num_heads, num_kv_heads)
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def shared_prefix_attention(q, k_cache, v_cache, block_tables, context_lens, group_starts, prefix_lens, *,
                            scale: float, out=None, workspace=None):
    """Attention of one query token per request, each over its whole context, where
    groups of consecutive requests share a prefix that is read once for the group.

    ``q`` BF16 [B, Hq, 128], ``block_tables`` INT32 [B, max_pages], ``context_lens``
    INT32 [B] (0: a padding row, whose output is zero).  Requests ``group_starts[g]``
    to ``group_starts[g + 1] - 1`` have ``prefix_lens[g]`` tokens in common (INT32
    [groups + 1], not falling, and [groups]); the whole pages of these are read
    through the table of the group's longest request, and the others' tables must
    name the same pages as far as their contexts go (and the values there must be finite,
    also those behind a shorter request's last token).  Requests of no group share
    nothing.  Probabilities are multiplied in two BF16 terms, so that the output's
    rounding is the only one that shows.  Returns ``out`` BF16 [B, Hq, 128] (32-byte
    aligned; over no input).

    It pays from about 16 requests over 900 common tokens, 8 over 4096 and 4 over 16,384;
    smaller groups are faster row by row (``_native.paged_decode_attention``).
    """
    return _native.serving().shared_attention(q, k_cache, v_cache, block_tables, context_lens, group_starts,
                                              prefix_lens, out, workspace, scale)
