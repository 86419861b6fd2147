"""Step metadata of a batch built on the GPU from request lengths
(csrc/step_tables.cu): what the reference's ``prepare_prefill`` and
``prepare_decode`` (nanovllm/engine/model_runner.py) build in Python lists.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from nanovllm import _native

MAX_BATCH = 28672


class StepTables(NamedTuple):
    block_tables: torch.Tensor   # INT32 [rows, max_pages]: the request's pages, then 0
    context_lens: torch.Tensor   # INT32 [rows]: cached + new tokens
    slot_mapping: torch.Tensor   # INT32 [tokens]: cache slot of every new token; -1 behind the last
    positions: torch.Tensor      # INT64 [tokens]: its position in the request; 0 behind the last
    query_starts: torch.Tensor   # INT32 [rows + 1]: first new token of each request, then their total


def alloc_step_tables(rows: int, tokens: int, max_pages: int, device) -> StepTables:
    """Output buffers, for instance a captured graph's static ones."""
    if rows < 1 or tokens < 0 or max_pages < 1:
        raise ValueError("Expected rows>0, tokens>=0, max_pages>0")
    return _like(torch.empty(0, dtype=torch.int32, device=device), rows, tokens, max_pages)


def _like(x, rows: int, tokens: int, max_pages: int) -> StepTables:
    return StepTables(x.new_empty((rows, max_pages)), x.new_empty(rows), x.new_empty(tokens),
                      x.new_empty(tokens, dtype=torch.int64), x.new_empty(rows + 1))


def build_step_tables(cached_lens, new_lens, pages, *, num_tokens: int, max_pages: int, page_size: int = 256,
                      out: StepTables | None = None) -> StepTables:
    """Block tables, context lengths, slots and positions of a step.

    Request b has ``cached_lens[b]`` tokens in the cache and ``new_lens[b]`` to
    compute (INT32 [B], B <= 28672); it owns the next ceil((cached + new) /
    page_size) entries of the flat list ``pages`` (INT32).  ``num_tokens`` is the
    number of new tokens.  ``out`` may have more rows and tokens than the step
    (the padding of a captured batch): rows behind the last request get context
    0 and pages 0, tokens behind the last slot -1 and position 0.

    A token whose page is not listed, is negative or lies beyond ``max_pages``
    gets slot -1 and records device error 6 (``_native.device_error``).
    """
    if cached_lens.ndim != 1 or cached_lens.shape[0] < 1 or cached_lens.dtype != torch.int32 \
            or new_lens.shape != cached_lens.shape or new_lens.dtype != torch.int32:
        raise ValueError("Expected INT32 cached_lens[B] and new_lens[B], B>0")
    b = cached_lens.shape[0]
    if b > MAX_BATCH:
        raise ValueError(f"Expected at most {MAX_BATCH} requests")
    if pages.ndim != 1 or pages.dtype != torch.int32:
        raise ValueError("Expected INT32 pages[P]")
    if num_tokens < 0 or max_pages < 1 or page_size < 1:
        raise ValueError("Expected num_tokens>=0, max_pages>0, page_size>0")
    if out is None:
        out = _like(cached_lens, b, num_tokens, max_pages)
    else:
        rows = out.block_tables.shape[0]
        if out.block_tables.shape != (rows, max_pages) or rows < b or out.context_lens.shape != (rows,) \
                or out.query_starts.shape != (rows + 1,) or out.slot_mapping.ndim != 1 \
                or out.slot_mapping.shape[0] < num_tokens or out.positions.shape != out.slot_mapping.shape:
            raise ValueError("Expected out with block_tables[rows>=B,max_pages], context_lens[rows], "
                             "query_starts[rows+1], slot_mapping and positions[tokens>=num_tokens]")
        if out.positions.dtype != torch.int64 or any(
                x.dtype != torch.int32 for x in (out.block_tables, out.context_lens, out.slot_mapping,
                                                 out.query_starts)):
            raise TypeError("Expected INT64 positions and INT32 other outputs")
    if not _native.on_one_device(cached_lens.get_device(), cached_lens, new_lens, pages, *out):
        raise ValueError("All tensors must be contiguous on one CUDA device")
    _native.step_tables(cached_lens, new_lens, pages, out.block_tables, out.context_lens, out.query_starts,
                        out.slot_mapping, out.positions, page_size)
    return out
