"""Step metadata of a batch built on the GPU from request lengths
(csrc/step_tables.cu): what the reference's ``prepare_prefill`` and
``prepare_decode`` (nanovllm/engine/model_runner.py) build in Python lists.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from nanovllm import _native

MAX_REQUESTS = 28672  # of a batch


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

    def new(*shape, dtype=torch.int32):
        return torch.empty(shape, dtype=dtype, device=device)
    return StepTables(new(rows, max_pages), new(rows), new(tokens), new(tokens, dtype=torch.int64), new(rows + 1))


def build_step_tables(cached_lens, new_lens, pages, *, num_tokens: int, max_pages: int, page_size: int = 256,
                      out: StepTables | None = None) -> StepTables:
    """Block tables, context lengths, slots and positions of a step.

    Request b has ``cached_lens[b]`` tokens in the cache and ``new_lens[b]`` to
    compute (INT32 [B], B <= 28672); it owns the next ceil((cached + new) /
    page_size) entries of the flat list ``pages`` (INT32).  ``num_tokens`` is the
    number of new tokens.  ``out`` may have more rows and tokens than the step
    (the padding of a captured batch): rows behind the last request get context
    0 and pages 0, tokens behind the last slot -1 and position 0.  Its tensors may
    overlap neither the inputs nor one another.

    A token whose page is not listed, is negative or lies beyond ``max_pages``
    gets slot -1 and records device error 6 (``_native.device_error``).
    """
    return StepTables._make(_native.serving().step_tables(cached_lens, new_lens, pages, num_tokens, max_pages,
                                                          page_size, *(out or ())))
