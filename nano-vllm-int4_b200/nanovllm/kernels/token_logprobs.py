"""Log-probabilities of given tokens with their ranks, the distribution's
entropy and the most likely alternatives (csrc/token_logprobs.cu), beside the
sampler of the reference (nanovllm/layers/sampler.py), which returns ids only.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from nanovllm import _native

MAX_TOP_K = 32
MAX_VOCAB = 1 << 24


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor              # FP32 [T]: of the given token, natural logarithm
    ranks: torch.Tensor                 # INT64 [T]: 1 + the number of logits above the token's
    entropy: torch.Tensor               # FP32 [T], in nats
    top_logprobs: torch.Tensor | None   # FP32 [T, top_k], falling
    top_ids: torch.Tensor | None        # INT64 [T, top_k], ties to the lowest id


def token_logprobs(logits, targets, *, top_k: int = 0) -> TokenLogprobs:
    """``logits`` BF16 or FP32 [T, V] (rows may be strided), ``targets`` INT64 [T].

    A target outside [0, V) is no token: logprob 0, rank 0.  Logits of -inf are
    no alternatives: where fewer than ``top_k`` (at most 32) are left, id -1 and
    -inf.  A row of nothing but -inf gives logprob -inf and entropy 0; a row that
    holds a NaN or +inf gives NaN.  With no rows the outputs are empty.
    """
    if logits.ndim != 2 or logits.shape[1] < 1 or logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("Expected BF16 or FP32 logits[T,V], V>0")
    t, v = logits.shape
    if v > MAX_VOCAB:
        raise ValueError(f"Expected a vocabulary of at most {MAX_VOCAB}")
    if targets.shape != (t,) or targets.dtype != torch.int64:
        raise ValueError("Expected INT64 targets[T]")
    if not 0 <= top_k <= MAX_TOP_K:
        raise ValueError(f"top_k must be in 0..{MAX_TOP_K}")
    if not logits.is_cuda or not _native.on_one_device(logits.get_device(), targets):
        raise ValueError("All tensors must be on one CUDA device, targets contiguous")
    if (v > 1 and logits.stride(1) != 1) or (t > 1 and logits.stride(0) < v):
        raise ValueError("The logits of a row must be contiguous, and rows must not overlap")
    new = logits.new_empty
    out = TokenLogprobs(new(t, dtype=torch.float32), new(t, dtype=torch.int64), new(t, dtype=torch.float32),
                        new((t, top_k), dtype=torch.float32) if top_k else None,
                        new((t, top_k), dtype=torch.int64) if top_k else None)
    if t:
        _native.token_logprobs(logits, targets, *out)
    return out
