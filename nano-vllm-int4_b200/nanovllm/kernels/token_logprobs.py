"""Log-probabilities of given tokens with their ranks, the distribution's
entropy and the most likely alternatives (csrc/token_logprobs.cu), beside the
sampler of the reference (nanovllm/layers/sampler.py), which returns ids only.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from nanovllm import _native

MAX_TOP_K = 32


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
    holds a NaN or +inf gives NaN.  With no rows the outputs are empty.  They
    carry no gradient, also for logits that require one.
    """
    return TokenLogprobs._make(_native.serving().logprobs(logits, targets, top_k))
