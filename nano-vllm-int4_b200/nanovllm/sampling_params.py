"""Sampling parameters (the reference's ``nanovllm/sampling_params.py``).

``temperature = 0`` selects greedy decoding, which the end-to-end benchmark
configuration uses; the reference rejects it (``sampling_params.py:10-11``).
``logprobs = k`` asks for every generated token's log-probability (of the model's
distribution, before the temperature), its rank, the entropy and the k most
likely alternatives; ``prompt_logprobs = k`` for the same of the prompt's tokens
after the first.  The reference returns neither.
"""
from dataclasses import dataclass
from operator import index

from nanovllm.kernels.token_logprobs import MAX_TOP_K


@dataclass(slots=True)
class SamplingParams:
    temperature: float = 1.0
    max_tokens: int = 64
    ignore_eos: bool = False
    logprobs: int | None = None
    prompt_logprobs: int | None = None

    def __post_init__(self):
        if self.temperature < 0:
            raise ValueError("temperature must be >= 0 (0 is greedy)")
        if self.max_tokens < 1:
            raise ValueError("max_tokens must be >= 1")
        for name in ("logprobs", "prompt_logprobs"):
            k = getattr(self, name)
            if k is None:
                continue
            try:
                k = index(k)
            except TypeError:
                k = -1
            if not 0 <= k <= MAX_TOP_K:
                raise ValueError(f"logprobs and prompt_logprobs must be None or an integer in 0..{MAX_TOP_K}")
            setattr(self, name, k)
