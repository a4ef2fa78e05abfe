"""Per-request sampling parameters.

The reference's engine imports a ``SamplingParams`` module that it does not ship; the one it does
ship (utils/sampler.py:7-23) has ``temperature``, ``max_tokens`` and ``ignore_eos`` and forbids
greedy decoding, while engine/sequence.py:31-34 also reads ``max_model_length``.  This class has
all four fields; ``temperature == 0`` selects greedy decoding (argmax, first maximum), which the
benchmark configurations require.  ``top_k`` (0: off), ``top_p`` (1: off) and ``min_p`` (0: off) narrow what a token
is drawn from (``ops.sample_filtered``; the reference has no such filters); greedy requests ignore them.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional


@dataclass
class SamplingParams:
    temperature: float = 1.0
    max_tokens: int = 256
    ignore_eos: bool = False
    max_model_length: Optional[int] = None
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0

    def __post_init__(self):
        if self.temperature < 0:
            raise ValueError("temperature must be >= 0 (0 = greedy)")
        if self.max_tokens < 1:
            raise ValueError("max_tokens must be >= 1")
        if not 0 <= self.top_k <= 0x7FFFFFFF:
            raise ValueError("top_k must be >= 0 (0 = off)")
        if not 0 < self.top_p <= 1:
            raise ValueError("top_p must be in (0, 1] (1 = off)")
        if not 0 <= self.min_p <= 1:
            raise ValueError("min_p must be in [0, 1] (0 = off)")

    @property
    def filtered(self) -> bool:
        return self.temperature > 0 and (self.top_k > 0 or self.top_p < 1 or self.min_p > 0)
