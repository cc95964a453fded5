"""Sampling options, with the reference's names, meanings and defaults
(src/runtime/engine.h:15-22): temperature 0.7 (<= 0: greedy), top_k 50,
top_p 0.95, repetition_penalty 1.05, seed 0 (= not fixed), max_new_tokens 512.

Beyond the reference's: `frequency_penalty` and `presence_penalty` (a token's logit falls by the first for every time it was
generated, by the second if it was at all), `logit_bias` (token id -> what is added to its logit; -inf bars it), and
`logprobs`: keep the log-probability of every generated token, under the model's own logits, and of the so many best tokens in its place
(None: keep none; 0: of the generated tokens only)."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Dict, Optional

_MOST = 3.4028234663852886e38   # the largest 32-bit float


@dataclass
class SamplingParams:
    temperature: float = 0.7
    top_k: int = 50
    top_p: float = 0.95
    repetition_penalty: float = 1.05
    seed: int = 0
    max_new_tokens: int = 512
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: Optional[Dict[int, float]] = None
    logprobs: Optional[int] = None

    def check(self, vocab: int, most_listed: int) -> None:
        """ValueError for what no row of `vocab` logits can be asked for."""
        for name in ("presence_penalty", "frequency_penalty"):
            if not abs(getattr(self, name)) <= _MOST:
                raise ValueError(f"{name} must be finite, is {getattr(self, name)}")
        for token, bias in (self.logit_bias or {}).items():
            if not 0 <= int(token) < vocab:
                raise ValueError(f"logit_bias names token {token}, the vocabulary is [0, {vocab})")
            if not (abs(bias) <= _MOST or bias == -math.inf):
                raise ValueError(f"logit_bias of token {token} is {bias}")
        if self.logprobs is not None and not 0 <= self.logprobs <= min(most_listed, vocab):
            raise ValueError(f"logprobs must be in [0, {min(most_listed, vocab)}], is {self.logprobs}")

    @staticmethod
    def greedy(max_new_tokens: int = 512) -> "SamplingParams":
        return SamplingParams(temperature=0.0, top_k=0, top_p=1.0, repetition_penalty=1.0,
                              seed=0, max_new_tokens=max_new_tokens)
