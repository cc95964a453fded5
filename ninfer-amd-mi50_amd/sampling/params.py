"""Sampling options, with the reference's names, meanings and defaults
(src/runtime/engine.h:15-22): temperature 0.7 (<= 0: greedy), top_k 50,
top_p 0.95, repetition_penalty 1.05, seed 0 (= not fixed), max_new_tokens 512.

Beyond the reference's: `frequency_penalty` and `presence_penalty` (a token's logit falls by the first for every time it was
generated, by the second if it was at all), `logit_bias` (token id -> what is added to its logit; -inf bars it), and
`logprobs`: keep the log-probability of every generated token, under the model's own logits, and of the so many best tokens in its place
(None: keep none; 0: of the generated tokens only)."""
from __future__ import annotations

import math
import operator
from collections.abc import Mapping
from dataclasses import dataclass
from typing import Dict, Optional

_MOST = 3.4028234663852886e38   # the largest 32-bit float


def _number(value) -> float:
    """`value`, NaN for what is no number."""
    try:
        return math.nan if isinstance(value, (str, bytes)) else float(value)
    except (TypeError, ValueError, OverflowError):
        return math.nan


def _count(value) -> int:
    """`value`, -1 for what is no whole number."""
    try:
        return operator.index(value)
    except TypeError:
        return -1


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
        """ValueError for what no row of `vocab` logits can be asked for, and for options that are no numbers."""
        for name in ("presence_penalty", "frequency_penalty"):
            if not abs(_number(getattr(self, name))) <= _MOST:
                raise ValueError(f"{name} must be finite, is {getattr(self, name)!r}")
        if self.logit_bias and not isinstance(self.logit_bias, Mapping):
            raise ValueError(f"logit_bias must be a dict of token ids and biases, is {self.logit_bias!r}")
        for token, bias in (self.logit_bias or {}).items():
            try:
                fine = 0 <= int(token) < vocab
            except (TypeError, ValueError, OverflowError):
                fine = False
            if not fine:
                raise ValueError(f"logit_bias names token {token!r}, the vocabulary is [0, {vocab})")
            if not (abs(_number(bias)) <= _MOST or _number(bias) == -math.inf):
                raise ValueError(f"logit_bias of token {token} is {bias!r}")
        if self.logprobs is not None and not 0 <= _count(self.logprobs) <= min(most_listed, vocab):
            raise ValueError(f"logprobs must be in [0, {min(most_listed, vocab)}], is {self.logprobs!r}")

    @staticmethod
    def greedy(max_new_tokens: int = 512) -> "SamplingParams":
        return SamplingParams(temperature=0.0, top_k=0, top_p=1.0, repetition_penalty=1.0,
                              seed=0, max_new_tokens=max_new_tokens)
