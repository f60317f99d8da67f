"""Sampling options of one request, named after the reference's SamplingConfig
(src/core/sampler/LLMSampler.h:55-63: _type, _temperature, _top_k, _top_p, _min_p,
_repetition_penalty, _seed).  The reference's ``sample`` ignores all of them and
returns the first maximum (LLMSampler.cpp:13-19); its helpers for temperature,
repetition penalty and multinomial draws exist unused (LLMSampler.cpp:21-54).  Here
they are honoured."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, List, Optional, Tuple

import numpy as np

GREEDY = "greedy"
RANDOM = "random"
TOP_K = "top_k"
TOP_P = "top_p"
STRATEGIES = ("default", GREEDY, RANDOM, TOP_K, TOP_P)   # FOR_EACH_STRATEGY, LLMSampler.h:18-24


_FLOAT32_MAX = float(np.finfo(np.float32).max)


@dataclass(frozen=True)
class SamplingParams:
    type: str = GREEDY                 # "greedy": temperature and filters are ignored
    temperature: float = 1.0
    top_k: int = 0                     # 0 = off
    top_p: float = 1.0                 # 1 = off
    min_p: float = 0.0                 # 0 = off
    repetition_penalty: float = 1.0    # 1 = off
    seed: int = 0
    max_new_tokens: int = 16
    eos_token_ids: Tuple[int, ...] = ()
    frequency_penalty: float = 0.0     # taken off a token's logit for every time it was generated
    presence_penalty: float = 0.0      # taken off a token's logit once it was generated
    logit_bias: Tuple[Tuple[int, float], ...] = ()        # (token, what is added to its logit; -infinity bans it)
    # a grammar: the generated tokens so far -> 32-bit words with a bit for every allowed token (token t: bit t % 32 of word
    # t // 32), or None for no limit.  Where it raises, allows no token or gives something else, its request ends (Engine:
    # reason "bad_mask")
    token_mask: Optional[Callable[[List[int]], Optional[np.ndarray]]] = None

    def __post_init__(self):
        if self.type not in STRATEGIES:
            raise ValueError(f"sampling type must be one of {STRATEGIES}, got '{self.type}'")
        if self.temperature < 0:
            raise ValueError("temperature must be >= 0")
        if self.top_k < 0 or not (0 < self.top_p <= 1.0) or not (0 <= self.min_p < 1.0):
            raise ValueError("top_k >= 0, 0 < top_p <= 1 and 0 <= min_p < 1 are required")
        if not 0 < self.repetition_penalty <= _FLOAT32_MAX or np.float32(self.repetition_penalty) == 0:
            raise ValueError("repetition_penalty must be > 0 and finite in float32")
        if not (abs(self.frequency_penalty) <= _FLOAT32_MAX and abs(self.presence_penalty) <= _FLOAT32_MAX):
            raise ValueError("frequency_penalty and presence_penalty must be finite in float32")
        if any(not 0 <= t < 2**31 or not v <= _FLOAT32_MAX for t, v in self.logit_bias):
            raise ValueError("logit_bias is pairs of a token id and a number that is finite in float32, or -infinity")
        if self.max_new_tokens < 0:
            raise ValueError("max_new_tokens must be >= 0")

    @property
    def controls_logits(self) -> bool:
        """Whether the logits are changed by more than a repetition penalty ahead of the draw."""
        return (self.frequency_penalty != 0.0 or self.presence_penalty != 0.0 or len(self.logit_bias) > 0
                or self.token_mask is not None)

    @property
    def needs_generated_tokens(self) -> bool:
        """Whether a draw depends on which tokens the request has generated (rather than had)."""
        return self.frequency_penalty != 0.0 or self.presence_penalty != 0.0 or self.token_mask is not None

    @property
    def needs_token_values(self) -> bool:
        """Whether a draw depends on which tokens the request has had."""
        return self.repetition_penalty != 1.0 or self.needs_generated_tokens

    @property
    def is_greedy(self) -> bool:
        return self.type in (GREEDY, "default") or self.temperature == 0.0

    @staticmethod
    def make(temperature: float = 0.0, **kw) -> "SamplingParams":
        """temperature 0 -> greedy; otherwise random sampling with the given filters."""
        if temperature == 0.0:
            return SamplingParams(type=GREEDY, temperature=1.0, **kw)
        t = TOP_K if kw.get("top_k", 0) > 0 else TOP_P if kw.get("top_p", 1.0) < 1.0 else RANDOM
        return SamplingParams(type=t, temperature=temperature, **kw)
