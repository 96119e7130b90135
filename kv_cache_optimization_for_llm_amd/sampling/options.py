"""What one request asks of the choice of its tokens, beyond its temperature.

The reference has one repetition penalty for all requests (``base/src/config.h:83``) and no cuts; here every request may bring its own.
In the order in which they act on its logits (:func:`~..ops.kernels.adjust_logits`, :func:`~..ops.kernels.sample_truncated`): the
repetition penalty, the frequency and presence penalties, the biases, the grammar; then, at a temperature, the first ``top_k`` tokens, of
these the share ``top_p``, of these the ones of at least ``min_p`` of the best one's probability.
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Callable, Mapping, Optional, Sequence

import numpy as np


_MOST = float(np.finfo(np.float32).max)         # what the kernels compute in


@dataclass(frozen=True)
class SampleOptions:
    """``repetition_penalty``: None is the server's.  ``penalize_prompt``: the repetition penalty takes the prompt's tokens as emitted
    ones, too (the other two count what the request itself has said).  ``logit_bias``: token id -> what its logit gains (-inf bans it).
    ``grammar``: called with the tokens emitted so far before every token, says which ones may come next - None (all of them), a
    truth value per token of the vocabulary, ids, or what :func:`pack_allowed` makes of them (:class:`AllowedWords`); a step that needs its
    answer waits for the tokens of the step before.  A request of whose vocabulary nothing is left ends with the error ``invalid_logits``."""

    top_k: int = 0                                  # 0: all tokens
    top_p: float = 1.0
    min_p: float = 0.0
    repetition_penalty: Optional[float] = None
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    penalize_prompt: bool = False
    logit_bias: Optional[Mapping[int, float]] = None
    grammar: Optional[Callable[[Sequence[int]], object]] = None

    def __post_init__(self):
        if not (isinstance(self.top_k, (int, np.integer)) and 0 <= self.top_k < 1 << 31):
            raise ValueError(f"top_k {self.top_k!r} is not a whole number from 0 on")
        for name, lo, hi in (("top_p", 0.0, 1.0), ("min_p", 0.0, 1.0)):
            v = getattr(self, name)
            if not lo <= v <= hi or (name == "top_p" and v == 0):
                raise ValueError(f"{name} {v!r} is not between 0 and 1")
        for name in ("presence_penalty", "frequency_penalty"):
            if not abs(getattr(self, name)) <= _MOST:
                raise ValueError(f"{name} must be finite in 32 bits")
        if self.repetition_penalty is not None and not 1 / _MOST <= self.repetition_penalty <= _MOST:
            raise ValueError("repetition_penalty must be positive and finite in 32 bits, as its inverse")
        for token, value in (self.logit_bias or {}).items():
            if int(token) != token or token < 0 or not value <= _MOST:
                raise ValueError(f"logit_bias {token!r}: {value!r} is not a token id and a number below the infinity of 32 bits")
        if self.grammar is not None and not callable(self.grammar):
            raise ValueError("grammar must be callable")

    @property
    def truncates(self) -> bool:
        return self.top_k > 0 or self.top_p < 1.0 or self.min_p > 0.0

    @property
    def penalizes(self) -> bool:
        return (self.repetition_penalty not in (None, 1.0) or self.presence_penalty != 0.0 or self.frequency_penalty != 0.0)


class AllowedWords(np.ndarray):
    """Allowed tokens as int32 words of 32 each (bit ``token % 32`` of word ``token / 32``): what :func:`pack_allowed` returns, or made of a
    row of int32 or uint32 words.  Words say by their class that they are; every other array of whole numbers is a row of ids, whatever its
    length."""

    def __new__(cls, words):
        a = np.asarray(words)
        if a.ndim != 1 or a.dtype not in (np.int32, np.uint32):
            raise ValueError("allowed words are a row of int32 or uint32")
        return a.view(np.int32).view(cls)


def pack_allowed(allowed, vocab_size: int) -> Optional[AllowedWords]:
    """Words of 32 tokens each from a truth value per token, from token ids, or from such words (:class:`AllowedWords`); ``None`` stays:
    everything is allowed."""
    if allowed is None:
        return None
    words = (vocab_size + 31) // 32
    if isinstance(allowed, AllowedWords):
        if allowed.shape != (words,) or allowed.dtype not in (np.int32, np.uint32):
            raise ValueError(f"allowed words {allowed.shape} {allowed.dtype} are not {words} of 32 tokens each")
        return allowed.view(np.int32)
    a = allowed if isinstance(allowed, np.ndarray) else np.asarray(list(allowed))
    if a.ndim != 1:
        raise ValueError("allowed tokens are a row of ids, of truth values, or of packed words")
    if a.dtype == np.bool_:
        if a.shape[0] != vocab_size:
            raise ValueError(f"{a.shape[0]} truth values for a vocabulary of {vocab_size}")
        bits = np.zeros(words * 32, dtype=np.uint8)
        bits[:vocab_size] = a
        return AllowedWords(np.packbits(bits, bitorder="little").view(np.int32))
    if a.shape[0] and not np.issubdtype(a.dtype, np.integer):
        raise ValueError("token ids must be whole numbers")
    ids = a.astype(np.int64)
    if ids.shape[0] and (ids.min() < 0 or ids.max() >= vocab_size):
        raise ValueError(f"an allowed token is outside [0, {vocab_size})")
    bits = np.zeros(words * 32, dtype=np.uint8)
    bits[ids] = 1
    return AllowedWords(np.packbits(bits, bitorder="little").view(np.int32))
