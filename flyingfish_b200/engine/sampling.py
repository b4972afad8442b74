"""Sampling settings of a request and the random numbers its tokens are drawn with.

The number for the token at index ``i`` of a sequence is a function of the request's seed and ``i`` alone (counter-based Philox4x32-10, Salmon et al. 2011),
so a request gives the same tokens whatever it is batched with, and goes on with the same numbers after it was preempted and recomputed."""
from __future__ import annotations

import math
from dataclasses import dataclass

import numpy as np

BLOCK = 256                      # numbers made at a time: the rounds are array operations, so a block costs little more than one number


@dataclass(frozen=True)
class Sampling:
    """How a sequence's tokens are chosen (``ops.sample_ops.sample_tokens``). ``temperature`` 0: the largest logit. ``top_k`` 0, ``top_p`` 1 and ``min_p`` 0
    leave every token."""
    temperature: float = 1.0
    top_k: int = 0
    top_p: float = 1.0
    min_p: float = 0.0
    seed: int = 0

    def __post_init__(self) -> None:
        number = lambda v: isinstance(v, (int, float)) and not isinstance(v, bool) and math.isfinite(v)
        whole = lambda v: isinstance(v, int) and not isinstance(v, bool)
        if not number(self.temperature) or not 0 <= self.temperature <= 1e6:
            raise ValueError("temperature must be a number from 0 to 1e6")
        if not whole(self.top_k) or not 0 <= self.top_k < 1 << 31:
            raise ValueError("top_k must be a whole number of 31 bits, 0 or more")
        if not number(self.top_p) or not 0 < self.top_p <= 1:
            raise ValueError("top_p must be above 0, at most 1")
        if not number(self.min_p) or not 0 <= self.min_p <= 1:
            raise ValueError("min_p must be from 0 to 1")
        if not whole(self.seed) or not 0 <= self.seed < 1 << 64:
            raise ValueError("seed must be a whole number of 64 bits")


def philox_uniforms(seed: int, start: int, n: int) -> np.ndarray:
    """Numbers ``start .. start + n`` of a seed, FP32 in [0, 1): number i is word ``i % 4`` of block ``i // 4``, its upper 24 bits."""
    lo32, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    block = np.arange(start // 4, (start + n + 3) // 4, dtype=np.uint64)
    c0, c1, c2, c3 = block & lo32, block >> shift, np.zeros_like(block), np.zeros_like(block)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c0, np.uint64(0xCD9E8D57) * c2
        c0, c1, c2, c3 = (p1 >> shift) ^ c1 ^ np.uint64(k0), p1 & lo32, (p0 >> shift) ^ c3 ^ np.uint64(k1), p0 & lo32
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = np.stack((c0, c1, c2, c3), axis=1).reshape(-1)[start % 4: start % 4 + n]
    return ((words >> np.uint64(8)).astype(np.float64) * 2.0 ** -24).astype(np.float32)


class Draws:
    """Settings of one live sequence with its random numbers, made a block at a time."""

    def __init__(self, settings: Sampling):
        self.settings = settings
        # as a step's metadata holds them: a row of settings is read once per token
        self.row = (np.float32(settings.temperature), np.int32(settings.top_k), np.float32(settings.top_p), np.float32(settings.min_p))
        self._block, self._numbers = -1, None

    def uniform(self, index: int) -> float:
        if index // BLOCK != self._block:
            self._block = index // BLOCK
            self._numbers = philox_uniforms(self.settings.seed, self._block * BLOCK, BLOCK)
        return self._numbers[index % BLOCK]
