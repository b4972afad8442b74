"""Sampling settings of a request and the random numbers its tokens are drawn with.

The number for the token at index ``i`` of a sequence is a function of the request's seed and ``i`` alone (counter-based Philox4x32-10, Salmon et al. 2011),
so a request draws with the same numbers whatever it is batched with, and goes on with them after it was preempted and recomputed. Its tokens are the same wherever its
logits are: rows keep their bits beside others in products of up to 128 rows, while a step of more rows, or a prompt in other portions, may sum in another order."""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np

BLOCK = 64                       # numbers made at a time: the rounds are array operations, so a block costs little more than one number


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
        number = lambda v: isinstance(v, (int, float)) and not isinstance(v, bool)          # NaN is in no range
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


def philox_uniforms(seed, start, n: int) -> np.ndarray:
    """Numbers ``start .. start + n`` of a seed, FP32 in [0, 1): number i is word ``i % 4`` of block ``i // 4``, its upper 24 bits. With lists of seeds and
    starts (all of one remainder by 4) a row for each."""
    lo32, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    seeds, starts = np.atleast_1d(np.asarray(seed, dtype=np.uint64)), np.atleast_1d(np.asarray(start, dtype=np.uint64))
    skip = int(starts[0]) % 4
    block = starts[:, None] // np.uint64(4) + np.arange((skip + n + 3) // 4, dtype=np.uint64)
    c0, c1, c2, c3 = block & lo32, block >> shift, np.zeros_like(block), np.zeros_like(block)
    k0, k1 = (seeds & lo32)[:, None], (seeds >> shift)[:, None]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * c0, np.uint64(0xCD9E8D57) * c2
        c0, c1, c2, c3 = (p1 >> shift) ^ c1 ^ k0, p1 & lo32, (p0 >> shift) ^ c3 ^ k1, p0 & lo32
        k0, k1 = (k0 + np.uint64(0x9E3779B9)) & lo32, (k1 + np.uint64(0xBB67AE85)) & lo32
    words = np.stack((c0, c1, c2, c3), axis=2).reshape(len(seeds), -1)[:, skip: skip + n]
    out = ((words >> np.uint64(8)).astype(np.float64) * 2.0 ** -24).astype(np.float32)
    return out if np.ndim(seed) else out[0]


class Draws:
    """Settings of one live sequence with its random numbers, made a block at a time."""

    def __init__(self, settings: Sampling):
        self.settings = settings
        # as a step's metadata holds them: a row of settings is read once per token
        self.row = (np.float32(settings.temperature), np.int32(settings.top_k), np.float32(settings.top_p), np.float32(settings.min_p))
        self._block, self._numbers = -1, None

    def uniform(self, index: int) -> float:
        if index // BLOCK != self._block:
            renew([(self, index)])
        return self._numbers[index % BLOCK]


def renew(draws: "list[tuple[Draws, int] | None]") -> None:
    """Makes the blocks that a step's ``(Draws, index of the new token)`` lack, all at once: 64 together take the host as long as one does, 0.2 ms."""
    need = [(d, i // BLOCK) for d, i in (e for e in draws if e is not None) if i // BLOCK != d._block]
    if need:
        numbers = philox_uniforms([d.settings.seed for d, _ in need], [b * BLOCK for _, b in need], BLOCK)
        for (d, b), row in zip(need, numbers):
            d._block, d._numbers = b, row
