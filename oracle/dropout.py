"""Dropout from Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy
as 1, 2, 3", 2011), in unsigned integers.

Element i has the 16 bits number i % 8 (low half of a word first) of the counter
(i / 8 modulo 2^32, i / 8 >> 32, site, step) under the key (seed modulo 2^32,
seed >> 32); it is kept where they are below the threshold.
"""

from __future__ import annotations

import numpy as np

WORD = np.uint64(0xFFFFFFFF)
SHIFT = np.uint64(32)


def philox4x32(counter, key, rounds: int = 10):
    """Four words (uint64 arrays below 2^32) of counters given as four words."""

    c = [np.asarray(w, np.uint64) for w in counter]
    k0, k1 = int(key[0]), int(key[1])
    for _ in range(rounds):
        first = c[0] * np.uint64(0xD2511F53)
        second = c[2] * np.uint64(0xCD9E8D57)
        c = [(second >> SHIFT) ^ c[1] ^ np.uint64(k0), second & WORD,
             (first >> SHIFT) ^ c[3] ^ np.uint64(k1), first & WORD]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def threshold(rate: float) -> int:
    return min(65536, max(1, round(65536 * (1.0 - rate))))


def kept(count: int, seed: int, step: int, site: int, below: int, first: int = 0) -> np.ndarray:
    """Whether elements ``first`` to ``first + count - 1`` are kept."""

    lead = first % 8
    block = np.arange(first // 8, (first + count + 7) // 8, dtype=np.uint64)
    words = philox4x32([block & WORD, block >> SHIFT, np.full_like(block, site),
                        np.full_like(block, step & 0xFFFFFFFF)],
                       (seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF))
    bits = np.stack([h for w in words for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], 1)
    return (bits.reshape(-1)[lead:lead + count] < below)
