"""Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as
1, 2, 3", 2011) in Python integers, and the elements that dropout keeps."""
from __future__ import annotations

import numpy as np

W32 = np.uint64(0xFFFFFFFF)


def philox(counter, key):
    """The four words of `counter` (four uint64 arrays or integers below 2^32) under `key` (two integers)."""
    c = [np.asarray(w, dtype=np.uint64) for w in counter]
    k = [int(w) for w in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & W32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & W32]
        k = [(k[0] + 0x9E3779B9) % 2**32, (k[1] + 0xBB67AE85) % 2**32]
    return c


def threshold(p):
    return int(round(65536 * p))


def kept(n, p, seed, offset=0, first=0):
    """bool [n]: whether the elements first .. first + n - 1 are kept."""
    b0 = first // 8
    block = np.arange(b0, (first + n + 7) // 8, dtype=np.uint64)
    offset %= 2**64
    c = philox([block & W32, block >> np.uint64(32), np.full_like(block, offset % 2**32), np.full_like(block, offset >> 32)],
               [seed % 2**32, seed >> 32])
    halves = np.stack([h for w in c for h in (w & np.uint64(0xFFFF), w >> np.uint64(16))], axis=1).reshape(-1)
    return halves[first - 8 * b0:][:n] >= threshold(p)
