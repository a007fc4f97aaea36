"""Philox 4x32 with 10 rounds (Salmon, Moraes, Dror and Shaw, SC11) in Python
integers and in numpy, for the dropout tests."""

from __future__ import annotations

import numpy as np

M0, M1, W0, W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
LOW = 0xFFFFFFFF


def philox(counter, key):
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = M0 * c[0], M1 * c[2]
        c = [(b >> 32) ^ c[1] ^ k[0], b & LOW, (a >> 32) ^ c[3] ^ k[1], a & LOW]
        k = [(k[0] + W0) & LOW, (k[1] + W1) & LOW]
    return c


def words(first: int, count: int, seed: int, offset: int) -> np.ndarray:
    """The words of mask elements ``first .. first + count - 1``."""

    g0, g1 = first // 4, (first + count + 3) // 4
    group = np.arange(g0, g1, dtype=np.uint64)
    low, half = np.uint64(LOW), np.uint64(32)
    c = [group & low, group >> half, np.full_like(group, offset & LOW), np.full_like(group, offset >> 32)]
    for r in range(10):
        k0, k1 = np.uint64((seed + r * W0) & LOW), np.uint64(((seed >> 32) + r * W1) & LOW)
        a, b = np.uint64(M0) * c[0], np.uint64(M1) * c[2]
        c = [(b >> half) ^ c[1] ^ k0, b & low, (a >> half) ^ c[3] ^ k1, a & low]
    return np.stack(c, 1).reshape(-1)[first - 4 * g0 : first - 4 * g0 + count]
