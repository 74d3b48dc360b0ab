"""Dropout's generator, CPU part: Philox4x32-10 in Python's integers against its
published vectors, as the GPU tests use it for any counter, offset and key."""

from __future__ import annotations

import pytest

LOW = 0xFFFFFFFF


def philox(counter, key):
    """Four words from four counter words and two key words (Salmon, Moraes, Dror, Shaw,
    "Parallel random numbers: as easy as 1, 2, 3", SC 2011)."""
    c, k = list(counter), list(key)
    for _ in range(10):
        p0, p1 = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [(p1 >> 32) ^ c[1] ^ k[0], p1 & LOW, (p0 >> 32) ^ c[3] ^ k[1], p0 & LOW]
        k = [(k[0] + 0x9E3779B9) & LOW, (k[1] + 0xBB67AE85) & LOW]
    return c


def words(first, n, seed, offset):
    """Words of elements first .. first + n - 1 (first a multiple of 4)."""
    out = []
    for g in range(first // 4, (first + n + 3) // 4):
        out += philox([g & LOW, g >> 32, offset & LOW, offset >> 32], [seed & LOW, seed >> 32])
    return out[:n]


# The published known answers: all zeros, all ones, the digits of pi.
@pytest.mark.parametrize("counter,key,want", [
    ([0] * 4, [0] * 2, [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]),
    ([LOW] * 4, [LOW] * 2, [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]),
    ([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0],
     [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]),
])
def test_published_vectors(counter, key, want):
    assert philox(counter, key) == want


def test_words_follow_their_element():
    assert words(8, 5, 3, 7) == words(0, 13, 3, 7)[8:]
    assert words(1 << 34, 4, 3, 7) == philox([0, 1, 7, 0], [3, 0])
