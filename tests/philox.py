"""Philox4x32-10 (Salmon et al., 2011) in 64-bit integers, for the dropout tests."""
import numpy as np


def philox(counter, key):
    """counter: four uint64 arrays of 32-bit words; key: two integers."""
    mask, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    c, k = list(counter), list(key)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & mask,
             (a >> half) ^ c[3] ^ np.uint64(k[1]), a & mask]
        k = [(k[0] + 0x9E3779B9) % (1 << 32), (k[1] + 0xBB67AE85) % (1 << 32)]
    return c


def dropout_bits(n, seed, offset):
    """The 16 random bits of each of n elements."""
    first, count = offset // 8, (offset % 8 + n + 7) // 8
    # block numbers wrap at 2^61, as positions do at 2^64
    block = (np.uint64(first) + np.arange(count, dtype=np.uint64)) % np.uint64(1 << 61)
    zero = np.zeros_like(block)
    words = philox([block & np.uint64(0xFFFFFFFF), block >> np.uint64(32), zero, zero],
                   [seed % (1 << 32), seed >> 32])
    bits = np.stack(words, 1).astype(np.uint32).view(np.uint16).reshape(-1)
    return bits[offset % 8:offset % 8 + n].astype(np.int64)
