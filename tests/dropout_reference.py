"""Which elements dropout keeps, from the generator's definition."""
import numpy as np


def philox(counter, key):
    """Philox4x32-10 over arrays of counters, in Python's whole numbers of 64 bits."""
    c, k = [np.asarray(v, np.uint64) for v in counter], list(key)
    low = np.uint64(0xFFFFFFFF)
    for _ in range(10):
        p0, p1 = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(p1 >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), p1 & low, (p0 >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), p0 & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return c


def kept(n, pe, seed, limit):
    block = np.arange(-(-n // 8), dtype=np.uint64)
    zero = np.zeros_like(block)
    words = philox([block & np.uint64(0xFFFFFFFF), (block >> np.uint64(32)) + np.uint64(pe << 16), zero + np.uint64(seed[1] & 0xFFFFFFFF),
                    zero + np.uint64(seed[1] >> 32)], [seed[0] & 0xFFFFFFFF, seed[0] >> 32])
    words = np.stack(words, 1)
    return np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], 2).reshape(-1)[:n] >= np.uint64(limit)
