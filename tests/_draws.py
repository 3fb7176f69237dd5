"""Dropout's draws restated in numpy: Philox4x32-10 (Salmon et al. 2011), eight values to a block, their upper 16 bits
from the counter (.., .., stream, 0) and their lower 16 from (.., .., stream, 1)."""
import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox(counter, key):
    """counter: four integers or uint64 arrays of 32-bit words; key: two integers."""
    c = [np.asarray(x, np.uint64) for x in counter]
    k = [int(x) for x in key]
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & M32, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & M32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def draws(first, n, seed, stream=0):
    """The 32 bits of values first .. first + n."""
    e = np.arange(first, first + n, dtype=np.uint64)
    block, j = e >> np.uint64(3), (e & np.uint64(7)).astype(np.int64)
    half = []
    for last in (0, 1):
        z = np.zeros_like(block)
        words = np.stack(philox((block & M32, block >> np.uint64(32), z + np.uint64(stream), z + np.uint64(last)),
                                (seed % 2 ** 32, seed // 2 ** 32)))
        half.append((words[j >> 1, np.arange(n)] >> (np.uint64(16) * (j & 1).astype(np.uint64))) & np.uint64(0xFFFF))
    return ((half[0] << np.uint64(16)) | half[1]).astype(np.uint64)


def kept(n, p, seed, stream=0, first=0):
    """(which of the values are kept, their factor)"""
    t = round(p * 2 ** 32)
    return draws(first, n, seed, stream) >= np.uint64(t), 0.0 if t == 2 ** 32 else 2 ** 32 / (2 ** 32 - t)
