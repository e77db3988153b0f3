"""Plain restatement of the dropout's decisions: Philox4x32-10 in numpy."""

import math

import numpy as np

M32 = np.uint64(0xFFFFFFFF)


def philox(counter, key):
    """Ten rounds on a counter of four and a key of two words (arrays)."""
    c = [np.asarray(v, np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(10):
        a, b = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & M32,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & M32]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return c


def keep(elements, p, seed, offset):
    """Which of the given element numbers stay (bool array of their shape)."""
    e = np.asarray(elements, np.uint64)
    offset %= 2 ** 64
    block = e >> np.uint64(2)
    words = philox([block & M32, block >> np.uint64(32),
                    np.full(e.shape, offset % 2 ** 32, np.uint64),
                    np.full(e.shape, offset // 2 ** 32, np.uint64)],
                   [seed % 2 ** 32, seed // 2 ** 32])
    word = np.choose((e & np.uint64(3)).astype(np.int64), words)
    return word >= np.uint64(math.floor(p * 2 ** 32))


def weight(shape, p, seed, offset, rows=False):
    """keep / (1 - p) for every element of `shape`, in 64 bits."""
    shape = tuple(shape)
    if p == 1:
        return np.zeros(shape)
    if rows:
        kept = keep(np.arange(math.prod(shape[:-1])), p, seed, offset)
        return np.broadcast_to(kept.reshape(shape[:-1] + (1,)), shape) / (1.0 - p)
    return keep(np.arange(math.prod(shape)), p, seed, offset).reshape(shape) / (1.0 - p)
