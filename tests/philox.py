"""The generator of cavs_dropout_mask, in numpy: Philox4x32 with a number of rounds, and the mask that is made of it."""
import numpy as np

_LOW = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=7):
    """counter: four arrays (or numbers), key: two numbers; four arrays of uint32"""
    c = [np.asarray(v, dtype=np.uint64) for v in counter]
    k = [int(v) for v in key]
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & _LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & _LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return [v.astype(np.uint32) for v in c]


def threshold(p):
    return min(65535, int(float(np.float32(p)) * 65536 + 0.5))


def factor(p):
    return 65536 / (65536 - threshold(p))


def kept(n, w, p, seed, step, ids=None):
    """[n, w] bool"""
    row = (np.arange(n) if ids is None else np.asarray(ids)).astype(np.int64).astype(np.uint32).astype(np.uint64)[:, None]
    block = np.arange((w + 7) // 8, dtype=np.uint64)[None, :]
    row, block = np.broadcast_arrays(row, block)
    words = philox4x32([block, row, np.full_like(block, step & 0xFFFFFFFF), np.full_like(block, step >> 32 & 0xFFFFFFFF)], [seed & 0xFFFFFFFF, seed >> 32])
    draws = np.stack([d for v in words for d in (v & np.uint32(0xFFFF), v >> np.uint32(16))], axis=2).reshape(n, -1)
    return draws[:, :w] >= threshold(p)
