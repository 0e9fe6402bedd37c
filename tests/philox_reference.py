"""Philox4x32-10 (Salmon, Moraes, Dror, Shaw, 2011) with numpy, and which elements a dropout keeps."""
import numpy as np

LOW, SHIFT = np.uint64(0xFFFFFFFF), np.uint64(32)


def words(counter, key):
    """[..., 4] uint32 of counters [..., 4] and a key of two words"""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [int(v) for v in key]
    for _ in range(10):
        p, q = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(q >> SHIFT) ^ c[1] ^ np.uint64(k[0]), q & LOW, (p >> SHIFT) ^ c[3] ^ np.uint64(k[1]), p & LOW]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(c, axis=-1).astype(np.uint32)


def kept(n, p, seed, call):
    """bool [n] and the factor of what is kept"""
    group = np.arange(-(-n // 8), dtype=np.uint64)
    seed, call = seed % 2 ** 64, call % 2 ** 64
    counter = np.stack([group & LOW, group >> SHIFT, np.full_like(group, call & 0xFFFFFFFF), np.full_like(group, call >> 32)],
                       axis=-1)
    w = words(counter, (seed & 0xFFFFFFFF, seed >> 32))
    halves = np.stack([w & np.uint32(0xFFFF), w >> np.uint32(16)], axis=-1).reshape(-1)[:n]
    steps = int(np.floor(p * 65536 + 0.5))
    return halves >= steps, (65536 / (65536 - steps) if steps < 65536 else 0.0)
