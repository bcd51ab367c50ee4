"""Philox4x32-10 (Salmon et al., SC 2011) on Python integers and numpy, and the dropout it drives."""
import numpy as np


def block(counter, key):
    """The four output words of one 4-word counter under a 2-word key."""
    c, (k0, k1) = list(counter), key
    for _ in range(10):
        p0, p1 = 0xD2511F53 * c[0], 0xCD9E8D57 * c[2]
        c = [(p1 >> 32) ^ c[1] ^ k0, p1 & 0xFFFFFFFF, (p0 >> 32) ^ c[3] ^ k1, p0 & 0xFFFFFFFF]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return c


def words(n, seed, offset, first=0):
    """Words `first` ... first + n - 1 of the sequence: word e % 4 of counter (e // 4, offset)."""
    lo, hi = first // 4, (first + n + 3) // 4
    c = np.arange(lo, hi, dtype=np.uint64)
    m, s = np.uint64(0xFFFFFFFF), np.uint64(32)
    x = [c & m, c >> s, np.full_like(c, offset & 0xFFFFFFFF), np.full_like(c, offset >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        p0, p1 = np.uint64(0xD2511F53) * x[0], np.uint64(0xCD9E8D57) * x[2]
        x = [(p1 >> s) ^ x[1] ^ np.uint64(k[0]), p1 & m, (p0 >> s) ^ x[3] ^ np.uint64(k[1]), p0 & m]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(x, 1).reshape(-1)[first - 4 * lo:][:n]


def keep(n, p, seed, offset):
    return words(n, seed, offset) >= np.uint64(int(p * 2 ** 32))
