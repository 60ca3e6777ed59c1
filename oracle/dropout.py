"""The counter-based dropout mask in plain integer arithmetic (numpy, on the CPU): what include/ulm_b200.h defines.

Philox4x32 with ten rounds is Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", SC 2011.
"""
import numpy as np

_M0, _M1 = 0xD2511F53, 0xCD9E8D57
_W0, _W1 = 0x9E3779B9, 0xBB67AE85
_LOW = np.uint64(0xFFFFFFFF)


def philox4x32(counter, key, rounds=10):
    """``counter`` [n, 4] and ``key`` (two integers) of 32-bit words -> [n, 4] of 32-bit words (uint64 arrays)."""
    c = [np.asarray(counter[:, i], dtype=np.uint64) for i in range(4)]
    k0, k1 = key
    for _ in range(rounds):
        a, b = np.uint64(_M0) * c[0], np.uint64(_M1) * c[2]
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k0), b & _LOW, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k1), a & _LOW]
        k0, k1 = (k0 + _W0) & 0xFFFFFFFF, (k1 + _W1) & 0xFFFFFFFF
    return np.stack(c, axis=1)


def threshold(p):
    """The 16-bit numbers below it drop their element."""
    if p <= 0 or p >= 1:
        return 0 if p <= 0 else 65536
    return min(65535, max(1, round(p * 65536)))


def keep_mask(n, p, seed, start=0):
    """Truth values of the elements ``start`` to ``start + n`` that stay."""
    g0, g1 = start // 8, (start + n + 7) // 8
    groups = np.arange(g0, g1, dtype=np.uint64)
    counter = np.stack([groups & _LOW, groups >> np.uint64(32), np.zeros_like(groups), np.zeros_like(groups)], axis=1)
    words = philox4x32(counter, (seed & 0xFFFFFFFF, seed >> 32 & 0xFFFFFFFF))
    u = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], axis=2).reshape(-1)
    return (u >= threshold(p))[start - 8 * g0:][:n]


def scale(p):
    """What the elements that stay are multiplied by."""
    t = threshold(p)
    return 65536.0 / (65536 - t) if t < 65536 else 0.0
