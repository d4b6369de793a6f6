"""Dropout, layer normalisation and their gradients in 64 bits on the CPU, with numpy, from the definitions."""
import numpy as np

# what one rounding to the type is off by, relative to the value; and the smallest normal value, below which steps are even
UNIT = {"f32": 2.0 ** -24, "bf16": 2.0 ** -8, "f16": 2.0 ** -11}
TINY = {"f32": 2.0 ** -126, "bf16": 2.0 ** -126, "f16": 2.0 ** -14}


def philox(counter, key, rounds):
    """Words [4, ...] of Philox4x32 (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011).
    counter: four arrays of 32-bit numbers, key: two numbers."""
    c = [np.asarray(x, dtype=np.uint64) for x in counter]
    k = [int(key[0]), int(key[1])]
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(rounds):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> shift) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> shift) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) & 0xFFFFFFFF, (k[1] + 0xBB67AE85) & 0xFFFFFFFF]
    return np.stack(np.broadcast_arrays(*c))


def kept(rows, width, p, seed, step):
    """bool [rows, width]: the values that dropout keeps"""
    quads = -(-width // 4)
    seed, step = seed % 2 ** 64, step % 2 ** 64
    at = np.arange(rows * quads, dtype=np.uint64)
    low, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    words = philox([at & low, at >> shift, np.uint64(step & 0xFFFFFFFF), np.uint64(step >> 32)],
                   (seed & 0xFFFFFFFF, seed >> 32), 7)
    return words.T.reshape(rows, quads * 4)[:, :width] >= np.uint64(round(p * 2 ** 32))


def factors(rows, width, drop):
    """float64 [rows, width] that dropout multiplies by; drop: None or (p, seed, step)"""
    if drop is None:
        return np.ones((rows, width))
    if drop[0] == 1:
        return np.zeros((rows, width))
    return kept(rows, width, *drop) / (1 - drop[0])


def statistics(x, eps):
    return x.mean(1), 1 / np.sqrt(x.var(1) + eps)


def normalise(x, weight, bias, eps):
    mean, rstd = statistics(x, eps)
    y = (x - mean[:, None]) * rstd[:, None]
    y = y if weight is None else y * weight
    return y if bias is None else y + bias


def gradient(dy, x, mean, rstd, weight):
    """(dx, dweight, dbias) of weight * h + bias, h = (x - mean) * rstd, and what the rounding errors of each scale with"""
    h = (x - mean[:, None]) * rstd[:, None]
    g = dy if weight is None else dy * weight
    dx = rstd[:, None] * (g - g.mean(1, keepdims=True) - h * (g * h).mean(1, keepdims=True))
    # h is off by some units of (|x| + |mean|) * rstd, each sum by some units of its terms' sizes
    off = np.abs(h) + (np.abs(x) + np.abs(mean)[:, None]) * rstd[:, None]
    size = rstd[:, None] * (np.abs(g) + np.abs(g).mean(1, keepdims=True) + off * np.abs(g * h).mean(1, keepdims=True)
                            + np.abs(h) * (np.abs(g) * off).mean(1, keepdims=True))
    return (dx, (dy * h).sum(0), dy.sum(0)), (size, (np.abs(dy) * off).sum(0), np.abs(dy).sum(0))
