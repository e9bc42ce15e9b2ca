"""A step of AdamW in numpy, 64 bits, straight from its formulas, with states in 32 or in 8 bits."""
import numpy as np

from .language_oracle import philox4x32

BLOCK = 256


def words(n, seed, step, number):
    """The 32-bit words of a tensor's n elements in a step."""
    block = np.arange(-(-n // 4), dtype=np.uint64)
    low, s32 = np.uint64(0xFFFFFFFF), np.uint64(32)
    counter = np.stack([block & low, block >> s32, np.full_like(block, step), np.full_like(block, number)], -1)
    return philox4x32(counter, np.array([seed % 2 ** 32, seed // 2 ** 32], np.uint64)).reshape(-1)[:n]


def each(scales, n):
    return np.repeat(scales.astype(np.float64), BLOCK)[:n]


def scales_of(x):
    """Largest magnitude / 448 of every 256 elements."""
    full = np.zeros(-(-x.size // BLOCK) * BLOCK)
    full[:x.size] = np.abs(x)
    most = full.reshape(-1, BLOCK).max(1)
    return np.where(most > 2.0 ** -110, most / 448, 0.0)


def position(x, scales, draws):
    """(steps, step): where |x| / scale lies among the e4m3 numbers, in steps of their distance there, with the draw [0, 65536) added: cut off
    to a whole it is the number that |x| becomes."""
    s = each(scales, x.size)
    v = np.divide(np.abs(x), s, out=np.zeros(x.size), where=s > 0)
    step = 2.0 ** (np.floor(np.log2(np.maximum(v, 2.0 ** -6))) - 3)
    return v / step + draws / 65536.0, step


def moments(m, v, g, beta1, beta2):
    """(m', v', the magnitudes that m' is the sum of)."""
    return beta1 * m + (1 - beta1) * g, beta2 * v + (1 - beta2) * g * g, beta1 * np.abs(m) + (1 - beta1) * np.abs(g)


def update(p, m, v, step, lr, beta1, beta2, eps, weight_decay):
    """p' from the new moments and the number of steps, this one counted."""
    return p - lr * (weight_decay * p + m / (1 - beta1 ** step) / (np.sqrt(v / (1 - beta2 ** step)) + eps))
