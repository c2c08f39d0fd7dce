"""Error bounds of log probabilities, entropies and log-sums by what contributes to a row's sums."""
import math

import numpy as np

from attn_reference import U


def sum_bounds(x, scale):
    """Absolute bounds of a row's (lse, entropy) and a function for those of its ln p, from what contributes.

    A term 2^d of weight p: the factor scale / ln 2, d and its moves of the reference are each off by half a
    step (U) of the term's distance from the largest value (`dist`, in nats), the exponential by a step (2 U). A thread adds
    every other element to its running sum, the rest of a turn of eight at least once, so that (5/8) / 256 of the
    row's additions are off by U of the sum, each turn may move it (4 U), and the joins take some 60 more. A sum of
    p d (entropy) carries all this times dist, and the logarithm, its factor and its product some 6 U of itself.
    What a reference is off the largest value (half a step of it) belongs to every distance."""
    z = x[np.isfinite(x)] * np.float64(np.float32(scale))
    top, n = z.max(), len(x)
    dist = top - z
    p = np.exp(-dist)
    total = np.log(p.sum())
    p /= p.sum()
    off = 2 * U * abs(top) if abs(top) < 2 ** 24 * math.log(2) else 0.0  # (summed about the largest value itself past it)
    near, far = np.sum(p * dist) + off, np.sum(p * (dist + off) ** 2)
    turns = -(-n // 2048)
    rel = ((5 / 8) * n / 256 + 4 * turns + 62 + 3 * near) * U
    log = rel + (6 * total + 4) * U
    lse = log + U * abs(top + total)
    entropy = (1 + near) * rel + U * (3 * far + 6 * total + 8 * near + 4 + (total + near))
    return 1.01 * lse, 1.01 * entropy, lambda lp: 1.01 * (log + 2 * U * np.abs(lp))
