"""Shaped logits, their log-probabilities, gradients and draws, and the clipping of gradient lists, in numpy float64, one row after the
other: the definition that the GPU operators are tested against.  Next to each value stands `scale`, the size of the largest
intermediate that a 32-bit evaluation rounds, from which the tests derive their tolerances."""
import math

import numpy as np


def shaped_row(l, ids, repetition=1.0, presence=0.0, frequency=0.0, bias=None, allowed=None, temperature=1.0):
    """(y, slope, scale) of one row: l [V] float64; ids: the tokens it has seen; bias [V] or None; allowed: bool [V] or None."""
    V = len(l)
    ids = np.asarray(ids, dtype=np.int64)
    ids = ids[(ids >= 0) & (ids < V)]
    n = np.bincount(ids, minlength=V).astype(np.float64)
    seen = n > 0
    with np.errstate(invalid='ignore'):
        factor = np.where(seen, np.where(l > 0, 1.0 / repetition, repetition), 1.0)
        a = np.where(seen, l * factor - frequency * n - presence, l)
        scale = np.abs(l * factor) + np.where(seen, abs(frequency) * n + abs(presence), 0.0)
        if bias is not None:
            a = a + bias
            scale = scale + np.abs(bias)
        y, slope, scale = a / temperature, factor / temperature, scale / temperature
    if allowed is not None:
        y, slope, scale = np.where(allowed, y, -math.inf), np.where(allowed, slope, 0.0), np.where(allowed, scale, 0.0)
    return y, slope, scale


def log_prob_row(y, slope, token, g=1.0):
    """(log-probability, gradient of g * it against the logits, probabilities)."""
    V = len(y)
    zero = np.zeros(V)
    m = y.max()
    if m == -math.inf:
        return (-math.inf if 0 <= token < V else 0.0), zero, zero
    e = np.where(y == -math.inf, 0.0, np.exp(y - m))
    s = math.fsum(e)
    p = e / s
    if not 0 <= token < V:
        return 0.0, zero, p
    d = -p
    d[token] += 1.0
    return y[token] - m - math.log(s), np.where(slope == 0.0, 0.0, g * d * slope), p


def draw_row(y, u, empty=-1):
    """(token, log-probability, distance of u * total from the nearest boundary of the running sum, relative to the total)."""
    m = y.max()
    if m == -math.inf:
        return empty, -math.inf, 1.0
    e = np.where(y == -math.inf, 0.0, np.exp(y - m))
    cdf = np.cumsum(e)
    thr = float(u) * cdf[-1]
    last = int(np.nonzero(e > 0)[0][-1])
    pick = min(int((cdf <= thr).sum()), last)
    return pick, y[pick] - m - math.log(cdf[-1]), float(np.abs(cdf - thr).min() / cdf[-1])


def unpack(words, V):
    """bool [S, V] of int32 mask words [S, ceil(V / 32)]."""
    w = np.ascontiguousarray(words).view(np.uint32)
    return ((w[:, np.arange(V) >> 5] >> (np.arange(V) & 31).astype(np.uint32)) & 1).astype(bool)


def clip(grads, max_norm):
    """(norm, scaled gradients) of a list of float64 arrays, torch.nn.utils.clip_grad_norm_'s rule."""
    norm = math.sqrt(math.fsum(float(np.dot(g.ravel(), g.ravel())) for g in grads))
    coef = max_norm / (norm + 1e-6)
    return norm, [g * (1.0 if coef > 1.0 else coef) for g in grads]
