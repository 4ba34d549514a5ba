"""Token sampling restated on the CPU, row by row in 64 bits, for the tests."""
import math

import numpy as np


def sample_row(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    x = np.asarray(x, np.float64).copy()
    x[np.isnan(x)] = -math.inf
    top = x.max()
    if top == -math.inf:
        return -1
    t, p, low = (float(np.float32(v)) for v in (temperature, top_p, min_p))
    if not t > 0:
        return int(np.argmax(x == top))
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == top, 1.0, 0.0 if top == math.inf else np.exp((x - top) / t))
    w[x == -math.inf] = 0.0
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < x.size:
        order = order[:int(top_k)]
    v = w[order]
    if p < 1:
        before = np.concatenate([[0.0], np.cumsum(v)[:-1]])
        keep = before < p * v.sum()
        keep[0] = True
        order, v = order[keep], v[keep]
    if low > 0:
        order = order[v >= min(low, 1.0)]
    order = np.sort(order[w[order] > 0])
    c = np.cumsum(w[order])
    u = float(np.float32(u))
    u = u if u > 0 else 0.0
    return int(order[min(int(np.searchsorted(c, u * c[-1], side="right")), order.size - 1)])


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """logits [R, V] as a float array; each limit a number or an array [R]."""
    r = range(len(logits))
    each = [np.broadcast_to(np.asarray(v), (len(logits),)) for v in (temperature, top_k, top_p, min_p)]
    return np.array([sample_row(logits[i], u[i], *(e[i] for e in each)) for i in r], np.int64)
