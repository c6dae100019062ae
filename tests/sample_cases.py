"""The draw of a token in 64 bits, word by word, for the tests of tkm_hip_sample."""
import math

import numpy as np


def draw_ref(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """x: a row of logits (floats).  Returns (token, how near u came to a border, relative to the kept sum)."""
    x = np.asarray(x, np.float64)
    x = np.where(np.isnan(x), -np.inf, x)
    m = x.max()
    if m == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(np.argmax(x)), 1.0
    w = np.zeros_like(x)
    with np.errstate(invalid="ignore", over="ignore"):
        for i in np.nonzero(x > -np.inf)[0]:
            t = 1.0 if x[i] == m else math.exp((x[i] - m) / temperature) if (x[i] - m) / temperature > -700 else 0.0
            w[i] = t
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    keep = order[:top_k] if 0 < top_k < len(x) else order
    if top_p < 1:
        total, run, n = math.fsum(w[i] for i in keep), 0.0, 0
        for i in keep:
            if n and run >= top_p * total:
                break
            run += w[i]
            n += 1
        keep = keep[:n]
    if min_p > 0:
        keep = [i for i in keep if w[i] >= min(min_p, 1.0)]
    keep = sorted(i for i in keep if w[i] > 0)
    run = np.cumsum(w[keep])
    u = min(max(u if u == u else 0.0, 0.0), 1 - 2.0 ** -60)
    at = int(np.searchsorted(run, u * run[-1], side="right"))
    at = min(at, len(keep) - 1)
    return keep[at], float(np.abs(np.concatenate(([0.0], run)) - u * run[-1])[1:-1].min() / run[-1]) if len(run) > 1 else 1.0
