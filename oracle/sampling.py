"""Oracle of the device draw: temperature, top-k, top-p, min-p in extended precision over the sorted row (test
oracle only).  Steps of vte/core/sampler.py:54-129 with the random number given, min-p behind top-p."""
from __future__ import annotations

import numpy as np


def order(logits) -> np.ndarray:
    """Indices by (value descending, index ascending); NaN last."""
    x = np.where(np.isnan(logits), -np.inf, np.asarray(logits, np.float64))
    return np.lexsort((np.arange(len(x)), np.isnan(logits), -x))


def sample(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.0) -> tuple[int, float]:
    """(token, how near u came to another token, relative to the kept mass)."""
    logits = np.asarray(logits, np.float32)
    o = order(logits)
    top = logits[o[0]]
    if np.isnan(top) or top == -np.inf:
        return -1, 1.0
    if not temperature > 0:
        return int(o[0]), 1.0
    o = o[:top_k] if top_k > 0 else o
    x = logits[o].astype(np.longdouble)
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.exp((x - np.longdouble(top)) / np.longdouble(temperature))
    w = np.where(x == top, np.longdouble(1), np.where(np.isnan(x) | (x == -np.inf), np.longdouble(0), w))
    near = 1.0
    if 0 < top_p < 1:
        mass = np.cumsum(w)
        edge = np.abs(mass[:-1] - np.longdouble(top_p) * mass[-1])
        near = float(edge.min() / mass[-1]) if len(edge) else 1.0
        w = w[:1 + int(np.searchsorted(mass[:-1], np.longdouble(top_p) * mass[-1], side="right"))]
    if min_p > 0:
        near = min(near, float(np.abs(w - np.longdouble(min(min_p, 1.0)))[1:].min(initial=1.0)))
        w = w[w >= min(min_p, 1.0)]
    mass = np.cumsum(w)
    t = np.longdouble(u if u > 0 else 0.0) * mass[-1]
    live = int(np.count_nonzero(mass < mass[-1]))  # the last kept token with weight
    near = min(near, float(np.abs(mass - t).min() / mass[-1])) if u > 0 else near
    return int(o[min(int(np.searchsorted(mass, t, side="right")), live)]), near
