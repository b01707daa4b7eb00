"""The choice of a token from its definition, in 64 bits."""
import numpy as np


def choose(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, its share of what stays)."""
    x = np.where(np.isnan(x), -np.inf, np.asarray(x, np.float64))
    best = x.max()
    if best == -np.inf:
        return -1, 0.0
    if temperature == 0:
        return int(x.argmax()), 1.0
    order = np.lexsort((np.arange(x.size), -x))[:top_k or None]
    with np.errstate(invalid="ignore"):
        w = np.where(x[order] == best, 1.0, np.exp((x[order] - best) / temperature))
    if top_p < 1:
        reached = np.nonzero(np.cumsum(w) >= top_p * w.sum())[0]
        end = reached[0] + 1 if reached.size else w.size
        order, w = order[:end], w[:end]
    order, w = order[w >= min_p], w[w >= min_p]
    by_index = order.argsort()
    order, w = order[by_index], w[by_index]
    running = np.cumsum(w)
    at = min(int(np.searchsorted(running, u * running[-1], side="right")), w.size - 1)
    return int(order[at]), float(w[at] / running[-1])
