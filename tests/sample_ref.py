"""Sampling with temperature, top-k, top-p and min-p from a given number, in 64 bits and plain numpy."""
import numpy as np


def ordered(x, t):
    """Tokens by logit, largest first, ties by index, and their weights; logits of -inf and NaN are none."""
    x = np.asarray(x, np.float64)
    at = np.nonzero(~np.isnan(x) & (x > -np.inf))[0]
    at = at[np.lexsort((at, -x[at]))]
    top = x[at[0]] if len(at) else 0.0
    if top == np.inf:
        return at, (x[at] == np.inf).astype(np.float64)
    return at, np.exp((x[at] - top) / t)


def sample(x, t, k, p, q, u, slack=0.0):
    """(tokens, probabilities by token and count, counts of kept tokens): every answer within `slack` of the whole mass
    of a border (one where slack is 0)."""
    at, w = ordered(x, t if t > 0 else 1.0)
    if not len(at):
        return {-1}, {(-1, 0): 0.0}, {0}
    if not t > 0:
        return {int(at[0])}, {(int(at[0]), 1): 1.0}, {1}
    n = min(k, len(at)) if k > 0 else len(at)
    mass = np.cumsum(w)
    kept = set()
    for s in {-slack, 0.0, slack}:
        m = n
        if p < 1:
            m = min(m, int(np.searchsorted(mass[:n], p * mass[n - 1] + s * mass[n - 1])) + 1)
        if q > 0:
            m = min(m, int((w >= q).sum()))
        kept.add(max(1, min(m, n)))
    kept = set(range(min(kept), max(kept) + 1))
    tokens, prob = set(), {}
    for m in kept:
        total = mass[m - 1]
        lo, hi = (min(m - 1, int(np.searchsorted(mass[:m], (u + s) * total, "right"))) for s in (-slack, slack))
        for i in range(lo, hi + 1):
            tokens.add(int(at[i]))
            prob[int(at[i]), m] = w[i] / total
    return tokens, prob, kept
