"""TEST INFRASTRUCTURE ONLY -- log probabilities, entropy and alternatives of logit rows in f64 (numpy)."""

from __future__ import annotations

import numpy as np


def order(x: np.ndarray) -> np.ndarray:
    """Indices of a row by value, ties to the lowest index, NaN above every number (numpy's argmax order)."""
    nan = np.isnan(x)
    return np.lexsort((np.arange(x.size), np.where(nan, 0, -x), ~nan))


def token_logprobs(x: np.ndarray, tokens, top_n: int):
    """x [rows, V] -> (logprobs, entropy, top_logprobs, top_ids, mean |x - max| under p)."""
    x = np.asarray(x, np.float64)
    rows, V = x.shape
    lp, ent, spread = np.zeros(rows), np.zeros(rows), np.zeros(rows)
    top, ids = np.zeros((rows, top_n)), np.zeros((rows, top_n), np.int64)
    with np.errstate(all="ignore"):
        for r in range(rows):
            m = x[r].max()  # (NaN if the row holds one)
            if m == -np.inf:
                y, ent[r] = np.full(V, -np.inf), 0.0
            else:
                d = x[r] - m
                e = np.exp(d)
                z = e.sum()
                y = d - np.log(z)
                w = np.where(e == 0, 0.0, e * d).sum() / z
                ent[r] = np.log(z) - w
                if np.isfinite(z):
                    spread[r] = -w
                else:
                    y = np.full(V, np.nan)
            t = int(tokens[r])
            lp[r] = y[t] if 0 <= t < V else -np.inf
            ids[r] = order(x[r])[:top_n]
            top[r] = y[ids[r]]
    return lp, ent, top, ids, spread
