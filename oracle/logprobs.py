"""numpy restatement, in 64 bits, of the log probabilities of given tokens -- test infrastructure only."""
from __future__ import annotations

import numpy as np


def token_logprobs(logits, tokens, num_top: int, temperatures=None):
    """(logprobs [T], entropy [T], top_ids [T, n], top_logprobs [T, n]); rows with a negative token are 0, 0, -1, 0."""
    T, V = logits.shape
    lp, entropy = np.zeros(T), np.zeros(T)
    ids, top = np.full((T, num_top), -1, dtype=np.int64), np.zeros((T, num_top))
    for t in range(T):
        if tokens[t] < 0:
            continue
        raw = np.asarray(logits[t], dtype=np.float64)
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            x = raw if temperatures is None else raw / float(temperatures[t])
            m = np.nan if np.isnan(x).any() else x.max()
            d = x - m
            p = np.exp(d)
            total = p.sum()
            log_p = d - np.log(total)
            lp[t] = log_p[tokens[t]] if tokens[t] < V else np.nan
            entropy[t] = np.log(total) - np.where(p > 0, d, 0.0) @ p / total if np.isfinite(total) else np.nan
        # the largest logits, NaN first, ties to the lowest index
        order = np.lexsort((np.arange(V), -np.where(np.isnan(raw), np.inf, raw), ~np.isnan(raw)))[:num_top]
        ids[t] = order
        top[t] = log_p[order]
    return lp, entropy, ids, top
