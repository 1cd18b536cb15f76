"""Plain 64-bit forms of the mixture-of-experts operators and of log probabilities (include/tgm_experts.h), in numpy, for the
tests."""

from __future__ import annotations

import numpy as np


def descending(keys: np.ndarray) -> np.ndarray:
    """Indexes by falling key, equal ones by index, NaN behind everything."""
    return np.array(sorted(range(len(keys)), key=lambda i: (1, 0.0, i) if keys[i] != keys[i] else (0, -keys[i], i)), dtype=np.int64)


def route(logits, top_k, score="softmax", bias=None, groups=1, top_groups=None, renormalize=True, scale=1.0):
    """ids and weights, [tokens, top_k]."""
    top_groups = groups if top_groups is None else top_groups
    tokens, n = logits.shape
    ids, weights = np.zeros((tokens, top_k), np.int64), np.zeros((tokens, top_k))
    with np.errstate(all="ignore"):
        for t in range(tokens):
            x = logits[t].astype(np.float64)
            if score == "softmax":
                p = np.zeros(n) if (x == -np.inf).all() else np.exp(x - x.max())
                p = p / p.sum() if p.sum() != 0 else p
            else:
                p = 1 / (1 + np.exp(-x))
            key = p if bias is None else p + bias.astype(np.float64)
            rank = x if bias is None else key
            left = []
            if top_groups < groups:
                best = [np.sort(key[g * (n // groups):(g + 1) * (n // groups)])[::-1][:2].sum() for g in range(groups)]
                keep = set(descending(np.array(best))[:top_groups].tolist())
                left = [e for e in range(n) if e // (n // groups) not in keep]
            order = [e for e in descending(rank) if e not in left]
            ids[t] = order[:top_k]
            w = p[ids[t]]
            total = w.sum() if renormalize else 1.0
            weights[t] = w * (scale / total) if total != 0 else 0.0
            if np.isnan(p).any():
                weights[t] = np.nan
    return ids, weights
