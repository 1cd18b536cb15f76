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
                numbers = np.where(key != key, -np.inf, key)
                best = [np.sort(numbers[g * (n // groups):(g + 1) * (n // groups)])[::-1][:2].sum() for g in range(groups)]
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


def experts(x, ids, weights, gate_up, down, eps):
    """y [tokens, hidden], and how far 32-bit sums and hidden values rounded to half a step ``eps / 2`` may be from it:
    gate_up [experts, 2 ffn, hidden] and down [experts, hidden, ffn] are the weights' values.

    A 32-bit sum of n products is off by at most n 2^-24 of their sizes' sum; silu has a slope below 1.1; exp, the quotient
    and two products are off by at most 2^-21 of the hidden value together."""
    y, tol, unit = np.zeros(x.shape), np.zeros(x.shape), 2.0 ** -24
    d, f = x.shape[1], down.shape[2]
    for e in sorted(set(ids.flatten().tolist())):
        if not 0 <= e < len(gate_up):
            continue
        t, j = np.nonzero(ids == e)
        g, u = (x[t] @ gate_up[e][i::2].T for i in (0, 1))
        eg, eu = (d * unit * (np.abs(x[t]) @ np.abs(gate_up[e][i::2]).T) for i in (0, 1))
        s = g / (1 + np.exp(-g))
        h = s * u
        eh = 1.1 * eg * (np.abs(u) + eu) + np.abs(s) * eu + (2.0 ** -21 + eps / 2) * np.abs(h)
        w = np.abs(weights[t, j])[:, None]
        np.add.at(y, t, weights[t, j][:, None] * (h @ down[e].T))
        np.add.at(tol, t, w * ((eh * (1 + f * unit) + (f + ids.shape[1] + 1) * unit * np.abs(h)) @ np.abs(down[e]).T))
    return y, tol


def log_probs(logits, tokens, top):
    """logprobs, ranks, entropy, top_ids and top_logprobs of logits [rows, vocab]."""
    rows, n = logits.shape
    got = np.zeros(rows), np.full(rows, -1), np.zeros(rows), np.zeros((rows, top), np.int64), np.zeros((rows, top))
    with np.errstate(all="ignore"):
        for r in range(rows):
            x = logits[r].astype(np.float64)
            m = x.max()
            p = np.exp(x - m) / np.exp(x - m).sum()
            logp = (x - m) - np.log(np.exp(x - m).sum())
            got[2][r] = -np.where(p == 0, 0.0, p * logp).sum()
            order = np.lexsort((np.arange(n), -np.where(x != x, -np.inf, x), x != x))
            got[3][r], got[4][r] = order[:top], logp[order[:top]]
            if 0 <= tokens[r] < n:
                got[0][r], got[1][r] = logp[tokens[r]], np.nonzero(order == tokens[r])[0][0]  # NaN behind everything
    return got
