"""fp64 oracle of the two selections of a decoded token, the router's further
forms (``vq2_router_select``) and the next token's draw (``vq2_sample``) --
TEST INFRASTRUCTURE ONLY, written from the definitions row by row in numpy.

The reference has neither (its router is the softmax top-k of
``vq2_oracle.router_topk``, its decoding greedy, legion/engine.py:288): parity
unpinned, held to closed forms and counts in tests/test_selection.py.
"""
from __future__ import annotations

import numpy as np


def router_select(logits, k, scoring="softmax", bias=None, n_groups=1, topk_groups=None, group_score="max",
                  renormalise=True, scale=1.0):
    """ids int64 [T, k], weights fp64 [T, k].  Without a bias the choices
    order as the logits do, which are compared themselves (a sum of two
    choices apart): scores of large logits may round to the same number."""
    lg = np.atleast_2d(np.asarray(logits, np.float64))
    T, E = lg.shape
    b = np.zeros(E) if bias is None else np.asarray(bias, np.float64)
    size = E // n_groups
    keep = n_groups if topk_groups is None else topk_groups
    ids, w = np.zeros((T, k), np.int64), np.zeros((T, k))
    for t in range(T):
        x = lg[t]
        masked = ~(x > -np.inf) | ~(b > -np.inf)
        present = x > -np.inf
        s = np.zeros(E)
        if scoring == "sigmoid":
            with np.errstate(over="ignore"):
                s[present] = 1.0 / (1.0 + np.exp(-x[present]))
        elif present.any():
            top = x[present].max()
            d = np.array([0.0 if v == top else v - top for v in x[present]])
            s[present] = np.exp(d)
            s /= s.sum()
        c = [-np.inf if masked[e] else s[e] + b[e] for e in range(E)]
        o = c if bias is not None else [-np.inf if masked[e] else x[e] for e in range(E)]
        groups = []
        for g in range(n_groups):
            v = o if group_score == "max" else c
            best = sorted((v[e] for e in range(g * size, (g + 1) * size) if not masked[e]), reverse=True)
            score = -np.inf if not best else best[0] if group_score == "max" else sum(best[:2])
            groups.append((-score, g))
        stay = {g for _, g in sorted(groups)[:keep]}
        order = sorted((bool(masked[e]), -o[e], e) for e in range(E) if e // size in stay)
        ids[t] = [e for _, _, e in order[:k]]
        raw = np.array([0.0 if masked[e] else s[e] for e in ids[t]])
        total = raw.sum() if renormalise else 1.0
        w[t] = raw / total * scale if total > 0 else 0.0
    return ids, w


def sample_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, fp64 logprob, fp64 weights that stayed by column)."""
    x = np.asarray(logits, np.float64)
    present = np.flatnonzero(x > -np.inf)
    stayed = np.zeros(len(x))
    if len(present) == 0:
        return -1, np.nan, stayed
    top = x[present].max()
    order = sorted(present, key=lambda i: (-x[i], i))
    if temperature <= 0:
        stayed[order[0]] = 1.0
        return int(order[0]), 0.0, stayed
    w = {i: 1.0 if x[i] == top else float(np.exp((x[i] - top) / temperature)) for i in order}
    if top_k > 0:
        order = order[:top_k]
    total = sum(w[i] for i in reversed(order))
    kept, before = [], 0.0
    for i in order:
        if kept and top_p < 1.0 and not before < top_p * total:
            break
        kept.append(i)
        before += w[i]
    for i in kept:
        if w[i] >= min(min_p, 1.0):
            stayed[i] = w[i]
    run = np.cumsum(stayed)
    over = np.flatnonzero(run > min(max(u, 0.0), 1.0) * run[-1])
    token = int(over[0] if len(over) else np.flatnonzero(stayed)[-1])
    return token, float(np.log(stayed[token] / run[-1])), stayed


def sample_long_row(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, fp64 logprob) of sample_row for a long row of finite logits and a
    temperature above 0, by sorting and running sums of whole arrays."""
    x = np.asarray(logits, np.float64)
    order = np.argsort(-x, kind="stable")
    if top_k > 0:
        order = order[:top_k]
    w = np.exp((x[order] - x[order[0]]) / temperature)
    if top_p < 1.0:
        before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
        n = max(1, int(np.count_nonzero(before < top_p * w[::-1].sum())))
        order, w = order[:n], w[:n]
    order, w = order[w >= min(min_p, 1.0)], w[w >= min(min_p, 1.0)]
    by_column = np.argsort(order, kind="stable")
    order, w = order[by_column], w[by_column]
    run = np.cumsum(w)
    at = min(int(np.searchsorted(run, min(max(u, 0.0), 1.0) * run[-1], side="right")), len(order) - 1)
    return int(order[at]), float(np.log(w[at] / run[-1]))


def sample(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """Rows of sample_row; each setting a number or one value per row."""
    x = np.atleast_2d(np.asarray(logits, np.float64))
    B = x.shape[0]
    s = [np.broadcast_to(np.asarray(v), (B,)) for v in (u, temperature, top_k, top_p, min_p)]
    got = [sample_row(x[r], float(s[0][r]), float(s[1][r]), int(s[2][r]), float(s[3][r]), float(s[4][r]))
           for r in range(B)]
    return np.array([g[0] for g in got]), np.array([g[1] for g in got])
