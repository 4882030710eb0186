"""Routing to experts in numpy, from its definition, in 64 bits."""
import numpy as np

import herbert_hip as hb


def route(s, bias=None, score=hb.Score.Softmax, top_k=1, groups=1, top_groups=None, group_top=1, renorm=True, scale=1.0):
    """(experts, weights) of f32 scores [m][e]."""
    m, e = s.shape
    top_groups = groups if top_groups is None else top_groups
    ids, weights = np.zeros((m, top_k), np.uint32), np.zeros((m, top_k))
    for r in range(m):
        x = s[r].astype(np.float64)
        live = x > -np.inf
        p = np.zeros(e)
        if live.any():
            with np.errstate(over="ignore", invalid="ignore"):
                if score == hb.Score.Sigmoid:
                    p = np.where(live, 1 / (1 + np.exp(-x)), 0.0)
                else:
                    top = x[live].max()
                    p = np.where(live, np.exp(np.where(x == top, 0.0, x - top)), 0.0)
                    p = p / p.sum()
        # Without a bias, and no sums of them, the scores' own order is p's.
        two = top_groups < groups and group_top == 2
        with np.errstate(invalid="ignore"):
            c = p + bias.astype(np.float64) if bias is not None else p if two else x
            live = live & (c > -np.inf)
        c = np.where(live, c, -np.inf)
        if top_groups < groups:
            total = []
            for g in c.reshape(groups, -1):
                best = sorted(g[g > -np.inf], reverse=True)[:group_top]
                total.append(sum(best) if best else -np.inf)
            keep = sorted(range(groups), key=lambda g: (-total[g], g))[:top_groups]
            c = np.where(np.isin(np.arange(e) // (e // groups), keep), c, -np.inf)
        order = sorted(range(e), key=lambda i: (-c[i], i))[:top_k]
        w = np.array([p[i] if c[i] > -np.inf else 0.0 for i in order])
        if renorm:
            total = w.sum()
            w = w / total if total > 0 else 0 * w
        rank = np.argsort(order)
        ids[r], weights[r] = np.array(order)[rank], (w * scale)[rank]
    return ids, weights
