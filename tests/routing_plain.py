"""Routing to experts in 64 bits, token by token: what the tests of route_experts compare with."""
import numpy as np


def scores(l, scoring):
    with np.errstate(all="ignore"):
        if scoring == "sigmoid":
            return 1.0 / (1.0 + np.exp(-l))
        m = l.max()
        z = np.exp(l - m) if m > -np.inf else np.zeros_like(l)
        return z / z.sum() if z.sum() != 0 else z


def falling(keys):
    """Indices by falling key: NaN first, equal ones by index."""
    return sorted(range(len(keys)), key=lambda i: (not np.isnan(keys[i]), -keys[i] if not np.isnan(keys[i]) else 0, i))


def choose(l, top, scoring="softmax", bias=None, groups=1, top_groups=1, group_best=1):
    """One token's experts, -1 for those that are not there."""
    s = scores(l, scoring)
    keys = l.copy() if bias is None else np.where(l == -np.inf, -np.inf, s + bias)
    ranked = s if bias is None and group_best == 2 else keys
    size = len(l) // groups
    ranks = []
    for g in range(groups):
        members = [i for i in falling(keys[g * size:(g + 1) * size]) if keys[g * size + i] != -np.inf][:group_best]
        ranks.append(sum(ranked[g * size + i] for i in members) if members else -np.inf)
    kept = falling(np.array(ranks))[:top_groups]
    keys = np.where(np.isin(np.arange(len(l)) // size, kept), keys, -np.inf)
    return [int(i) if keys[i] != -np.inf else -1 for i in falling(keys)[:top]]


def weigh(l, experts, scoring="softmax", renormalize=False, scale=1.0):
    s = scores(l, scoring)
    w = np.array([s[e] if e >= 0 else 0.0 for e in experts])
    if renormalize and any(e >= 0 for e in experts):
        with np.errstate(all="ignore"):
            # ratios of the scores, by their logarithms
            log = (lambda v: v) if scoring == "softmax" else (lambda v: -np.logaddexp(0.0, -v))
            a = np.array([log(l[e]) if e >= 0 else -np.inf for e in experts])
            w = np.exp(a - a.max())
            w = w / w.sum()
    return w * scale


def order_by_expert(experts, E):
    """experts [T, top] -> sizes, places, order."""
    flat = np.asarray(experts).reshape(-1)
    has = np.where(flat >= 0, flat, E)
    by = np.argsort(has, kind="stable")
    n = int((flat >= 0).sum())
    places = np.full(len(flat), -1)
    places[by[:n]] = np.arange(n)
    return np.bincount(has, minlength=E + 1)[:E], places.reshape(np.shape(experts)), np.where(np.arange(len(flat)) < n, by, -1 - by)


def route(logits, top, scoring="softmax", bias=None, groups=1, top_groups=None, group_best=1, renormalize=False, scale=1.0):
    """logits fp64 [T, E] -> weights, experts, sizes, places, order."""
    top_groups = groups if top_groups is None else top_groups
    experts = np.array([choose(l, top, scoring, bias, groups, top_groups, group_best) for l in logits]).reshape(len(logits), top)
    weights = np.array([weigh(l, e, scoring, renormalize, scale) for l, e in zip(logits, experts)]).reshape(len(logits), top)
    return (weights, experts, *order_by_expert(experts, logits.shape[1]))
