"""The head operators' definitions in 64 bits, and inputs for their tests."""

from __future__ import annotations

import numpy as np

EPS32 = 2.0**-24  # half a step of float32, relative


def logprobs64(x, tokens=None, *, top=0, allowed=None, temperature=1.0):
    """float64 ``[rows, vocab]`` -> (logprobs, entropy, top_logprobs, top_ids) from the definition."""
    rows, vocab = x.shape
    tokens = np.zeros((rows, 0), np.int64) if tokens is None else tokens.reshape(rows, -1)
    lp = np.zeros(tokens.shape)
    ent = np.zeros(rows)
    top_lp = np.full((rows, top), -np.inf)
    top_ids = np.full((rows, top), -1, np.int64)
    for r in range(rows):
        on = np.ones(vocab, bool) if allowed is None else np.broadcast_to(allowed, (rows, vocab))[r].copy()
        on &= ~(x[r] == -np.inf)
        y = x[r][on] / temperature
        full = np.full(vocab, -np.inf)
        if y.size == 0:
            pass
        elif np.isnan(y).any() or (y == np.inf).any():
            full[:], ent[r] = np.nan, np.nan
        else:
            d = y - y.max()  # far values would lose the logarithm in the sum max + log
            lp_on = d - np.log(np.exp(d).sum())
            full[on] = lp_on
            ent[r] = -(np.exp(lp_on) * lp_on).sum()
        for j, t in enumerate(tokens[r]):
            lp[r, j] = 0.0 if t < 0 else np.nan if t >= vocab else full[t]
        ranked = np.where(on & ~np.isnan(x[r]), x[r], -np.inf) + 0.0
        order = np.argsort(-ranked, kind="stable")[:top]
        order = order[ranked[order] > -np.inf]
        top_ids[r, : len(order)] = order
        top_lp[r, : len(order)] = full[order]
    return lp, ent, top_lp, top_ids


def route64(x, top_k, *, scores="softmax", bias=None, groups=1, top_groups=1, group_score="max",
            renormalise=True, scale=1.0):
    """float64 ``[rows, experts]`` -> (weights float64, ids) from the definition: scores in 64 bits
    rounded once to 32, one 32-bit rounding for each sum that decides an order."""
    rows, experts = x.shape
    b = np.zeros(experts, np.float32) if bias is None else bias.astype(np.float32)
    weights, ids = np.zeros((rows, top_k)), np.full((rows, top_k), -1, np.int32)
    for r in range(rows):
        on = (x[r] > -np.inf) & (b > -np.inf)  # False for NaN
        l = np.minimum(x[r], np.finfo(np.float32).max)
        s = np.zeros(experts, np.float32)
        with np.errstate(over="ignore", under="ignore"):
            if scores == "sigmoid":
                s[on] = (1.0 / (1.0 + np.exp(-l[on]))).astype(np.float32)
            elif on.any():
                e = np.exp(l[on] - l[on].max())
                s[on] = (e / e.sum()).astype(np.float32)
        c = np.where(on, s + b, -np.inf).astype(np.float32)
        if groups > 1:
            g = np.sort(c.reshape(groups, -1), axis=1)[:, ::-1]
            value = g[:, 0].copy()
            if group_score == "top2" and g.shape[1] > 1:
                both = g[:, 1] > -np.inf
                value[both] = g[both, 0] + g[both, 1]
            best = [k for k in np.argsort(-value, kind="stable")[:top_groups] if value[k] > -np.inf]
            c = np.where(np.isin(np.arange(experts) // (experts // groups), best), c, -np.inf)
        order = np.argsort(-c, kind="stable")[:top_k]
        order = order[c[order] > -np.inf]
        w = s[order].astype(np.float64)
        if renormalise:
            w = w / w.sum() if w.sum() > 0 else np.zeros_like(w)
        ids[r, : len(order)], weights[r, : len(order)] = order, w * np.float64(np.float32(scale))
    return weights, ids


def plan64(ids, experts):
    """(order, slots, offsets) by a stable sort."""
    rows, k = ids.shape
    flat = ids.reshape(-1)
    kept = np.flatnonzero((flat >= 0) & (flat < experts))
    by = kept[np.argsort(flat[kept], kind="stable")]
    order, slots = np.full(rows * k, -1, np.int32), np.full(rows * k, -1, np.int32)
    order[: len(by)] = by // k
    slots[by] = np.arange(len(by))
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[kept], minlength=experts))]).astype(np.int32)
    return order, slots.reshape(rows, k), offsets


def combine64(y, weights, slots):
    """(sum, sum of magnitudes) in float64."""
    out, size = np.zeros((slots.shape[0], y.shape[1])), np.zeros((slots.shape[0], y.shape[1]))
    for j in range(slots.shape[1]):
        on = (slots[:, j] >= 0) & (slots[:, j] < y.shape[0])
        term = weights[on, j, None].astype(np.float64) * y[slots[on, j]]
        out[on] += term
        size[on] += np.abs(term)
    return out, size
