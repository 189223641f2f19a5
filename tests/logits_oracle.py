"""The class-logit operators in 64-bit numpy, row by row, from their
definitions: what the kernels' tests compare with."""
from __future__ import annotations

import numpy as np

INF = np.inf


def _softmax(z, t):
    """p and ln p of a row with at least one class that is not masked."""
    x = z / t
    x = x - x.max()
    with np.errstate(over="ignore", under="ignore"):
        e = np.exp(x)
    logp = x - np.log(e.sum())
    return np.exp(logp), logp


def _state(z):
    if np.isnan(z).any() or (z == INF).any():
        return "bad"
    return "empty" if (z == -INF).all() else "fine"


def order(z):
    """Classes by value, equal ones by index, without masked ones."""
    at = np.lexsort((np.arange(z.size), -z))
    return at[z[at] > -INF]


def token_logprobs(z, tokens, k, t):
    n, v = z.shape
    out = {"logprob": np.zeros(n), "entropy": np.zeros(n), "rank": np.full(n, -1, np.int32),
           "stats": np.zeros((n, 2)), "top_ids": np.full((n, k), -1, np.int32),
           "top_logprobs": np.full((n, k), -INF)}
    z = z.astype(np.float64)
    for i in range(n):
        state = _state(z[i])
        token = -1 if tokens is None else int(tokens[i])
        given = token >= 0
        if state == "bad":
            out["logprob"][i] = np.nan if given else 0.0
            out["entropy"][i] = np.nan
            out["top_logprobs"][i] = np.nan
            out["stats"][i] = np.nan
            continue
        if token >= v:
            out["logprob"][i] = np.nan
        if state == "empty":
            if 0 <= token < v:
                out["logprob"][i] = -INF
            out["stats"][i] = -INF, 0.0
            continue
        p, logp = _softmax(z[i], t)
        out["entropy"][i] = -(p[p > 0] * logp[p > 0]).sum()
        out["stats"][i] = z[i].max(), np.exp((z[i] - z[i].max()) / t).sum()
        if 0 <= token < v:
            out["logprob"][i] = logp[token]
            before = (z[i] > z[i][token]) | ((z[i] == z[i][token]) & (np.arange(v) < token))
            out["rank"][i] = before.sum()
        best = order(z[i])[:k]
        out["top_ids"][i, :best.size] = best
        out["top_logprobs"][i, :best.size] = logp[best]
    return out


def _first_of_each(ids, v):
    """Which entries count: inside the classes, and not listed before."""
    seen, use = set(), np.zeros(ids.size, bool)
    for j, c in enumerate(ids):
        if 0 <= c < v and c not in seen:
            use[j] = True
            seen.add(int(c))
    return use


def token_logprobs_backward(z, tokens, top_ids, g_logprob, g_entropy, g_top, t):
    """From the formula: every listed log p pulls its class up and all down.
    (d, size): size is the same sum of absolute values, what rounding is
    relative to."""
    n, v = z.shape
    z = z.astype(np.float64)
    d, size = np.zeros((n, v)), np.zeros((n, v))
    for i in range(n):
        g = float(g_logprob[i]) if g_logprob is not None and tokens[i] >= 0 else 0.0
        h = float(g_entropy[i]) if g_entropy is not None else 0.0
        weight = np.zeros(v)
        use = np.zeros(0, bool)
        if g_top is not None:
            use = _first_of_each(top_ids[i], v)
            weight[top_ids[i][use]] += g_top[i][use]
        any_top = bool(use.size and (g_top[i][use] != 0).any())
        state = _state(z[i])
        if state == "empty" or (g == 0 and h == 0 and not any_top):
            continue
        if state == "bad" or (g != 0 and tokens[i] >= v):
            d[i] = np.nan
            continue
        p, logp = _softmax(z[i], t)
        if g != 0:
            weight[tokens[i]] += g
        d[i] = weight - p * weight.sum()
        live = p > 0
        entropy = -(p[live] * logp[live]).sum()
        d[i][live] -= h * p[live] * (logp[live] + entropy)
        d[i] /= t
        size[i] = np.abs(weight) + p * np.abs(weight).sum()
        size[i][live] += abs(h) * p[live] * (np.abs(logp[live]) + entropy)
        size[i] /= t
    return d, size


def distill(z, ids, teacher, kind, t, weights=None):
    """(loss, d_logits) of the weighted sum, and the sums of absolute values that
    their rounding is relative to."""
    n, v = z.shape
    z, teacher = z.astype(np.float64), teacher.astype(np.float64)
    loss, d = np.zeros(n), np.zeros((n, v))
    loss_size, size = np.zeros(n), np.zeros((n, v))
    for i in range(n):
        w = 1.0 if weights is None else float(weights[i])
        state = _state(z[i])
        if w == 0 or state == "empty":
            continue
        use = _first_of_each(ids[i], v)
        at, values = ids[i][use], teacher[i][use]
        if state == "bad" or (ids[i] >= v).any() or np.isnan(values).any():
            loss[i], d[i] = np.nan, np.nan
            continue
        p, logp = _softmax(z[i], t)
        if kind == "logits":
            q = np.zeros(at.size)
            if at.size and values.max() > -INF:
                q = np.exp((values - values.max()) / t)
                q /= q.sum()
        else:
            q = np.exp(values)
        rest = np.ones(v, bool)
        rest[at] = False
        rest &= z[i] > -INF
        q_rest = max(0.0, 1.0 - q.sum()) if kind == "logprobs" and rest.any() else 0.0
        loss[i] = sum(a * (np.log(a) - b) for a, b in zip(q, logp[at]) if a > 0)
        loss_size[i] = sum(a * (abs(np.log(a)) + abs(b) + 1) for a, b in zip(q, logp[at]) if a > 0)
        d[i] = p * (q.sum() + q_rest)
        d[i][at] -= q
        size[i] = p * (q.sum() + q_rest)
        size[i][at] += q
        if q_rest > 0:
            top = logp[rest].max()
            share = np.exp(logp[rest] - top)
            logp_rest = top + np.log(share.sum())
            loss[i] += q_rest * (np.log(q_rest) - logp_rest)
            # 1 - sum q is rounded relative to 1: 10 u of an error, here in units of
            # the tests' tolerances (130 u of the loss, 3e-5 of the gradient)
            loss_size[i] += (q_rest + 0.1) * (abs(np.log(q_rest)) + abs(logp_rest) + 1)
            d[i][rest] -= q_rest * share / share.sum()
            size[i][rest] += (q_rest + 0.02) * share / share.sum()
        loss[i] *= w * t * t
        d[i] *= w * t
        loss_size[i] *= abs(w) * t * t
        size[i] *= abs(w) * t
    return loss, d, loss_size, size
