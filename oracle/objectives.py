"""Token scoring and distillation in float64 NumPy, from the formulas: the oracle of csrc/token_objectives.hip.

The reference has neither operator (its losses and scores come from the Hugging Face models' own forward), so nothing of
it is restated here."""
import numpy as np

IGNORE = -100


def log_softmax(z, temperature=1.0):
    """Rows without a softmax (NaN, +inf, only -inf) are NaN."""
    y = np.asarray(z, np.float64) / temperature
    with np.errstate(all="ignore"):
        m = y.max(-1, keepdims=True)
        d = y - m
        return d - np.log(np.exp(d).sum(-1, keepdims=True))


def alternatives(z, k):
    """Indices of the k largest: value falling, NaN first, equal values (and -0, +0) by index."""
    z = np.asarray(z, np.float64)
    rank = np.where(np.isnan(z), np.inf, z)
    return np.lexsort((np.arange(z.shape[-1]), -rank, ~np.isnan(z)))[:k]


def token_logprobs(z, labels, top_k=0, temperature=1.0, ignore=IGNORE):
    """z (n, V), labels (n,) or None -> logprobs, entropy, top_ids, top_logprobs."""
    n, V = z.shape
    lp = log_softmax(z, temperature)
    p = np.exp(lp)
    with np.errstate(all="ignore"):
        h = -np.where(p == 0, 0.0, p * lp).sum(-1)
    logprob, ids, top = np.zeros(n), np.full((n, top_k), -1), np.full((n, top_k), -np.inf)
    for r in range(n):
        if labels is not None and labels[r] == ignore:
            h[r] = 0.0
            continue
        if labels is not None:
            logprob[r] = lp[r, labels[r]] if 0 <= labels[r] < V else np.nan
        ids[r] = alternatives(z[r], top_k)
        top[r] = lp[r, ids[r]]
    return logprob, h, ids, top


def token_logprobs_grad(z, labels, g_logprobs=None, g_entropy=None, ids=None, g_top=None, temperature=1.0, ignore=IGNORE):
    """-> gradient (n, V) and the sum of the sizes of the terms that make each value."""
    n, V = z.shape
    lp = log_softmax(z, temperature)
    grad, size = np.zeros((n, V)), np.zeros((n, V))
    for r in range(n):
        if labels is not None and labels[r] == ignore:
            continue
        p = np.exp(lp[r])
        h = -np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, lp[r])).sum()
        if g_logprobs is not None:
            one = np.arange(V) == labels[r]
            grad[r] += g_logprobs[r] * (one - p)
            size[r] += abs(g_logprobs[r]) * (one + p)
        if g_top is not None:
            for k, i in enumerate(ids[r]):
                one = np.arange(V) == i
                grad[r] += g_top[r, k] * (one - p)
                size[r] += abs(g_top[r, k]) * (one + p)
        if g_entropy is not None:
            t = np.where(p == 0, 0.0, p * np.where(p == 0, 0.0, lp[r]))
            grad[r] -= g_entropy[r] * (t + p * h)
            size[r] += abs(g_entropy[r]) * (abs(t) + p * abs(h))
    return grad / temperature, size / temperature


def teacher(ids, logits, temperature):
    kept = ids >= 0
    q = np.zeros(len(ids))
    if not kept.any() or logits[kept].max() == -np.inf:
        return q
    q[kept] = np.exp(log_softmax(logits[kept], temperature))
    return q


def distillation(z, labels, ids, logits, temperature=1.0, alpha=0.5, ignore=IGNORE):
    """-> losses (n,), gradients of their sum (n, V), sum of the sizes of the gradients' terms."""
    n, V = z.shape
    tau = temperature
    lp1, lpt = log_softmax(z), log_softmax(z, tau)
    losses, grad, size = np.zeros(n), np.zeros((n, V)), np.zeros((n, V))
    for r in range(n):
        if labels[r] == ignore:
            continue
        if not 0 <= labels[r] < V or (ids[r] >= V).any():
            losses[r] = np.nan
            grad[r] = np.nan
            continue
        q = teacher(ids[r], np.asarray(logits[r], np.float64), tau)
        on = q > 0
        if alpha > 0 and on.any():
            losses[r] += alpha * tau ** 2 * (q[on] * (np.log(q[on]) - lpt[r, ids[r][on]])).sum()
            grad[r] += alpha * tau * q.sum() * np.exp(lpt[r])
            size[r] += alpha * tau * np.exp(lpt[r])
            for k in np.flatnonzero(on):
                grad[r, ids[r, k]] -= alpha * tau * q[k]
                size[r, ids[r, k]] += alpha * tau * q[k]
        if alpha < 1:
            losses[r] -= (1 - alpha) * lp1[r, labels[r]]
            grad[r] += (1 - alpha) * np.exp(lp1[r])
            size[r] += (1 - alpha) * np.exp(lp1[r])
            grad[r, labels[r]] -= 1 - alpha
            size[r, labels[r]] += 1 - alpha
    return losses, grad, size
