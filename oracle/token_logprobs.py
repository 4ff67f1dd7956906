"""Token log-probabilities, entropy, best alternatives and their gradient in fp64 (numpy), from the
definition: logp = log_softmax(x / temperature) with -inf logits as tokens without probability."""

import numpy as np


def log_softmax(x, temperature=1.0):
    """Rows [n, V]; a row without a finite logit is -inf everywhere, one with NaN or +inf is NaN."""
    z = np.asarray(x, np.float64) / temperature
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = z.max(axis=-1, keepdims=True)
        d = np.where(np.isneginf(m), -np.inf, z - m)
        return d - np.where(np.isneginf(m), 0.0, np.log(np.exp(d).sum(axis=-1, keepdims=True)))


def top_order(x):
    """Indices by descending logit, NaN first, ties (-0 and +0 too) by the lower index."""
    x = np.asarray(x, np.float64)
    return np.argsort(np.where(np.isnan(x), -np.inf, -x), axis=-1, kind="stable") if not np.isnan(x).any() else np.stack(
        [np.array(sorted(range(x.shape[1]), key=lambda j: (not np.isnan(r[j]), 0.0 if np.isnan(r[j]) else -r[j], j)))
         for r in x])


def _plogp(logp):
    with np.errstate(invalid="ignore"):
        return np.where(np.isneginf(logp), 0.0, np.exp(logp) * logp)


def forward(x, ids, top_k=0, temperature=1.0, ignore_index=-100):
    """(logprobs, entropy, top_logprobs, top_indices); tokens outside [0, V) give NaN."""
    logp = log_softmax(x, temperature)
    n, vocab = logp.shape
    rows = np.arange(n)
    valid = (ids >= 0) & (ids < vocab)
    chosen = np.where(valid, logp[rows, np.where(valid, ids, 0)], np.nan)
    chosen = np.where(ids == ignore_index, 0.0, chosen)
    order = top_order(x)[:, :top_k]
    return chosen, -_plogp(logp).sum(axis=-1), np.take_along_axis(logp, order, axis=-1), order


def grad(x, ids, g_logprob, g_entropy, g_top, top_k=0, temperature=1.0, ignore_index=-100):
    """Gradient of sum(g_logprob logprobs + g_entropy entropy + g_top top_logprobs) to x."""
    logp = log_softmax(x, temperature)
    n, vocab = logp.shape
    rows = np.arange(n)
    p = np.exp(logp)
    plogp = _plogp(logp)
    entropy = -plogp.sum(axis=-1, keepdims=True)
    scored = ids != ignore_index
    g = np.where(scored, g_logprob, 0.0)
    out = -g[:, None] * p - g_entropy[:, None] * (plogp + p * entropy)
    direct = np.zeros_like(out)
    valid = scored & (ids >= 0) & (ids < vocab)
    np.add.at(direct, (rows[valid], ids[valid]), g[valid])
    if top_k:
        out -= g_top.sum(axis=-1, keepdims=True) * p
        np.add.at(direct, (rows[:, None], top_order(x)[:, :top_k]), g_top)
    out = (out + direct) / temperature
    out[scored & ~valid] = np.nan
    out[np.isneginf(logp).all(axis=-1)] = 0.0
    return out
