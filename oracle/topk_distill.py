"""Distillation from a teacher's kept tokens in fp64 (numpy), from the definition: the student's tail
mass as a logsumexp over the tokens that were not kept, everything in log space."""

import numpy as np

from oracle.token_logprobs import log_softmax, top_order

NO_TAIL = 2.0 ** -20


def _logsumexp(z):
    with np.errstate(divide="ignore", invalid="ignore"):
        m = z.max(axis=-1)
        base = np.where(np.isneginf(m), 0.0, m)
        return base + np.log(np.exp(z - base[..., None]).sum(axis=-1))


def _teacher(tokens, logprobs, tail):
    """Per row: (tokens, q, log q, r, q mass + r) of the used slots."""
    used = tokens >= 0
    if not used.any():
        return tokens[used], np.zeros(0), np.zeros(0), 0.0, 0.0
    logq = logprobs[used].astype(np.float64)
    mass = np.exp(logq).sum()
    if tail == "renormalize":
        if mass == 0.0:
            return tokens[used], np.zeros(len(logq)), logq, 0.0, 0.0
        logq = logq - np.log(mass)
        return tokens[used], np.exp(logq), logq, 0.0, 1.0
    r = max(0.0, 1.0 - mass)
    r = 0.0 if r <= NO_TAIL else r
    return tokens[used], np.exp(logq), logq, r, mass + r


def forward(x, targets, tokens, logprobs, tail="bucket", temperature=1.0, ignore_index=-100):
    """(ce, kl, accept, argmax) of rows [n, V] against teacher rows [n, K]."""
    x = np.asarray(x, np.float64)
    n, vocab = x.shape
    ce, kl, accept = np.zeros(n), np.zeros(n), np.zeros(n)
    one, logp = log_softmax(x), log_softmax(x, temperature)
    for i in range(n):
        if targets[i] != ignore_index:
            ce[i] = -one[i, targets[i]]
        kept, q, logq, r, mass = _teacher(tokens[i], logprobs[i], tail)
        if mass == 0.0:
            continue
        if np.isneginf(logp[i]).all():
            kl[i] = np.inf
            continue
        outside = np.delete(logp[i], kept)
        log_tail = _logsumexp(outside[None])[0] if outside.size else -np.inf
        some = q > 0
        with np.errstate(invalid="ignore"):
            kl[i] = (q[some] * (logq[some] - logp[i, kept][some])).sum()
            accept[i] = np.minimum(q, np.exp(logp[i, kept])).sum()
            if r > 0:
                kl[i] += r * (np.log(r) - log_tail)
                accept[i] += min(r, np.exp(log_tail))
    return ce, kl, accept, top_order(x)[:, 0]


def grad(x, targets, tokens, logprobs, g_ce, g_kl, tail="bucket", temperature=1.0, ignore_index=-100):
    """(gradient of sum(g_ce ce + g_kl kl) to x, sum of the magnitudes of its terms)."""
    x = np.asarray(x, np.float64)
    out, size = np.zeros_like(x), np.zeros_like(x)
    one, logp = log_softmax(x), log_softmax(x, temperature)
    for i in range(x.shape[0]):
        if np.isneginf(logp[i]).all():
            continue
        if targets[i] != ignore_index:
            out[i] += g_ce[i] * np.exp(one[i])
            out[i, targets[i]] -= g_ce[i]
            size[i] += abs(g_ce[i]) * np.exp(one[i])
            size[i, targets[i]] += abs(g_ce[i])
        kept, q, logq, r, mass = _teacher(tokens[i], logprobs[i], tail)
        if mass == 0.0:
            continue
        g = g_kl[i] / temperature
        p = np.exp(logp[i])
        direct = mass * p
        terms = direct.copy()
        direct[kept] -= q
        terms[kept] += q
        if r > 0:
            outside = np.ones(x.shape[1], bool)
            outside[kept] = False
            log_tail = _logsumexp(logp[i, outside][None])[0] if outside.any() else -np.inf
            if not np.isneginf(log_tail):
                within = np.where(outside, r * np.exp(logp[i] - log_tail), 0.0)
                direct -= within
                terms += within
        out[i] += g * direct
        size[i] += abs(g) * terms
    return out, size
