"""Preference and policy losses in numpy and 64 bits, sequence by sequence
(written from the definitions; nothing of the package is used)."""

from __future__ import annotations

import numpy as np


def _spans(cu, tokens):
    return [(0, tokens)] if cu is None else [(int(a), int(b)) for a, b in zip(cu[:-1], cu[1:])]


def preference(policy, reference, cu, mask=None, beta=0.1, loss_type="sigmoid", smoothing=0.0, normalized=False,
               order="interleaved", items=None):
    """``(loss, chosen rewards, rejected rewards, d loss / d policy)``."""
    policy = np.asarray(policy, dtype=np.float64)
    reference = np.zeros_like(policy) if reference is None else np.asarray(reference, dtype=np.float64)
    mask = np.ones(policy.shape, bool) if mask is None else np.asarray(mask, dtype=bool)
    spans = _spans(cu, policy.size)
    n = len(spans) // 2
    score, width = np.zeros(2 * n), np.ones(2 * n)
    for s, (a, b) in enumerate(spans):
        m = mask[a:b]
        width[s] = max(m.sum(), 1) if normalized else 1
        score[s] = (policy[a:b][m] - reference[a:b][m]).sum() / width[s]
    c = np.arange(n) * (2 if order == "interleaved" else 1)
    r = c + 1 if order == "interleaved" else c + n
    x = score[c] - score[r]
    z = beta * x
    if loss_type == "sigmoid":
        loss = (1 - smoothing) * np.logaddexp(0, -z) + (smoothing * np.logaddexp(0, z) if smoothing else 0.0)
        dx = beta * (smoothing / (1 + np.exp(-z)) - (1 - smoothing) / (1 + np.exp(z)))
    elif loss_type == "ipo":
        loss, dx = (x - 0.5 / beta) ** 2, 2 * (x - 0.5 / beta)
    else:
        loss, dx = np.maximum(0, 1 - z), np.where(z < 1, -beta, 0.0)
    div = n if items is None else items
    grad = np.zeros_like(policy)
    for i in range(n):
        for s, sign in ((c[i], 1.0), (r[i], -1.0)):
            a, b = spans[s]
            grad[a:b][mask[a:b]] = sign * dx[i] / (div * width[s])
    return loss.sum() / div, beta * score[c], beta * score[r], grad


def policy(logps, old, adv, cu=None, mask=None, reference=None, low=0.2, high=None, dual=None, kl_coef=0.0,
           kl_type="k3", aggregation="token", items=None):
    """``(loss, mean kl, share of cut tokens, d loss / d logps)``."""
    logps, old, adv = (np.asarray(v, dtype=np.float64) for v in (logps, old, adv))
    mask = np.ones(logps.shape, bool) if mask is None else np.asarray(mask, dtype=bool)
    high = low if high is None else high
    spans = _spans(cu, logps.size)
    total, kls, cuts, count = 0.0, 0.0, 0, 0
    grad = np.zeros_like(logps)
    counted = sum(int(mask[a:b].sum()) for a, b in spans)
    for s, (a, b) in enumerate(spans):
        at = a + np.flatnonzero(mask[a:b])
        A = adv[at] if adv.shape == logps.shape else np.full(at.size, adv[s])
        d = logps[at] - old[at]
        r = np.exp(d)
        over, under = (A > 0) & (d > np.log1p(high)), (A < 0) & (d < np.log1p(-low) if low < 1 else False)
        far = (A < 0) & (d > np.log(dual)) if dual else np.zeros(at.size, bool)
        obj = A * np.where(over, 1 + high, np.where(under, 1 - low, np.where(far, dual or 0, r)))
        cut = over | under | far
        loss, g, kl = -obj, np.where(cut, 0.0, -A * r), np.zeros(at.size)
        if reference is not None:
            x = np.asarray(reference, dtype=np.float64)[at] - logps[at]
            kl, dkl = {"k1": (-x, np.ones_like(x)), "k2": (x * x / 2, -x),
                       "k3": (np.expm1(x) - x, -np.expm1(x))}[kl_type]
            loss, g = loss + kl_coef * kl, g + kl_coef * dkl
        if aggregation == "token":
            w = 1.0 / (max(counted, 1) if items is None else items)
        else:
            w = 1.0 / ((len(spans) if items is None else items) * max(at.size, 1))
        total += w * loss.sum()
        grad[at] = w * g
        kls, cuts, count = kls + kl.sum(), cuts + int(cut.sum()), count + at.size
    return total, kls / max(count, 1), cuts / max(count, 1), grad
