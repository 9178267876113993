"""Distillation from a teacher's named tokens, and its gradients, in numpy and 64
bits (written from the definitions; nothing of the package is used)."""

from __future__ import annotations

import numpy as np

from .token_stats import FP32, HALF, SUM, log_softmax, logits


def named(ids, log_probs, vocab):
    """The tokens that one row's teacher names, as ``(ids, log t, bad)``: without ids of -1, probabilities of zero, ids
    outside the vocabulary and tokens that were named before (the last two are bad)."""
    seen, lts, bad = [], [], 0
    for i, lt in zip(ids, log_probs):
        if i == -1:
            continue
        if i < 0 or i >= vocab:
            bad += 1
        elif lt == -np.inf:
            continue
        elif i in seen:
            bad += 1
        else:
            seen.append(int(i))
            lts.append(float(lt))
    return np.array(seen, dtype=np.int64), np.array(lts), bad


def linear_distillation(hidden, weight, labels, top_ids, top_log_probs, temperature=1.0, ce_weight=0.0,
                        divergence="forward", tail=True, divisor=None, ignore_index=-100, redone=False):
    """dict(loss, divergence, cross_entropy, count, bad, bad_tokens, dh, dw) and what rounding may make of them (``*_off``).

    dZ: all but one listed token of a row are rounded once to bf16 (twice where a row's tiles are ``redone``), in dw the
    rows of ``hidden`` times the row's factor once too, and each result once.
    """
    h, w, y, at, z, off, bad = logits(hidden, weight, labels, temperature, ignore_index)
    c, vocab = ce_weight, w.shape[0]
    lp = log_softmax(z)
    p = np.exp(lp)
    n = at.size
    den = float(n if divisor is None else divisor)
    div, ce, div_off, ce_off = (np.zeros(n) for _ in range(4))
    dz, size = np.zeros_like(z), np.zeros_like(z)
    bad_tokens = 0
    twice = 2 if redone else 1
    for k, row in enumerate(at):
        ids, lt, wrong = named(np.asarray(top_ids)[row], np.asarray(top_log_probs, dtype=np.float64)[row], vocab)
        bad_tokens += wrong
        inside = np.zeros(vocab, dtype=bool)
        inside[ids] = True
        t, s, ls = np.exp(lt), p[k, ids], lp[k, ids]
        has_tail = tail and ids.size < vocab
        m = t.sum()
        r = max(0.0, 1.0 - m)
        if divergence == "reverse":
            r = max(r, 2.0 ** -24)
        others = lp[k, ~inside]
        lq = np.log(np.exp(others - others.max()).sum()) + others.max() if others.size else -np.inf
        q = np.exp(lq)
        e = 2 * off[k] + 2 * SUM + 8 * FP32  # of a probability, relative to it
        if divergence == "forward":
            div[k] = (t * (lt - ls)).sum() + (r * (np.log(r) - lq) if has_tail and r > 0 else 0.0)
            div_off[k] = e * (m + r)
            outer = m + r - r / q if has_tail else m
            inner = s * (m + r if has_tail else m) - t
            size[k, ids] += e * s * (m + r)
            size[k, ~inside] += e * p[k, ~inside] * (m + r + (r / q if has_tail else 0.0))
        else:
            div[k] = (s * (ls - lt)).sum() + (q * (lq - np.log(r)) if has_tail else 0.0)
            dev = np.abs(s * (ls - lt - div[k])).sum() + (abs(q * (lq - np.log(r) - div[k])) if has_tail else 0.0)
            div_off[k] = e * (dev + 1)
            outer = lq - np.log(r) - div[k] if has_tail else 0.0
            inner = s * (ls - lt - div[k])
            size[k, ids] += e * s * (np.abs(ls - lt - div[k]) + 2 + dev)
            size[k, ~inside] += e * p[k, ~inside] * (abs(outer) + 2 + dev)
        ce[k] = -lp[k, y[row]]
        ce_off[k] = e
        dz[k] = (1 - c) * p[k] * outer + c * p[k]
        dz[k, ids] = (1 - c) * inner + c * s
        dz[k, y[row]] -= c
        size[k] *= 1 - c
        size[k] += c * e * p[k]
        size[k, y[row]] += c * 4 * FP32
        listed = np.union1d(ids, [y[row]])
        big = np.abs(dz[k, listed]).max()
        rest = np.setdiff1d(np.arange(vocab), listed)
        if rest.size:  # the others' factor may be held at 2^-20 of the largest listed gradient
            size[k, rest] += 2.0 ** -20 * big * p[k, rest] / max(p[k, rest].sum(), 1e-300)
    dz /= den * temperature
    size /= den * temperature
    rounded = HALF * np.abs(dz)
    # (of the listed ones the largest is not rounded; nothing is made of that here)
    loss = (1 - c) * div + c * ce
    loss_off = (1 - c) * div_off + c * ce_off
    with np.errstate(invalid="ignore", divide="ignore"):
        out = {"loss": loss.sum() / den, "divergence": div.sum() / den, "cross_entropy": ce.sum() / den,
               "loss_off": loss_off.sum() / den, "divergence_off": div_off.sum() / den, "cross_entropy_off": ce_off.sum() / den}
    for name in ("loss", "divergence", "cross_entropy"):
        out[name + "_off"] += 4 * FP32 * abs(out[name])
    slack = 1.05  # of the products' sums in fp32 and of second-order terms
    dh, dho = np.zeros_like(h), np.zeros_like(h)
    dh[at] = dz @ w
    dho[at] = (twice * rounded + size) @ np.abs(w) + HALF * np.abs(dh[at])
    dw = dz.T @ h[at]
    dwo = ((twice + 1) * rounded + size).T @ np.abs(h[at]) + HALF * np.abs(dw)
    out.update(count=n, bad=bad, bad_tokens=bad_tokens, dh=dh, dw=dw, dh_off=slack * dho + 1e-30, dw_off=slack * dwo + 1e-30,
               dz=dz)
    return out
