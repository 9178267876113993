"""Token statistics (log-probabilities, entropies, most probable tokens) and their
gradients in numpy and 64 bits (written from the definitions; nothing of the
package is used)."""

from __future__ import annotations

import numpy as np

HALF = 2.0 ** -8  # half a step of bf16, relative to the value
FP32 = 2.0 ** -24  # ... of fp32
# fp32 sums of a part of a row: 64 terms one after the other and two halves, the exponential's own error and that of its
# argument, weighed with the terms
SUM = 72 * FP32


def logits(hidden, weight, labels, temperature, ignore_index):
    """Rows that count, their logits over ``temperature`` and what fp32 sums of hdim products, 16 at once, may make of them."""
    h, w = (np.asarray(x, dtype=np.float64) for x in (hidden, weight))
    y = np.asarray(labels, dtype=np.int64)
    known = (y >= 0) & (y < w.shape[0])
    at = np.flatnonzero((y != ignore_index) & known)
    z = h[at] @ w.T / temperature
    depth = h.shape[1] / 8 + 4
    off = depth * FP32 * (np.abs(h[at]) @ np.abs(w).T).max(1, initial=0.0) / temperature
    off += 2 * FP32 * np.abs(z).max(1, initial=0.0)  # (the scale's rounding)
    return h, w, y, at, z, off, int(((y != ignore_index) & ~known).sum())


def log_softmax(z):
    z = z - z.max(1, keepdims=True, initial=-np.inf) if z.size else z
    return z - np.log(np.exp(z).sum(1, keepdims=True))


def linear_token_stats(hidden, weight, labels, top_k=0, dlogp=None, dentropy=None, temperature=1.0, ignore_index=-100,
                       roundings=1):
    """dict(logp, entropy, count, bad, at, z, off): ``at`` the counted rows, ``off`` what their logits may be off by;
    ``logp_off`` and ``entropy_off`` follow from it.  With ``top_k`` also ``top_ids``, each row's tokens by falling logit
    (equal ones by id; -1 in rows that do not count).

    With upstream gradients also dh and dw, and ``dh_off`` / ``dw_off``: each element of dZ but the given token's rounded
    ``roundings`` times to bf16 (the first of them before a logarithm is taken, where there are two), and the result once.
    """
    h, w, y, at, z, off, bad = logits(hidden, weight, labels, temperature, ignore_index)
    rows = np.arange(at.size)
    lp = log_softmax(z)
    p = np.exp(lp)
    with np.errstate(invalid="ignore"):
        plp = np.where(p > 0, p * lp, 0.0)
    ent = -plp.sum(1)
    out = {"count": at.size, "bad": bad, "z": z, "off": off, "at": at}
    for name, v in (("logp", lp[rows, y[at]]), ("entropy", ent)):
        out[name] = np.zeros(y.size)
        out[name][at] = v
    slope = np.abs(p * (lp + ent[:, None]))  # of the entropy, by logit
    out["logp_off"], out["entropy_off"] = np.zeros(y.size), np.zeros(y.size)
    out["logp_off"][at] = 2 * off + SUM + 4 * FP32 * np.abs(lp[rows, y[at]])
    out["entropy_off"][at] = off * slope.sum(1) + SUM * (1 + 2 * np.abs(plp).sum(1)) + 4 * FP32 * ent
    if top_k:
        order = np.argsort(-z, axis=1, kind="stable")[:, :top_k]
        out["top_ids"] = np.full((y.size, top_k), -1, dtype=np.int64)
        out["top_ids"][at] = order
        out["top_logp"] = np.zeros((y.size, top_k))
        out["top_logp"][at] = np.take_along_axis(lp, order, 1)
        out["lp"] = lp
    if dlogp is not None or dentropy is not None:
        none = np.zeros(y.size)
        g, e = (np.asarray(none if x is None else x, dtype=np.float64)[at, None] / temperature for x in (dlogp, dentropy))
        dz = -p * (g + e * (lp + ent[:, None]))
        soft = np.abs(dz)
        if roundings > 1:  # a rounded numerator's logarithm is off by as much
            soft = roundings * soft + np.abs(e) * p
        soft[rows, y[at]] = 0.0
        # the logits', the sums' and the entropy's errors, relative to p or to its logarithm
        rel = (2 * off + 2 * SUM + 8 * FP32)[:, None]
        fine = rel * p * (np.abs(g) + np.abs(e) * (np.abs(lp + ent[:, None]) + 1 + np.abs(ent[:, None])))
        dz[rows, y[at]] += g[:, 0]
        fine[rows, y[at]] += rel[:, 0] * (np.abs(g) + np.abs(e))[:, 0] + 8 * FP32 * np.abs(dz[rows, y[at]])
        size = HALF * soft + fine
        slack = 1.05  # of the products' sums in fp32 and of second-order terms
        dh, dho = np.zeros_like(h), np.zeros_like(h)
        dh[at] = dz @ w
        dho[at] = size @ np.abs(w) + HALF * np.abs(dh[at])
        dw = dz.T @ h[at]
        dwo = size.T @ np.abs(h[at]) + HALF * np.abs(dw)
        out.update(dh=dh, dw=dw, dh_off=slack * dho + 1e-30, dw_off=slack * dwo + 1e-30)
    return out
