"""Log-probabilities of labels and their gradients in numpy and 64 bits
(written from the definitions; nothing of the package is used)."""

from __future__ import annotations

import numpy as np

HALF = 2.0 ** -8  # half a step of bf16, relative to the value


def linear_log_probs(hidden, weight, labels, dlogp=None, temperature=1.0, ignore_index=-100):
    """dict(logp, count, bad) and, with the upstream gradients ``dlogp``, dh and
    dw with what rounding to bf16 may make of them: ``dh_off`` / ``dw_off``, each
    softmax numerator (and each scaled row of ``hidden`` in dw) rounded once to
    bf16 and the result once more."""
    h, w = (np.asarray(x, dtype=np.float64) for x in (hidden, weight))
    y = np.asarray(labels, dtype=np.int64)
    known = (y >= 0) & (y < w.shape[0])
    at = np.flatnonzero((y != ignore_index) & known)
    z = h[at] @ w.T / temperature
    top = z.max(1, keepdims=True) if at.size else np.zeros((0, 1))
    e = np.exp(z - top)
    total = e.sum(1, keepdims=True)
    rows = np.arange(at.size)
    logp = np.zeros(y.size)
    logp[at] = z[rows, y[at]] - top[:, 0] - np.log(total[:, 0])
    out = {"logp": logp, "count": at.size, "bad": int(((y != ignore_index) & ~known).sum())}
    # sums of hdim products in fp32, 16 of them at once
    depth = h.shape[1] / 8 + 4
    out["logp_off"] = np.zeros(y.size)
    if at.size:
        out["logp_off"][at] = 2 * depth * 2.0 ** -24 * (np.abs(h[at]) @ np.abs(w).T).max(1) / temperature
    out["logp_off"] += 1e-6 + 4 * 2.0 ** -24 * np.abs(logp)
    if dlogp is not None:
        g = np.asarray(dlogp, dtype=np.float64)[at, None] / temperature
        p = e / total
        dz = -g * p
        soft = np.abs(dz)
        soft[rows, y[at]] = 0.0
        dz[rows, y[at]] += g[:, 0]
        # label terms are in fp32: the probability's own error there
        label = np.abs(g) * (8 * 2.0 ** -24 + out["logp_off"][at, None])
        dh = np.zeros_like(h)
        dh[at] = dz @ w
        slack = 1.05  # of the sums in fp32 and of second-order terms
        off = np.zeros_like(h)
        off[at] = HALF * (soft @ np.abs(w)) + label * np.abs(w[y[at]]) + HALF * np.abs(dh[at])
        off[at] += out["logp_off"][at, None] * (soft @ np.abs(w))
        dw = dz.T @ h[at]
        dwo = 2 * HALF * (soft.T @ np.abs(h[at])) + HALF * np.abs(dw)
        dwo += (out["logp_off"][at, None] * soft).T @ np.abs(h[at])
        np.add.at(dwo, y[at], label * np.abs(h[at]))
        out.update(dh=dh, dw=dw, dh_off=slack * off + 1e-30, dw_off=slack * dwo + 1e-30)
    return out
