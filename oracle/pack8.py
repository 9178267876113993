"""8-bit storage of activations and the gated MLP activation over it, in numpy
and 64 bits (written from the definitions; nothing of the package is used)."""

from __future__ import annotations

import numpy as np

GROUP = 32


def _e4m3_values() -> np.ndarray:
    """The 256 OCP e4m3 numbers (bias 7, no infinities, 0x7f / 0xff NaN)."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        v = np.nan if (e, m) == (15, 7) else (m / 8 * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
        out[c] = -v if c & 128 else v
    return out


E4M3 = _e4m3_values()


def encode(x: np.ndarray, fmt: str):
    """``(codes uint8 [n], scales uint8 [ceil(n / 32)])`` of a flat fp32 / bf16-valued array."""
    x = np.asarray(x, dtype=np.float64).reshape(-1)
    n = x.size
    groups = np.concatenate([x, np.zeros(-n % GROUP)]).reshape(-1, GROUP)
    codes = np.zeros(groups.shape, dtype=np.uint8)
    scales = np.empty(groups.shape[0], dtype=np.uint8)
    bits, limit, lowest = (6, 127.5, 7) if fmt == "int8" else (8, 464.0, 9)
    for i, v in enumerate(groups):
        if not np.isfinite(v).all():
            scales[i] = 255
            continue
        a = np.abs(v).max()
        e = int(np.frexp(a)[1]) - 1 if a else -1000  # a in [2^e, 2^(e+1))
        if a and (a / 2.0 ** (e - bits) >= limit if fmt == "int8" else a / 2.0 ** (e - bits) > limit):
            e += 1
        scales[i] = min(max(e + 127, lowest), 254)
        y = v / 2.0 ** (int(scales[i]) - 127 - bits)
        if fmt == "int8":
            codes[i] = np.clip(np.rint(y), -127, 127).astype(np.int8).view(np.uint8)
        else:
            # nearest of the positive numbers, ties to the even code
            pos = E4M3[:127]
            m = np.minimum(np.abs(y), 448.0)
            hi = np.clip(np.searchsorted(pos, m), 0, 126)
            lo = np.maximum(hi - 1, 0)
            up, down = pos[hi] - m, m - pos[lo]
            pick = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
            codes[i] = (pick + 128 * np.signbit(y)).astype(np.uint8)
    return codes.reshape(-1)[:n], scales


def decode(codes: np.ndarray, scales: np.ndarray, fmt: str) -> np.ndarray:
    s = np.repeat(scales.astype(np.int64), GROUP)[:codes.size]
    v = codes.view(np.int8).astype(np.float64) if fmt == "int8" else E4M3[codes]
    return np.where(s == 255, np.nan, v * 2.0 ** (s - (133 if fmt == "int8" else 135)))


def rounded(x: np.ndarray, fmt: str) -> np.ndarray:
    """``x`` as the values its codes stand for."""
    return decode(*encode(x, fmt), fmt).reshape(np.shape(x))


def swiglu(g: np.ndarray, u: np.ndarray) -> np.ndarray:
    return g / (1 + np.exp(-g)) * u


def swiglu_bwd(dh: np.ndarray, g: np.ndarray, u: np.ndarray):
    s = 1 / (1 + np.exp(-g))
    return dh * u * s * (1 + g * (1 - s)), dh * g * s
