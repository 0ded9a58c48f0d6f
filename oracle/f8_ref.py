"""Block-scaled e4m3 in 64 bits: the definition that rms_f8, quant_f8 and gemm_f8 are checked against."""
from __future__ import annotations

import numpy as np

from h3metal_b200 import quant

G = quant.F8_GROUP


def norm_rows(h: np.ndarray, w: np.ndarray, eps: float) -> np.ndarray:
    h = h.astype(np.float64)
    return h / np.sqrt((h * h).mean(1, keepdims=True) + eps) * w.astype(np.float64)


def gated_rows(x: np.ndarray, D: int) -> np.ndarray:
    v, g = x[:, :D].astype(np.float64), x[:, D:2 * D].astype(np.float64)
    with np.errstate(over="ignore"):
        return v * (g / (1 + np.exp(-g)))


def scales(v: np.ndarray) -> np.ndarray:
    """[groups][rows] fp64: a group's largest magnitude / 448 (NaN left out), at least 2^-126; 1 for zeros."""
    m, d = v.shape
    top = np.zeros((-(-d // G), m))
    for g in range(top.shape[0]):
        top[g] = np.nanmax(np.abs(np.nan_to_num(v[:, g * G:(g + 1) * G], nan=0.0, posinf=np.inf, neginf=-np.inf)), axis=1)
    return np.where(top > 0, np.maximum(top / 448.0, 2.0 ** -126), 1.0)


def spread(s: np.ndarray, D: int) -> np.ndarray:
    """Group scales [groups][rows] -> one per value [rows][D]."""
    return np.repeat(s.T, G, axis=1)[:, :D]


def product(a: np.ndarray, sa: np.ndarray, w: np.ndarray, sw: np.ndarray, K: int, bias=None):
    """(C, S): codes a [M][>= K], w [N][>= K] (bytes), sa [groups][M], sw [ceil(N/128)][groups]; S[m][n] is the same sum
    over magnitudes, the yardstick of rounding errors."""
    av = quant.e4m3_to_f32(a[:, :K]).astype(np.float64) * spread(sa.astype(np.float64), K)
    wv = quant.e4m3_to_f32(w[:, :K]).astype(np.float64)
    wv *= np.repeat(np.repeat(sw.astype(np.float64), G, axis=0)[:len(w)], G, axis=1)[:, :K]
    c, s = av @ wv.T, np.abs(av) @ np.abs(wv).T
    return (c, s) if bias is None else (c + bias.astype(np.float64), s + np.abs(bias))
