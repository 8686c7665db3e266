"""Attention with capped scores and a bias by distance in 64 bits on the CPU, and how far a result may be from it.

The bound adds to attention_oracle.py's what the scores cost, key by key, e_j:

- the product's sum, (D + 2) 2^-24 scale sum |q k|, which the cap's tanh does
  not enlarge;
- a cap C: 2^-20 of the score (the polynomial's 6e-7 and seven roundings), or,
  where the exponential is used, 2^-22 C (its own error, the quotient's, and the
  difference from C);
- a bias b: its product with the distance and its rounded slope, the sum with
  the score and the score's own last place: 3 2^-24 (|score| + |b|).

Weights move by e_j, the row's maximum by that of its key: to first order an
output is off by sum p_j (|v_j| + |out|) e_j / sum p, a logarithm of the sum by
sum p_j e_j / sum p.
"""
import math

import numpy as np

from attention_oracle import ROUNDOFF


def scored(q, k, v, limits, dtype, scale=None, cap=0.0, slopes=None, places=None):
    """q (rows, heads, D), k, v (keys, kv_heads, D) in 64 bits; row i sees the first limits[i] keys and stands at
    places[i] (None: at its last key).  Returns out, its bound, lse (heads, rows), its bound."""
    rows, heads, dim = q.shape
    keys, group = k.shape[0], heads // k.shape[1]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    u, tiny = ROUNDOFF[dtype], 2.0 ** -25 if dtype == "fp16" else 0.0
    limits = np.asarray(limits)
    places = limits - 1 if places is None else np.asarray(places)
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    lse, lse_tol = np.full((heads, rows), -math.inf), np.zeros((heads, rows))
    if not keys or not rows:
        return out, tol, lse, lse_tol
    seen = np.arange(keys)[None, :] < limits[:, None]
    some = limits > 0
    distance = np.abs(places[:, None] - np.arange(keys)[None, :]).astype(np.float64)
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
            x = scale * (q[:, h] @ kk.T)
            e = (dim + 2) * 2.0 ** -24 * scale * (np.abs(q[:, h]) @ np.abs(kk).T)
            if cap:
                x = cap * np.tanh(x / cap)
                e = np.where(np.isfinite(e), e, 0.0) + np.abs(x) * 2.0 ** -20 + cap * 2.0 ** -22
            if slopes is not None:
                b = slopes[h] * distance
                x = x - b
                e = e + 3 * 2.0 ** -24 * (np.abs(x) + np.abs(b))
            x = np.where(seen, x, -math.inf)
            e = np.where(seen, e, 0.0)
            top = x.max(1, keepdims=True)
            p = np.exp(x - np.where(some[:, None], top, 0.0))
            total = np.where(some, p.sum(1), 1.0)[:, None]
            y = p @ vv / total
            mass = p @ np.abs(vv) / total
            moved = (p * e) @ np.abs(vv) / total + np.abs(y) * (p * e).sum(1, keepdims=True) / total
            arith = (limits[:, None] + 40 + 3 * np.abs(np.where(some[:, None], top, 0.0))) * 2.0 ** -24
            n = limits[:, None]
            bound = 1.25 * (moved + mass * (u + arith) + u * np.abs(y) + (n * np.abs(vv).max() / total + 1) * tiny)
            out[some, h], tol[some, h] = y[some], bound[some]
            if some.any():
                lse[h, some] = (top + np.log(total))[some, 0]
                off = (p * e).sum(1, keepdims=True) / total + arith
                far = 0.0 if slopes is None else abs(slopes[h]) * np.maximum(-places, 0)[:, None] * 2.0 ** -23
                lse_tol[h, some] = 1.25 * (off + far + np.abs(lse[h][:, None]) * 2.0 ** -23)[some, 0]
    return out, tol, lse, lse_tol
