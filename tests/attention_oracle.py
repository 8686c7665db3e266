"""Attention in 64 bits on the CPU, and how far a result may be from it.

The bound of an output element follows from the kernels' number formats, with
u the unit roundoff of the operands' type (2^-11 for fp16, 2^-8 for bf16), D
the head size, n the number of keys a row sees, p the softmax weights of the
row scaled to a largest one of 1, and A = sum p |v| / sum p:

- a score is a sum of D products in 32 bits, off by at most (D + 2) 2^-24
  sum |q k| times the scale; weights move by the factor e^2d, d the largest
  such error of the row (its own and the maximum's);
- the exponential and the sums over keys: n + 8 roundings of 2^-24 each, and
  the log2-scaled score rounded once, |m| 2^-24 in the exponent;
- each weight is rounded to the operands' type: u A, and where that type is
  fp16 a weight below 2^-14 is off by up to 2^-25: n 2^-25 max |v| / sum p;
- a row is joined from parts and rescaled a few times: 32 more roundings;
- the output is rounded once: u |out|, 2^-25 where fp16 is subnormal.

First-order terms are summed and the sum is taken 1.25 times for the rest.
"""
import math

import numpy as np
import torch

TORCH = {"fp16": torch.float16, "bf16": torch.bfloat16}
ROUNDOFF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def attention(q, k, v, limits, dtype, scale=None):
    """q (rows, heads, D), k, v (keys, kv_heads, D) in 64 bits; row i sees the
    first limits[i] keys.  Returns out, its bound, lse (heads, rows), its bound."""
    rows, heads, dim = q.shape
    group = heads // k.shape[1]
    scale = 1.0 / math.sqrt(dim) if scale is None else scale
    u = ROUNDOFF[dtype]
    out = np.zeros((rows, heads, dim))
    tol = np.zeros((rows, heads, dim))
    lse = np.full((heads, rows), -math.inf)
    lse_tol = np.zeros((heads, rows))
    for i in range(rows):
        n = int(limits[i])
        if n <= 0:
            continue
        for h in range(heads):
            kk, vv = k[:n, h // group], v[:n, h // group]
            with np.errstate(invalid="ignore", over="ignore"):
                x = scale * (kk @ q[i, h])
                top = x.max()
                p = np.exp(x - top)
                total = p.sum()
                # 0 * inf is not a term of the sum: weights are positive, however small.
                out[i, h] = p @ vv / total
                mass = p @ np.abs(vv) / total
                d = (dim + 2) * 2.0 ** -24 * scale * (np.abs(kk) @ np.abs(q[i, h])).max()
                arith = 2 * d + (n + 40 + 2 * abs(top) * 1.5) * 2.0 ** -24
                tol[i, h] = 1.25 * (mass * (u + arith) + u * np.abs(out[i, h])
                                    + (n * np.abs(vv).max() / total + 1) * (2.0 ** -25 if dtype == "fp16" else 0.0))
                lse[h, i] = top + math.log(total)
                lse_tol[h, i] = 1.25 * (arith + abs(lse[h, i]) * 2.0 ** -23)
    return out, tol, lse, lse_tol


def f64(x):
    """A torch tensor's values in 64 bits."""
    return x.detach().double().cpu().numpy()


def assert_within(got, want, tol, what):
    """Within the bound where the value is finite, and the same infinities and NaNs elsewhere."""
    fine = np.isfinite(want)
    np.testing.assert_array_equal(np.isnan(got), np.isnan(want), err_msg=what)
    with np.errstate(invalid="ignore"):
        np.testing.assert_array_equal(got[~fine & ~np.isnan(want)], want[~fine & ~np.isnan(want)], err_msg=what)
        off = np.where(fine, np.abs(got - want), 0.0)
    room = np.where(fine, tol, 1.0)
    worst = (off - room).max() if off.size else -1.0
    assert worst <= 0, f"{what}: {(off / np.maximum(room, 1e-300)).max():.3g} times the bound"
