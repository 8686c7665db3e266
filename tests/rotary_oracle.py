"""Norms and rotations of heads in 64 bits on the CPU, and how far a result may be from them.

The bound of a channel follows from the kernels' number formats, with u the
unit roundoff of the output's type (2^-11 for fp16, 2^-8 for bf16), p the
position, m the magnitude, and n_a, n_b the channel and its partner after the
norm (without one, the inputs):

- a cosine or sine is off by the rounding of its angle (2^-24, of at most
  pi / 4), of the polynomial's value (2^-24, its own error of 2e-9 among them)
  and of the product with m (2^-24): 3 2^-24 m; the frequency's last place adds
  |p| 2^-63 turns, of which |p| 2^-60 is more than enough in radians;
- two products and a sum: 2 2^-24 m (|n_a| + |n_b|);
- the norm: its D squares' sum, (D + 1) 2^-24 of it and half that of the root,
  the mean, the root and the quotient 4 2^-24, the products with w and the
  root 2 2^-24;
- the output is rounded once: u |y|, 2^-25 where fp16 is subnormal.

First-order terms are summed and the sum is taken 1.25 times for the rest.
"""
import numpy as np

from attention_oracle import ROUNDOFF


def pairs(dims, interleaved):
    i = np.arange(dims // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + dims // 2)


def ready(x, dtype, positions=None, frequencies=(), interleaved=False, magnitude=1.0, weight=None, eps=0.0):
    """x (tokens, heads, D) in 64 bits, normed and rotated; the bound of each element."""
    dim, dims = x.shape[-1], 2 * len(frequencies)
    n, rel = x, 0.0
    with np.errstate(invalid="ignore", over="ignore"):
        if weight is not None:
            n = x * weight / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
            rel = (dim / 2 + 7) * 2.0 ** -24
        y, tol = n.copy(), np.abs(n) * rel
        if dims:
            a, b = pairs(dims, interleaved)
            angle = np.asarray(positions).astype(np.longdouble)[:, None] * np.asarray(frequencies).astype(np.longdouble)
            c, s = (magnitude * f(angle).astype(np.float64)[:, None] for f in (np.cos, np.sin))
            y[..., a], y[..., b] = n[..., a] * c - n[..., b] * s, n[..., b] * c + n[..., a] * s
            both = abs(magnitude) * (np.abs(n[..., a]) + np.abs(n[..., b]))
            far = np.abs(np.asarray(positions, np.float64))[:, None, None] * 2.0 ** -60
            tol[..., a] = tol[..., b] = both * (rel + 5 * 2.0 ** -24 + far)
        tol = 1.25 * (tol + ROUNDOFF[dtype] * np.abs(y) + (2.0 ** -25 if dtype == "fp16" else 0.0))
    return y, tol
