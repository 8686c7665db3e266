"""Angles of far positions at frequencies of many turns a position, against exact integers on the CPU.

The bound of a cosine or sine: the frequency's part of a turn is held to 2^-65, so |p| 2^-64 turns at position p are more
than enough; the rest of the angle is cut at 2^-32 turns; then rotary_oracle.py's 3 2^-24 and the output's rounding.
"""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

from attention_oracle import f64

pytestmark = pytest.mark.gpu

BITS = 400


def inverse_tangent(n):
    """atan(1 / n) in units of 2^-BITS."""
    term = total = (1 << BITS) // n
    k, sign = 1, -1
    while term:
        term //= n * n
        k += 2
        total += sign * (term // k)
        sign = -sign
    return total


TWO_PI = 8 * (4 * inverse_tangent(5) - inverse_tangent(239))


def rest(position, radians):
    """position * radians less whole turns, in radians: from -pi to pi."""
    f = Fraction(radians) * position
    angle = (f.numerator << BITS) // f.denominator % TWO_PI
    return (angle - TWO_PI if angle > TWO_PI // 2 else angle) / (1 << BITS)


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kind", ["trained", "a turn", "many turns", "tiny"])
def test_far_positions(tctx, kind, interleaved):
    rng = np.random.default_rng(3)
    f = {"trained": 10000.0 ** (-np.arange(64) / 64), "a turn": 2 * np.pi * (1 + rng.standard_normal(64) * 1e-3),
         "many turns": np.concatenate([[1024.0, -1024.0, 1023.999, -0.0], rng.uniform(-1024, 1024, 60)]),
         "tiny": 2.0 ** -rng.uniform(20, 70, 64) * rng.choice([-1, 1], 64)}[kind]
    at = [0, 1, -1, 7, 10 ** 6, 2 ** 31 + 1, 2 ** 40 + 12345, -2 ** 43 - 99, 2 ** 45 + 1, 2 ** 46 - 12345, -10 ** 13]
    x = torch.zeros(len(at), 1, 128, dtype=torch.float16, device="cuda")
    (x[..., 0::2] if interleaved else x[..., :64]).fill_(1.0)
    out = torch.zeros_like(x)
    tctx.rotate_async(tctx.rotary(128, frequencies=f, interleaved=interleaved),
                      torch.tensor(at, dtype=torch.int64, device="cuda"), x, out)
    got = f64(out)[:, 0]
    cos, sin = (got[:, 0::2], got[:, 1::2]) if interleaved else (got[:, :64], got[:, 64:])
    angle = np.array([[rest(p, float(r)) for r in f] for p in at])
    far = 2 * math.pi * (np.abs(np.array(at, np.float64))[:, None] * 2.0 ** -64 + 2.0 ** -32)
    for value, want in ((cos, np.cos(angle)), (sin, np.sin(angle))):
        room = 1.25 * (far + 3 * 2.0 ** -24 + 2.0 ** -11 * np.abs(want) + 2.0 ** -25)
        assert (np.abs(value - want) <= room).all(), (np.abs(value - want) / room).max()
