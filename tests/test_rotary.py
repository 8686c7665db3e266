"""Rotary frequencies, and what the binding and the C entry points refuse of positions and norms (CPU)."""
import ctypes
import math
import types

import numpy as np
import pytest

from test_attention_arguments import array_on


@pytest.mark.parametrize("dims", [2, 4, 20, 64, 126, 128])
@pytest.mark.parametrize("base", [10000.0, 500000.0, 1.0])
def test_frequencies(cvs, dims, base):
    f = np.array([base ** (-2 * i / dims) for i in range(dims // 2)])
    np.testing.assert_allclose(cvs.rotary_frequencies(dims, base), f, rtol=1e-14)
    np.testing.assert_allclose(cvs.rotary_frequencies(dims, base, "linear", 8.0), f / 8, rtol=1e-14)
    if dims > 2:
        scaled = base * 4.0 ** (dims / (dims - 2))
        want = [scaled ** (-2 * i / dims) for i in range(dims // 2)]
        got = cvs.rotary_frequencies(dims, base, "base", 4.0)
        np.testing.assert_allclose(got, want, rtol=1e-13)
        assert got[0] == 1.0 and math.isclose(got[-1], f[-1] / 4, rel_tol=1e-13)
    got = cvs.rotary_frequencies(dims, base, "turns", 16.0, 8192, 1.0, 32.0)
    for x, y in zip(got, f):
        n = 8192 * y / (2 * math.pi)
        want = y if n > 32 else y / 16 if n < 1 else y * ((n - 1) / 31 + (32 - n) / 31 / 16)
        assert math.isclose(x, want, rel_tol=1e-12)


@pytest.mark.parametrize("bad", [dict(dims=0), dict(dims=3), dict(dims=130), dict(dims=-2), dict(base=0.5),
                                 dict(base=math.inf), dict(base=math.nan), dict(scaling="linear", factor=0.0),
                                 dict(scaling="base", factor=2.0, dims=2), dict(scaling="linear", factor=math.nan),
                                 dict(scaling="turns", factor=2.0),
                                 dict(scaling="turns", factor=2.0, original_length=10, low=4, high=4),
                                 dict(scaling="turns", factor=2.0, original_length=10, low=-1, high=4),
                                 dict(scaling="turns", factor=2.0, original_length=math.inf), dict(scaling="other")])
def test_frequencies_refused(cvs, bad):
    with pytest.raises(ValueError):
        cvs.rotary_frequencies(**{"dims": 64, **bad})


def test_null_arguments_are_refused(cvs):
    lib, bad, h = cvs.load(), cvs.CVS_ERR_INVALID_ARGUMENT, ctypes.c_void_p()
    f, view = (ctypes.c_double * 4)(), cvs.Heads()
    assert lib.cvs_rotary_frequencies(8, 1e4, None, None) == bad
    assert lib.cvs_rotary_frequencies(8, 1e4, None, f) == cvs.CVS_OK and f[0] == 1.0
    assert lib.cvs_rotary_frequencies(8, 1e4, cvs.RotaryScaling(9, 1.0, 1.0, 1.0, 2.0), f) == bad
    assert lib.cvs_rotary_create(None, 8, 0, f, 1.0, ctypes.byref(h)) == bad
    assert lib.cvs_rotate_async(None, None, None, view, view) == bad
    assert lib.cvs_norm_rotate_async(None, None, None, view, view, None, None, None, None) == bad
    assert "null" in lib.cvs_last_error().decode()
    assert lib.cvs_rotary_destroy(None) == cvs.CVS_OK


def test_arrays_the_binding_refuses(cvs):
    ctx = types.SimpleNamespace(device=0)
    at = lambda device, shape, dtype: array_on(cvs, device, shape, dtype)
    assert cvs._vector(ctx, at(0, (5,), np.int64), "positions", 5, ("int64",)) == (4096, "int64")
    for x in (at(0, (4,), np.int64), at(0, (5, 1), np.int64), at(0, (5,), np.int32), at(0, (5,), np.float64)):
        with pytest.raises(ValueError, match="positions must be 5 elements of int64"):
            cvs._vector(ctx, x, "positions", 5, ("int64",))
    with pytest.raises(ValueError, match="on the context's device"):
        cvs._vector(ctx, at(1, (5,), np.int64), "positions", 5, ("int64",))
    heads = cvs.Heads(4096, 1, 64, 64, 1, 64, cvs.BF16)
    assert cvs._norm(ctx, None, heads, 1e-6, "w") is None
    assert cvs._norm(ctx, at(0, (64,), np.float32), heads, 1e-6, "w").type == cvs.FP32
    assert cvs._norm(ctx, at(0, (64,), np.uint16), heads, 1e-6, "w").type == cvs.BF16
    for x in (at(0, (64,), np.float16), at(0, (63,), np.float32), at(0, (64,), np.float64)):
        with pytest.raises(ValueError, match="w must be 64 elements"):
            cvs._norm(ctx, x, heads, 1e-6, "w")


def test_a_closed_rotary_is_not_none(cvs):
    """A closed rotary's handle is None, which C takes for a call without rotation."""
    assert cvs._open(None) is None
    assert cvs._open(types.SimpleNamespace(handle=5)) == 5
    with pytest.raises(ValueError, match="closed"):
        cvs._open(types.SimpleNamespace(handle=None))
