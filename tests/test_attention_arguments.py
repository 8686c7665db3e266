"""What the binding refuses of attention's arrays before any call (CPU)."""
import types

import numpy as np
import pytest


def array_on(cvs, device, shape, dtype):
    """A DeviceArray without memory."""
    a = cvs.DeviceArray.__new__(cvs.DeviceArray)
    a.ctx = types.SimpleNamespace(device=device, handle=None)
    a.shape, a.dtype, a.ptr = shape, np.dtype(dtype), types.SimpleNamespace(value=4096)
    return a


def test_arrays_of_another_device(cvs):
    ctx = types.SimpleNamespace(device=0)
    view, layers, _ = cvs._heads(ctx, array_on(cvs, 0, (5, 2, 64), np.float16), "q")
    assert (view.data, view.tokens, view.heads, view.head_dim, layers) == (4096, 5, 2, 64, 1)
    with pytest.raises(ValueError, match="q must be on the context's device"):
        cvs._heads(ctx, array_on(cvs, 1, (5, 2, 64), np.float16), "q")
    assert cvs._lse(ctx, array_on(cvs, 0, (2, 5), np.float32), 2, 5) is not None
    with pytest.raises(ValueError, match="lse must be on the context's device"):
        cvs._lse(ctx, array_on(cvs, 1, (2, 5), np.float32), 2, 5)
