"""Norms of heads at the ends of their type's range (cvs_norm_rotate_async, cvs_kv_append_async).

Bounds: rotary_oracle.py.
"""
import pytest
import torch

from attention_oracle import TORCH, assert_within, f64
from rotary_oracle import ready
from test_kv_cache_gpu import bits, rand

pytestmark = pytest.mark.gpu

# Halves that lie whole pieces apart, that do not, neighbours, a part of the channels, no rotation.
ROTARIES = [(64, False), (20, False), (64, True), (32, True), (0, False)]


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def norm(ctx, x, weight, dims, interleaved, eps=1e-6, magnitude=1.0):
    """x as queries from array to array, and as keys into the cache: the same bits."""
    t, heads, dim = x.shape
    out, kept, at = torch.full_like(x, 7.0), torch.full_like(x, 7.0), torch.arange(3, 3 + t, device="cuda")
    rotary = ctx.rotary(dims, interleaved=interleaved, magnitude=magnitude) if dims else None
    ctx.norm_rotate_async(rotary, at if dims else None, x, out, q_weight=weight, eps=eps)
    cache = ctx.kv_cache(1, 2, 32, heads, dim, "bf16" if x.dtype == torch.bfloat16 else "fp16")
    (s,) = cache.sequences(1)
    cache.extend([s], [t])
    plan, v = cache.plan([s], [t]), torch.empty_like(x)
    cache.append_async(plan, x, x, rotary=rotary, positions=at if dims else None, k_weight=weight, eps=eps)
    cache.read_async(plan, kept, v)
    assert torch.equal(bits(kept), bits(out))
    del plan
    cache.close()
    return out


@pytest.mark.parametrize("dims,interleaved", ROTARIES)
@pytest.mark.parametrize("size", [1e20, 2e38, 3.38e38])
def test_heads_beyond_their_squares(tctx, dims, interleaved, size):
    """Heads whose squares pass fp32 come out 0, however large their channels and weights; those beside them as ever."""
    x = rand(1, 5, 3, 64, dtype="bf16")
    x[1, 2] = x[1, 2].sign() * size
    x[4, 0, 7], x[4, 0, 39] = size, size  # a pair of each kind of rotation is large in one of them
    x[2, 1, 6], x[2, 1, 7] = -size, size
    weight = 1.0 + rand(2, 64, dtype="bf16").abs()
    out = norm(tctx, x, weight, dims, interleaved, magnitude=1.5)
    large = torch.zeros(5, 3, dtype=torch.bool, device="cuda")
    large[1, 2] = large[4, 0] = large[2, 1] = True
    assert (out[large] == 0).all()
    f = () if not dims else [10000.0 ** (-2 * i / dims) for i in range(dims // 2)]
    want, tol = ready(f64(x), "bf16", range(3, 8), f, interleaved, 1.5, f64(weight), 1e-6)
    rest = ~large.cpu().numpy()
    assert_within(f64(out)[rest], want[rest], tol[rest], "beside them")


@pytest.mark.parametrize("dims,interleaved", ROTARIES)
@pytest.mark.parametrize("size,w", [(1e10, 1e32), (1e-12, 1e-30), (1e15, 1e-20), (1e-15, 1e20), (3e16, 3e33)])
def test_products_with_weights_of_any_size(tctx, dims, interleaved, size, w):
    """A channel times its weight may leave fp32 where the normed one does not."""
    x = (rand(1, 5, 3, 64, dtype="bf16").float() * size).to(torch.bfloat16)
    weight = ((1.0 + rand(2, 64, dtype="bf16").float().abs()) * w).to(torch.bfloat16)
    out = norm(tctx, x, weight, dims, interleaved, eps=0.0)
    f = () if not dims else [10000.0 ** (-2 * i / dims) for i in range(dims // 2)]
    want, tol = ready(f64(x), "bf16", range(3, 8), f, interleaved, 1.0, f64(weight), 0.0)
    assert_within(f64(out), want, tol, "normed")


@pytest.mark.parametrize("dims,interleaved", ROTARIES)
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_infinite_channels(tctx, dims, interleaved, dtype):
    """The formula's: a head with an infinity has an infinite norm, so that it is NaN where the infinity goes, else 0."""
    x = rand(1, 4, 3, 64, dtype=dtype)
    x[2, 1, 5] = float("-inf")
    weight = torch.ones(64, dtype=TORCH[dtype], device="cuda")
    out = norm(tctx, x, weight, dims, interleaved)
    where = torch.zeros(64, dtype=torch.bool, device="cuda")
    where[5] = True
    if dims:
        where[4 if interleaved else 5 + dims // 2 if 5 < dims // 2 else 5 - dims // 2] = True
    assert torch.isnan(out[2, 1][where]).all() and (out[2, 1][~where] == 0).all()
    rest = torch.ones(4, 3, dtype=torch.bool, device="cuda")
    rest[2, 1] = False
    assert torch.isfinite(out[rest]).all()
