"""Attention with scores whose last place in 32 bits is more than 1: the largest one still has its whole weight, equal ones
share it evenly, and rows with small scores beside them keep their bits.  Plain, capped and biased; prompts and the cache."""
import numpy as np
import pytest
import torch

from attention_oracle import TORCH, f64
from test_kv_cache_gpu import Filled, bits, rand

pytestmark = pytest.mark.gpu

KINDS = ["plain", "cap", "bias", "both"]
# Products of the rows' one channel and their keys' times the scale.
SIZES = [3e5, 1.3e7, 2e7, 2e8, 1.7e9, 5e9, 3e11, 7e14]
ROUNDOFF = {"fp16": 2.0 ** -11, "bf16": 2.0 ** -8}


def unsure(size):
    """How far weights of equal scores may be apart: below 2^24 in log2 units a score less its row's largest is one rounding
    in some tiles, and two in others."""
    m = size * 1.4427
    return np.expm1(m * 2.0 ** -23) if m < 2.0 ** 24 else 0.0


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def options(kind, heads, size):
    """A cap that such scores are beyond, or slopes that only tell equal ones apart: by less than their last places."""
    slopes = torch.full((heads,), size * 2.0 ** -60, device="cuda") if kind in ("bias", "both") else None
    return dict(cap=20.0 * size if kind in ("cap", "both") else 0.0, slopes=slopes)


def loud(size, scale, rows, heads, dtype, seed=1):
    """Queries of one channel: products with keys of 64 there are +-size / scale."""
    q = torch.zeros(rows, heads, 64)
    q[..., 3] = size / scale / 64.0
    q[1::2, ..., 3] *= -1.0
    return q.to(TORCH[dtype]).cuda()


def quiet(q, k, seed):
    """Every third row, and the keys, in another channel, of which loud rows see nothing."""
    q[::3] = 0.0
    q[::3, ..., 7] = rand(seed, *q[::3, ..., 7].shape, dtype="fp16").to(q.dtype)
    k[..., 7] = rand(seed + 1, *k[..., 7].shape, dtype="fp16").to(k.dtype)


def same(got, want, size, dtype, what):
    """A weight of 1 gives its value's bits; one near 1, rounded to the type, is beside one that is not: 2^-8, 2^-11."""
    if unsure(size):
        assert (np.abs(f64(got) - f64(want)) <= 2.5 * ROUNDOFF[dtype] * np.abs(f64(want)) + 2.0 ** -24).all(), what
    else:
        assert torch.equal(bits(got), bits(want)), what


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("keys", [1, 40, 300])
def test_equal_keys_share_evenly(tctx, dtype, kind, size, keys):
    heads, kv, rows, scale = 4, 2, 70, max(1.0, size / 1e6)
    q = loud(size, scale, rows, heads, dtype)
    k = torch.zeros(keys, kv, 64, dtype=TORCH[dtype], device="cuda")
    k[..., 3] = 64.0
    v = rand(2, keys, kv, 64, dtype=dtype)
    opts, out, lse = options(kind, heads, size), torch.full_like(q, 7.0), torch.zeros(heads, rows, device="cuda")
    tctx.prompt_attention_async(tctx.prompt_plan([rows], heads, kv, [keys], causal=False), q, k, v, out, lse, scale, **opts)
    mean, size_v = f64(v).mean(0).repeat(2, axis=0), np.abs(f64(v)).mean(0).repeat(2, axis=0)
    # A weight is rounded to the type, sums and the quotient are in 32 bits, the output is rounded.
    u = ROUNDOFF[dtype]
    room = (u + unsure(size) + 400 * 2.0 ** -24) * size_v + u * np.abs(mean)
    assert (np.abs(f64(out) - mean) <= 1.25 * room + 2.0 ** -24).all()
    real = scale * f64(q)[:, :, 3].T * 64.0
    if opts["cap"]:
        real = opts["cap"] * np.tanh(real / opts["cap"])
    off = np.abs(f64(lse) - real - np.log(keys))
    # The score, its cap's 2^-20 and 2^-22 of the cap, the last places of a logarithm: 2^-22 of all.
    assert (off <= 1.25 * ((2.0 ** -22 + 2.0 ** -20 * bool(opts["cap"])) * np.abs(real) + opts["cap"] * 2.0 ** -22 + 1e-4)).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("size", SIZES)
def test_the_largest_takes_all(tctx, dtype, kind, size):
    """One key's score is an eighth larger, wherever it stands: its value is the result."""
    heads, kv, rows, scale = 4, 2, 5, max(1.0, size / 1e6)
    q = loud(size, scale, rows, heads, dtype).abs()
    v, opts = rand(2, 300, kv, 64, dtype=dtype), options(kind, heads, size)
    plan = tctx.prompt_plan([rows], heads, kv, [300], causal=False)
    for at in (0, 31, 64, 130, 299):
        k = torch.zeros(300, kv, 64, dtype=TORCH[dtype], device="cuda")
        k[..., 3] = 64.0
        k[at, :, 3] = 72.0
        out = torch.zeros_like(q)
        tctx.prompt_attention_async(plan, q, k, v, out, None, scale, **opts)
        same(out, v[at].repeat_interleave(2, 0).expand(rows, heads, 64), size, dtype, at)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", ["plain", "bias", "both"])
def test_small_scores_beside_large_ones(tctx, dtype, kind):
    """Rows with scores of some thousands give the same bits whatever the other rows' are."""
    heads, kv, rows, keys = 4, 2, 70, 300
    v, outs = rand(2, keys, kv, 64, dtype=dtype), []
    opts = options(kind, heads, 1e9) if kind == "both" else options(kind, heads, 2.0 ** 53)
    for size in (1.0, 1e5, 4e6):
        q, k = loud(size, 1.0, rows, heads, dtype), torch.zeros(keys, kv, 64, dtype=TORCH[dtype], device="cuda")
        k[..., 3] = 64.0
        quiet(q, k, 5)
        outs.append(torch.zeros_like(q))
        # fp16 holds a query of 6e4: at a scale of 1e3 the largest is 4e9.
        tctx.prompt_attention_async(tctx.prompt_plan([rows], heads, kv, [keys], causal=False), q, k, v, outs[-1], None, 1e3,
                                    **opts)
        assert torch.isfinite(outs[-1].float()).all()
    for o in outs[1:]:
        assert torch.equal(bits(o[::3]), bits(outs[0][::3]))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new", [1, 60])
def test_over_the_cache(tctx, dtype, kind, new):
    """Few rows and many, in one part and in several."""
    heads, kv = 4, 2
    for length in (40, 300, 9000):
        for size in SIZES[2:]:
            f, scale, at = Filled(tctx, 1, 400, 32, kv, 64, dtype, 5), max(1.0, size / 1e6), length // 3
            (s,) = f.new()

            def make(seed, *shape):
                x = rand(seed, *shape, dtype=dtype)
                if seed == 7:  # keys
                    x.zero_()
                    x[..., 3] = 64.0
                    x[:, at, :, 3] = 72.0
                return x

            f.append([s], [length], make)
            new_here = min(new, length - at - 1)
            q = loud(size, scale, new_here, heads, dtype).abs()
            out = torch.full_like(q, 7.0)
            f.cache.attention_async(f.cache.plan([s], [new_here], heads=heads), q, out, 0, None, scale,
                                    **options(kind, heads, size))
            same(out, f.held[s][1][0, at].repeat_interleave(2, 0).expand(new_here, heads, 64), size, dtype, (length, size))
            f.cache.close()
