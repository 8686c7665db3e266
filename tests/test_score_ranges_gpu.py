"""Capped scores at the ends of what a call takes: caps far above and below the scale's, products at every share of them.

Bounds: scored_oracle.py.  A row's keys are all the same, so that the logarithm of its sum is its score and log(keys).
"""
import numpy as np
import pytest
import torch

from attention_oracle import assert_within, f64
from scored_oracle import scored
from test_kv_cache_gpu import Filled, bits, rand

pytestmark = pytest.mark.gpu

# Of the cap: far below it, about the ends of a polynomial of each degree, about one half, beyond.
SHARES = [0.0, 1e-5, 3e-4, 0.9e-3, 1.1e-3, 0.01, 0.03, 0.033, 0.06, 0.1, 0.124, 0.126, 0.2, 0.3, 0.4, 0.44, 0.47, 0.49,
          0.499, 0.501, 0.52, 0.6, 1.0, 3.0, 20.0]
SHARES += [-s for s in SHARES[1:]]


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def check(ctx, scale, cap, steep):
    """SHARES of the cap, a key alone and many."""
    heads, kv, n = 4, 2, len(SHARES)
    v = rand(3, 400, kv, 64, dtype="bf16")
    slopes = None if steep is None else torch.full((heads,), steep, device="cuda")
    for keys in (1, 400):
        q, k = products(scale, cap, heads, kv, keys)
        out, lse = torch.full_like(q, 7.0), torch.full((heads, n), 7.0, device="cuda")
        plan = ctx.prompt_plan([n], heads, kv, [keys], causal=False)
        ctx.prompt_attention_async(plan, q, k, v[:keys], out, lse, scale, cap, slopes)
        want, tol, l, l_tol = scored(f64(q), f64(k), f64(v[:keys]), np.full(n, keys), "bf16", scale, cap,
                                     None if slopes is None else f64(slopes), np.arange(n) + keys - n)
        assert_within(f64(lse), l, l_tol, f"{keys} keys")
        assert_within(f64(out), want, tol, f"{keys} keys")
    return f64(out), f64(lse), f64(v)


def products(scale, cap, heads, kv, keys):
    """Queries and keys whose products, each of one channel, are SHARES of cap / scale."""
    whole = cap / scale
    one = 2.0 ** np.floor(np.log2(whole) / 2)  # about its root, so that both are in range
    q = torch.zeros(len(SHARES), heads, 64, dtype=torch.float64)
    q[:, :, 3] = torch.tensor([s * whole / one for s in SHARES], dtype=torch.float64)[:, None]
    k = torch.zeros(keys, kv, 64, dtype=torch.float64)
    k[:, :, 3] = one
    return (x.to(torch.bfloat16).cuda() for x in (q, k))


@pytest.mark.parametrize("scale,cap", [(0.125, 1e4), (0.125, 1e5), (0.125, 2e6), (0.125, 1e7), (0.0884, 1e7),
                                       (1e-6, 5.0), (1e-8, 50.0), (1e-18, 1.0), (1e-25, 1e-9), (1.0, 1.0), (1e4, 5.0),
                                       (1e-38, 1e-30)])
@pytest.mark.parametrize("steep", [None, 1e-3])
def test_caps_of_any_size_beside_the_scale(tctx, scale, cap, steep):
    """Every share of the cap keeps the bound, whatever the cap, in masked tiles and in others."""
    check(tctx, scale, cap, steep)


@pytest.mark.parametrize("scale,cap", [(0.125, 1e8), (0.125, 1e9), (0.125, 1e12), (0.125, 1e17), (1e12, 1e9),
                                       (1e18, 2e14), (1e21, 1e38), (2e38, 2e35)])
def test_scores_beyond_2_to_the_24(tctx, scale, cap):
    """Scores whose last place is more than 1: the same ones of a row still share evenly, whatever their size."""
    out, lse, v = check(tctx, scale, cap, None)
    even = v.mean(0).repeat(2, axis=0)
    # Weights of 1 are exact, as are their sums: the sums of values and the quotient, in 32 bits, and the output's rounding.
    room = 400 * 2.0 ** -24 * np.abs(v).mean(0).repeat(2, axis=0) + 2.0 ** -8 * np.abs(even) * 1.01
    assert (np.abs(out - even) <= room).all()
    check(tctx, scale, cap, 1e-3)


def test_larger_products_have_no_smaller_scores(tctx):
    """About one half of a cap far above the scale: of two keys the one with the larger product is taken."""
    scale, cap = 0.0884, 1e7
    whole = cap / scale
    shares = np.arange(0.495, 0.505, 0.0002)
    q = torch.zeros(1, 1, 64, dtype=torch.bfloat16, device="cuda")
    q[..., 3], q[..., 4] = 8192.0, 8.0
    k = torch.zeros(len(shares), 1, 64, dtype=torch.bfloat16, device="cuda")
    k[:, 0, 3] = 0.48 * whole / 8192.0  # the rest, in finer steps, is another channel's
    k[:, 0, 4] = torch.tensor((shares * whole - 8192.0 * k[0, 0, 3].item()) / 8.0).to(torch.bfloat16).cuda()
    assert (k[1:, 0, 4] > k[:-1, 0, 4]).all()
    plan = tctx.prompt_plan([1], 1, 1, [2])
    v = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    v[1] = 1.0
    for i in range(len(shares) - 1):
        out = torch.zeros_like(q)
        tctx.prompt_attention_async(plan, q, k[i:i + 2], v, out, None, scale, cap)
        assert (out == 1).all(), shares[i]


def test_coefficients_beyond_32_bits(tctx):
    """A scale of 5,000 caps and 1e18: products of 0 and small ones are not NaN, and share what the others leave."""
    scale, cap = 1e18, 2e14
    q = torch.zeros(2, 1, 64, dtype=torch.bfloat16, device="cuda")
    q[1, :, 3] = 2.0 ** -40
    k = torch.zeros(200, 1, 64, dtype=torch.bfloat16, device="cuda")
    k[100:, :, 3] = -(2.0 ** 40)
    v, out = rand(1, 200, 1, 64, dtype="bf16"), torch.zeros_like(q)
    lse = torch.full((1, 2), 7.0, device="cuda")
    tctx.prompt_attention_async(tctx.prompt_plan([2], 1, 1, [200], causal=False), q, k, v, out, lse, scale, cap)
    # Scores of 0, and of -cap for the second row's later keys, which leaves them no weight.
    for row, n in ((0, 200), (1, 100)):
        want, tol, l, l_tol = scored(f64(q[:1]), f64(k[:n]), f64(v[:n]), [n], "bf16", scale, 0.0, None, [n - 1])
        assert_within(f64(out[row:row + 1]), want, tol, f"row {row}")
        assert_within(f64(lse[:, row:row + 1]), l, l_tol, f"row {row}")


def test_caps_beyond_32_bits_are_refused(tctx):
    """Twice the cap in log2 units has to be a number of 32 bits."""
    q, k, v = (rand(i, 16, h, 64, dtype="bf16") for i, h in enumerate((4, 2, 2)))
    out, plan = torch.full_like(q, 2.0), tctx.prompt_plan([16], 4, 2)
    for cap in (1.001e38, 1.2e38, 3e38):
        with pytest.raises(ValueError, match="cap"):
            tctx.prompt_attention_async(plan, q, k, v, out, cap=cap, scale=1e25)
    torch.cuda.synchronize()
    assert (out == 2).all()


STEEP = [1e20, 1e28, 1e33, 1e37, 2.4e38, 3.4028234e38]


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_the_steepest_slopes(tctx, dtype, cap):
    """Of any finite slope a row has its nearest key alone, of a negative one its farthest."""
    slopes = torch.tensor(STEEP + [-s for s in STEEP], device="cuda")
    heads, kv = len(slopes), 1
    # Rows before the first key, tiles that end at a row's place, a row alone behind whole tiles, many rows.
    for ql, kl in ((300, 300), (1, 64), (1, 128), (64, 192), (70, 40), (1, 777), (130, 700)):
        q, k, v = (rand(i, n, h, 64, dtype=dtype) for i, n, h in ((1, ql, heads), (2, kl, kv), (3, kl, kv)))
        out, lse = torch.zeros_like(q), torch.zeros(heads, ql, device="cuda")
        tctx.prompt_attention_async(tctx.prompt_plan([ql], heads, kv, [kl], prefixes=[min(kl, 20)]), q, k, v, out, lse,
                                    cap=cap, slopes=slopes)
        place = torch.arange(ql, device="cuda") + kl - ql
        seen = torch.maximum(place + 1, torch.tensor(min(kl, 20), device="cuda")).clamp(max=kl)
        near = place.clamp(min=0)
        far = torch.where(place >= seen - 1 - place, 0, seen - 1)
        alone = place * 2 != seen - 1  # not as far from the first key as from the last
        for h in range(heads):
            at = near if slopes[h] > 0 else far
            rows = alone if slopes[h] < 0 else torch.ones_like(alone)
            assert torch.equal(bits(out[:, h][rows]), bits(v[at, 0][rows])), (ql, kl, slopes[h].item())
        want = -slopes.double().clamp(-1e28, 1e28)[:, None] * torch.stack(
            [(place - (near if s > 0 else far)).abs().double() for s in slopes])
        assert ((lse.double() - want).abs() <= 2.0 ** -21 * want.abs() + 30.0).all(), (ql, kl)


@pytest.mark.parametrize("cap", [0.0, 20.0])
@pytest.mark.parametrize("new", [1, 3, 80])
def test_the_steepest_slopes_over_the_cache(tctx, cap, new):
    slopes = torch.tensor(STEEP + [-s for s in STEEP], device="cuda")
    f = Filled(tctx, 1, 400, 32, 1, 64, "fp16", 3)
    seqs = f.new(4)
    lengths = [64, 100, 777, 9000]
    f.append(seqs, lengths)
    here = [min(new, n) for n in lengths]
    q = rand(9, sum(here), len(slopes), 64, dtype="fp16")
    out, start = torch.zeros_like(q), 0
    f.cache.attention_async(f.cache.plan(seqs, here, heads=len(slopes)), q, out, cap=cap, slopes=slopes)
    for s, n, m in zip(seqs, here, lengths):
        v = f.held[s][1][0, :, 0]
        for h in range(len(slopes)):
            want = v[m - n:] if slopes[h] > 0 else v[:1].expand(n, 64)
            assert torch.equal(bits(out[start:start + n, h]), bits(want)), (m, slopes[h].item())
        start += n
    f.cache.close()


def test_scales_beyond_32_bits_are_refused(tctx):
    """log2(e) times the scale has to be a number of 32 bits, or products of 0 would be NaN."""
    q = torch.zeros(3, 1, 64, dtype=torch.bfloat16, device="cuda")
    q[1:, :, 3] = 2.0 ** -130
    k = q + 0.0
    v, out = rand(1, 3, 1, 64, dtype="bf16"), torch.full_like(q, 2.0)
    plan = tctx.prompt_plan([3], 1, 1)
    f = Filled(tctx, 1, 2, 32, 1, 64, "bf16")
    (s,) = f.new()
    f.append([s], [3])
    step = f.cache.plan([s], [3], heads=1)
    for scale in (2.01e38, 2.4e38, 3.4028234e38):
        for options in ({}, {"cap": 5.0}):
            with pytest.raises(ValueError, match="scale must be at most"):
                tctx.prompt_attention_async(plan, q, k, v, out, scale=scale, **options)
            with pytest.raises(ValueError, match="scale must be at most"):
                f.cache.attention_async(step, q, out, scale=scale, **options)
    torch.cuda.synchronize()
    assert (out == 2).all()
    tctx.prompt_attention_async(plan, q, k, v, out, scale=2e38)
    want = torch.cumsum(v.float(), 0) / torch.arange(1, 4, device="cuda")[:, None, None]
    assert (out.float() - want).abs().max() <= 2.0 ** -7 * v.float().abs().max()
    del step
    f.cache.close()
