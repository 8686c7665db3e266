"""Attention rows most of whose weight is on one key: the small weights of all the others still count.

A weight leaves the softmax of the kernels as fp16 or bf16. fp16 holds weights down to 2^-22 of the row's largest with all
their bits if that one stands at 2^8, and those below within 2^-33 of it: with n keys, values v and weights scaled to a
largest one of 1 whose sum is s, an output is off by at most n 2^-33 max |v| / s for it. The bound of attention_oracle.py
has 2^-25 there; all its other terms stand."""
import math

import numpy as np
import pytest
import torch

from attention_oracle import TORCH, assert_within, attention, f64

pytestmark = pytest.mark.gpu

KEYS = 100_000
DIM = 64


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def check(got, q, k, v, limits, dtype, what):
    group = q.shape[1] // k.shape[1]
    want, tol, _, _ = attention(q, k, v, limits, dtype, 1.0)
    if dtype == "fp16":
        for i, n in enumerate(limits):
            for h in range(q.shape[1]):
                x = k[:n, h // group] @ q[i, h]
                total = np.exp(x - x.max()).sum()
                tol[i, h] -= 1.25 * n * np.abs(v[:n, h // group]).max() / total * (2.0 ** -25 - 2.0 ** -33)
    assert (tol > 0).all()
    assert_within(got, want, tol, what)


def heavy(dtype, at, share, seed):
    """Keys whose first column is their score, one of them with `share` of the weight and a value of 0."""
    g = torch.Generator().manual_seed(seed)
    k, v = torch.zeros(KEYS, 1, DIM), torch.randn(KEYS, 1, DIM, generator=g) + 1.0
    k[:, 0, 0] = torch.randn(KEYS, generator=g) * math.log(2.0)
    rest = k[:, 0, 0].to(TORCH[dtype]).double().exp().sum().item()
    k[at, 0, 0] = math.log(rest * share / (1.0 - share))
    v[at] = 0.0
    return k.to(TORCH[dtype]).cuda(), v.to(TORCH[dtype]).cuda()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("share", [0.99, 0.998])
@pytest.mark.parametrize("at", [0, 5000, KEYS - 9])
def test_prompt(tctx, dtype, share, at):
    k, v = heavy(dtype, at, share, 1)
    q = torch.zeros(3, 2, DIM, dtype=TORCH[dtype], device="cuda")
    q[..., 0] = 1.0
    out = torch.empty_like(q)
    tctx.prompt_attention_async(tctx.prompt_plan([3], 2, 1, [KEYS]), q, k, v, out, scale=1.0)
    check(f64(out), f64(q), f64(k), f64(v), [KEYS - 2, KEYS - 1, KEYS], dtype, "prompt")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("group", [1, 40])
@pytest.mark.parametrize("at", [0, 5000, KEYS - 9])
def test_cache(tctx, dtype, group, at):
    """Up to 32 rows a key, and more; many kv heads, so that a row's keys are in few parts."""
    kv = 128
    k, v = heavy(dtype, at, 0.998, 2)
    cache = tctx.kv_cache(1, KEYS // 128 + 1, 128, kv, DIM, dtype)
    s = cache.sequence()
    cache.extend([s], [KEYS])
    cache.write_async(cache.plan([s], [KEYS]), k.expand(KEYS, kv, DIM), v.expand(KEYS, kv, DIM))
    q = torch.zeros(1, kv * group, DIM, dtype=TORCH[dtype], device="cuda")
    q[..., 0] = 1.0
    out = torch.empty_like(q)
    cache.attention_async(cache.plan([s], [1], heads=kv * group), q, out, scale=1.0)
    check(f64(out[:, :2]), f64(q[:, :2]), f64(k), f64(v), [KEYS], dtype, "cache")
    assert torch.equal(out.view(torch.int16), out[:, :1].expand_as(out).contiguous().view(torch.int16))
    cache.close()
