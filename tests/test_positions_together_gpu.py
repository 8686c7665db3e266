"""A layer's calls as a program makes them: passages and a question through norm, rotation and prompt attention, their
keys into the cache, then token by token over it - against the same tokens as one prompt, and against 64 bits."""
import numpy as np
import pytest
import torch

from attention_oracle import TORCH, assert_within, f64
from rotary_oracle import ready
from scored_oracle import scored
from test_kv_cache_gpu import bits, rand

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved,dims,cap,steep", [(False, 64, 20.0, 0.0), (True, 32, 0.0, 0.3), (False, 64, 5.0, 0.1)])
def test_prompt_then_tokens(cvs, dtype, interleaved, dims, cap, steep):
    passages, asked, steps, answers, heads, kv, dim = 150, 21, 5, 3, 8, 2, 64
    slopes = steep * 2.0 ** -torch.arange(heads, dtype=torch.float32, device="cuda") if steep else None
    prompt = passages + asked
    side = torch.cuda.Stream()
    with cvs.Context(0, stream=side.cuda_stream) as ctx, torch.cuda.stream(side):
        rotary = ctx.rotary(dims, 500000.0, interleaved, scaling="turns", factor=8.0, original_length=64, low=1, high=4)
        wq, wk = rand(8, dim, dtype=dtype), rand(9, dim, dtype=dtype)
        # Every answer's tokens behind the shared prompt, as projections of a layer.
        first = rand(1, prompt, heads + 2 * kv, dim, dtype=dtype)
        later = [rand(10 + i, answers, heads + 2 * kv, dim, dtype=dtype) for i in range(steps)]

        cache = ctx.kv_cache(1, 30, 32, kv, dim, dtype)
        root = cache.sequence()
        cache.extend([root], [prompt])
        rows = cache.plan([root], [prompt])
        q, k, v = first.split([heads, kv, kv], dim=1)
        q_out, k_out = torch.empty(prompt, heads, dim, dtype=TORCH[dtype], device="cuda"), torch.empty(
            prompt, kv, dim, dtype=TORCH[dtype], device="cuda")
        ctx.norm_rotate_async(rotary, torch.arange(prompt, device="cuda"), q, q_out, k, k_out, wq, wk)
        plan, out = ctx.prompt_plan([prompt], heads, kv, prefixes=[passages]), torch.empty_like(q_out)
        ctx.prompt_attention_async(plan, q_out, k_out, v, out, cap=cap, slopes=slopes)
        cache.append_async(rows, k, v, rotary=rotary, k_weight=wk)
        held = [torch.empty_like(k_out), torch.empty(prompt, kv, dim, dtype=TORCH[dtype], device="cuda")]
        cache.read_async(rows, *held)
        assert torch.equal(bits(held[0]), bits(k_out)) and torch.equal(bits(held[1]), bits(v))

        sequences, outs = cache.fork(root, answers), []
        for x in later:
            cache.extend(sequences, [1] * answers)
            step = cache.plan(sequences, [1] * answers, heads=heads)
            q1, k1, v1 = x.split([heads, kv, kv], dim=1)
            ready_q, o = torch.empty_like(x[:, :heads]), torch.empty(answers, heads, dim, dtype=TORCH[dtype], device="cuda")
            cache.append_async(step, k1, v1, rotary=rotary, k_weight=wk, q=q1, q_out=ready_q, q_weight=wq)
            cache.attention_async(step, ready_q, o, cap=cap, slopes=slopes)
            outs.append(o)

        # The formula in 64 bits, over keys as they are held: rounded once, on their way.
        freq = cvs.rotary_frequencies(dims, 500000.0, "turns", 8.0, 64, 1, 4)
        for a, s in enumerate(sequences):
            whole = torch.cat([first] + [x[a:a + 1] for x in later])
            n = len(whole)
            every = cache.plan([s], [n])
            kk, vv = (torch.empty(n, kv, dim, dtype=TORCH[dtype], device="cuda") for _ in "kv")
            cache.read_async(every, kk, vv)
            want, tol = ready(f64(whole[:, heads:heads + kv]), dtype, range(n), freq, interleaved, 1.0, f64(wk), 1e-6)
            assert_within(f64(kk), want, tol, "keys")
            qq = torch.empty(n, heads, dim, dtype=TORCH[dtype], device="cuda")
            ctx.norm_rotate_async(rotary, torch.arange(n, device="cuda"), whole[:, :heads], qq, q_weight=wq)
            limits = np.maximum(np.arange(n) + 1, passages)
            want, tol, _, _ = scored(f64(qq), f64(kk), f64(vv), limits, dtype, None, cap,
                                     None if slopes is None else f64(slopes), np.arange(n))
            got = torch.cat([out] + [o[a:a + 1] for o in outs])
            assert_within(f64(got), want, tol, f"answer {a}")
            again = torch.empty_like(qq)
            ctx.prompt_attention_async(ctx.prompt_plan([n], heads, kv, prefixes=[passages]), qq, kk, vv, again, cap=cap,
                                       slopes=slopes)
            assert_within(f64(again), want, tol, f"answer {a} as one prompt")
            del every
        del rows, step
        cache.close()
