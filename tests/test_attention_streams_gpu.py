"""Attention and the cache on torch tensors whose stream is not the context's: in order with torch's current stream all
the same, and tensors that require grad refused."""
import ctypes

import pytest
import torch

from test_kv_cache_gpu import bits, rand

pytestmark = pytest.mark.gpu


def slow(x):
    """x, made on torch's current stream behind some milliseconds of work."""
    big = torch.randn(4096, 4096, device="cuda")
    for _ in range(8):
        big = big @ big * 1e-3
    return x + (big[0, 0] * 0).to(x.dtype)


def calls(ctx, make):
    """A prompt, its tokens into a cache and out of it, and a step over it, on tensors that exist during a call alone."""
    q, k, v = (rand(i, 700, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    plan = ctx.prompt_plan([300, 400], 4, 2)
    cache = ctx.kv_cache(2, 30, 32, 2, 64, "fp16")
    seqs = cache.sequences(2)
    cache.extend(seqs, [300, 400])
    rows, step = cache.plan(seqs, [300, 400]), cache.plan(seqs, [2, 3], heads=4)
    outs = [torch.zeros(s, device="cuda", dtype=t) for s, t in (
        (q.shape, q.dtype), ((4, 700), torch.float32), (k.shape, k.dtype), (v.shape, v.dtype), ((5, 4, 64), q.dtype),
        ((4, 5), torch.float32))]
    torch.cuda.synchronize()
    ctx.prompt_attention_async(plan, make(q), make(k), make(v), outs[0], outs[1])
    junk = [torch.full_like(x, float("nan")) for x in (q, k, v)]
    cache.write_async(rows, make(k), make(v), layer=1)
    junk += [torch.full_like(x, float("nan")) for x in (k, v)]
    cache.read_async(rows, outs[2], outs[3], layer=1)
    cache.attention_async(step, make(q[:5]), outs[4], 1, outs[5])
    junk.append(torch.full_like(q[:5], float("nan")))
    results = [x * 1 for x in outs]  # on torch's stream, with nothing waited for
    torch.cuda.synchronize()
    cache.close()
    return results


@pytest.mark.parametrize("case", ["the context's own", "the default one", "another stream"])
def test_in_order_with_torch(cvs, case):
    with cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream) as c:
        want = calls(c, lambda x: x)
    side = torch.cuda.Stream()
    if case == "the context's own":
        ctx, current = cvs.Context(0), torch.cuda.current_stream()
    elif case == "the default one":
        ctx, current = cvs.Context(0, stream=torch.cuda.default_stream().cuda_stream), side
    else:
        ctx, current = cvs.Context(0, stream=torch.cuda.Stream().cuda_stream), side
    with ctx, torch.cuda.stream(current):
        got = calls(ctx, slow)
    for x, y in zip(got, want):
        assert torch.equal(x.view(torch.int16), y.view(torch.int16))


def test_the_streams_address(cvs):
    lib, p = cvs.load(), ctypes.c_void_p()
    s = torch.cuda.Stream()
    with cvs.Context(0, stream=s.cuda_stream) as c, cvs.Context(0) as own, cvs.Context(0, stream=0) as default:
        assert c.stream == s.cuda_stream and default.stream == 0 and own.stream not in (0, s.cuda_stream)
        assert lib.cvs_context_stream(c.handle, None) == cvs.CVS_ERR_INVALID_ARGUMENT
    assert lib.cvs_context_stream(None, ctypes.byref(p)) == cvs.CVS_ERR_INVALID_ARGUMENT
    with pytest.raises(ValueError, match="null"):
        own.prompt_attention_async(own.prompt_plan([1], 1, 1), *[rand(0, 1, 1, 64, dtype="fp16")] * 4)


def test_tensors_that_require_grad(cvs):
    with cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream) as c:
        q, k, v = (rand(i, 9, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
        plan, out, lse = c.prompt_plan([9], 4, 2), torch.empty_like(q), torch.empty(4, 9, device="cuda")
        cache = c.kv_cache(1, 4, 32, 2, 64, "fp16")
        s = cache.sequence()
        cache.extend([s], [9])
        rows = cache.plan([s], [9], heads=4)
        for x in (q, k, v, lse):
            x.requires_grad_()
            with pytest.raises(ValueError, match="requires grad"):
                c.prompt_attention_async(plan, q, k, v, out, lse)
            x.requires_grad_(False)
        k.requires_grad_()
        with pytest.raises(ValueError, match="requires grad"):
            cache.write_async(rows, k, v)
        cache.write_async(rows, k.detach(), v)
        with torch.no_grad():
            c.prompt_attention_async(plan, q, k, v, out, lse)
            cache.write_async(rows, k, v)
        q.requires_grad_()
        other = torch.empty_like(out)
        with pytest.raises(ValueError, match="requires grad"):
            cache.attention_async(rows, q, other)
        with torch.inference_mode():
            cache.attention_async(rows, q, other)
        assert torch.equal(bits(out), bits(other))
        cache.close()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs a second GPU")
def test_a_stream_of_another_device(cvs):
    with pytest.raises(ValueError, match="the stream is device 1's"):
        cvs.Context(0, stream=torch.cuda.Stream(device=1).cuda_stream)
