"""Attention over packed sequences (cvs_prompt_attention_async) against 64 bits.

Bounds: attention_oracle.py, derived from the number formats alone.
"""
import numpy as np
import pytest
import torch

from attention_oracle import TORCH, assert_within, attention, f64

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def rand(seed, *shape, dtype, spread=1.0, device="cuda"):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread).to(TORCH[dtype]).to(device)


def limits_of(ql, kl, causal):
    return [max(0, min(kl, i + 1 + kl - ql)) if causal else kl for i in range(ql)]


def check(ctx, q, k, v, q_lengths, k_lengths, dtype, causal, scale=None, out=None):
    heads, kv = q.shape[1], k.shape[1]
    out = torch.full_like(q, 7.0) if out is None else out
    lse = torch.full((heads, q.shape[0]), 7.0, device="cuda")
    plan = ctx.prompt_plan(q_lengths, heads, kv, k_lengths, causal)
    ctx.prompt_attention_async(plan, q, k, v, out, lse, 0.0 if scale is None else scale)
    got, got_lse = f64(out), f64(lse)
    plain = torch.full_like(q, 9.0)
    ctx.prompt_attention_async(plan, q, k, v, plain, None, 0.0 if scale is None else scale)
    assert torch.equal(plain.view(torch.int16), out.contiguous().view(torch.int16)), "without lse"
    a = b = 0
    for ql, kl in zip(q_lengths, k_lengths or q_lengths):
        want, tol, l, l_tol = attention(f64(q[a:a + ql]), f64(k[b:b + kl]), f64(v[b:b + kl]),
                                        limits_of(ql, kl, causal), dtype, scale)
        assert_within(got[a:a + ql], want, tol, f"sequence {ql}/{kl}")
        assert_within(got_lse[:, a:a + ql], l, l_tol, f"lse of {ql}/{kl}")
        a, b = a + ql, b + kl
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 128), (5, 1, 80), (3, 3, 96), (2, 1, 8), (6, 2, 40),
                                          (10, 2, 72), (2, 2, 120)])
def test_ragged(tctx, dtype, causal, heads, kv, dim):
    lengths = [0, 1, 2, 31, 32, 33, 0, 63, 64, 65, 130, 7]
    t = sum(lengths)
    q, k, v = (rand(dim + i, t, h, dim, dtype=dtype) for i, h in enumerate((heads, kv, kv)))
    check(tctx, q, k, v, lengths, None, dtype, causal)


@pytest.mark.parametrize("dim", list(range(8, 129, 8)))
def test_every_head_size(tctx, dim):
    lengths, dtype = [70, 129, 1], "fp16" if dim % 16 else "bf16"
    q, k, v = (rand(dim + i, 200, h, dim, dtype=dtype) for i, h in enumerate((6, 2, 2)))
    check(tctx, q, k, v, lengths, None, dtype, True)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_key_lengths_of_their_own(tctx, dtype, causal):
    """More keys than queries (a chunk behind earlier ones), fewer (rows that see nothing), none, and keys alone."""
    ql, kl = [5, 70, 3, 9, 0, 1, 40, 64], [200, 30, 0, 9, 17, 1, 41, 1]
    q = rand(1, sum(ql), 8, 64, dtype=dtype)
    k, v = rand(2, sum(kl), 2, 64, dtype=dtype), rand(3, sum(kl), 2, 64, dtype=dtype)
    out = check(tctx, q, k, v, ql, kl, dtype, causal)
    assert not out[75:78].any(), "queries of a sequence without keys"
    if causal:
        assert not out[5:45].any(), "queries before the first key"


@pytest.mark.parametrize("lengths", [[1], [300], [1000, 1], [0], [0, 0], []])
def test_lengths(tctx, lengths):
    t = sum(lengths)
    q, k, v = (rand(9 + i, t, h, 128, dtype="bf16") for i, h in enumerate((4, 2, 2)))
    check(tctx, q, k, v, lengths, None, "bf16", True)


@pytest.mark.parametrize("dim", [64, 80, 128])
def test_strides(tctx, dim):
    """Views of one projection, head-major arrays, rows with a gap, keys shared by all heads, an output in a wider array."""
    lengths, heads, kv, dtype = [50, 3, 90], 6, 2, "fp16"
    t = sum(lengths)
    qkv = rand(4, t, heads + 2 * kv, dim, dtype=dtype)
    check(tctx, qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], lengths, None, dtype, True)
    q = rand(5, heads, t, dim, dtype=dtype).transpose(0, 1)
    k = rand(6, kv, t, dim, dtype=dtype).transpose(0, 1)
    v = rand(7, t, kv, dim + 24, dtype=dtype)[..., 8:8 + dim]
    wide = torch.full((t, heads, dim + 8), 5.0, dtype=TORCH[dtype], device="cuda")
    check(tctx, q, k, v, lengths, None, dtype, True, out=wide[..., :dim])
    assert (wide[..., dim:] == 5).all(), "past the output's rows"
    one = rand(8, t, 1, dim, dtype=dtype).expand(t, kv, dim)
    check(tctx, q, one, one, lengths, None, dtype, False)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("spread", [1e-3, 4.0, 30.0])
def test_scores_of_any_size(tctx, dtype, spread):
    """Nearly equal weights, one weight that takes all, scores in the thousands."""
    lengths = [90, 130]
    q = rand(1, 220, 4, 64, dtype=dtype, spread=spread)
    k = rand(2, 220, 2, 64, dtype=dtype, spread=spread)
    v = rand(3, 220, 2, 64, dtype=dtype)
    check(tctx, q, k, v, lengths, None, dtype, True)
    check(tctx, q, k, v, lengths, None, dtype, False, scale=0.5)


def test_growing_and_falling_maxima(tctx):
    """Each later key outweighs all before it, then the reverse: every tile rescales, or none."""
    n, dtype = 400, "bf16"
    q = torch.ones(n, 2, 64, dtype=TORCH[dtype], device="cuda")
    ramp = torch.arange(n, device="cuda", dtype=torch.float32)[:, None, None] / 16
    v = rand(3, n, 2, 64, dtype=dtype)
    for r in (ramp, -ramp):
        k = r.expand(n, 2, 64).to(TORCH[dtype]).contiguous()
        check(tctx, q, k, v, [n], None, dtype, True)
        check(tctx, q, k, v, [n], None, dtype, False)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), "lowest"])
def test_values_in_keys_not_seen(tctx, dtype, value):
    """What stands in keys that a row does not see has no part in its result: the same bits as with zeros there."""
    x = torch.finfo(TORCH[dtype]).min if value == "lowest" else value
    lengths, heads, kv, dim = [70, 40, 5], 4, 2, 64
    t = sum(lengths)
    q, k, v = (rand(20 + i, t, h, dim, dtype=dtype) for i, h in enumerate((heads, kv, kv)))
    plan = tctx.prompt_plan(lengths, heads, kv)
    out = torch.zeros_like(q)
    for at in (0, 1, 33, 69, 70, 100, 109, 112):  # the key that holds it, and every later row of its sequence sees it
        seq0 = 0 if at < 70 else 70 if at < 110 else 110
        end = 70 if at < 70 else 110 if at < 110 else 115
        clean = []
        for fill in (0.0, x):
            kk, vv = k.clone(), v.clone()
            kk[at], vv[at] = fill, fill
            vv[at, :, 5:] = v[at, :, 5:]
            tctx.prompt_attention_async(plan, q, kk, vv, out)
            clean.append(torch.cat([out[:at], out[end:]]).clone())
        assert torch.equal(clean[0].view(torch.int16), clean[1].view(torch.int16)), (at, value)
        assert at == seq0 or torch.isfinite(clean[1].float()).all()
    # Seen, they count: an infinite value of positive weight is the result's sign of infinity, a NaN a NaN.
    if value != "lowest":
        vv = v.clone()
        vv[33, :, 3] = x
        tctx.prompt_attention_async(plan, q, k, vv, out)
        seen = out[33:70, :, 3].float()
        assert torch.isnan(seen).all() if x != x else (seen == x).all()
        rest = torch.cat([out[:33].flatten(), out[70:].flatten(), out[33:70, :, 4:].flatten()])
        assert torch.isfinite(rest.float()).all()


def test_rows_outside_the_sequences(tctx):
    """Rows of the arrays that no sequence of the plan has are neither read nor written: NaN around the tokens."""
    q, k, v = (rand(30 + i, 64, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    for x in (q, k, v):
        x[:16], x[48:] = float("nan"), float("nan")
    big = torch.full_like(q, 3.0)
    check(tctx, q[16:48], k[16:48], v[16:48], [20, 12], None, "fp16", False, out=big[16:48])
    assert (big[:16] == 3).all() and (big[48:] == 3).all()


def test_strides_that_are_not_used(tctx):
    """A single token or head may have any stride."""
    q, k, v = (rand(70 + i, 40, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    one = torch.as_strided(q, (1, 4, 64), ((1 << 40) + 3, 64, 1))
    check(tctx, one, k, v, [1], [40], "fp16", True, out=torch.zeros(1, 4, 64, dtype=torch.float16, device="cuda"))
    head = torch.as_strided(k, (40, 1, 64), (128, 7, 1))
    check(tctx, q, head, head, [40], None, "fp16", True)


def test_same_bits_again(tctx):
    q, k, v = (rand(40 + i, 700, h, 128, dtype="bf16") for i, h in enumerate((8, 2, 2)))
    plan = tctx.prompt_plan([300, 400], 8, 2)
    outs = [torch.zeros_like(q) for _ in range(3)]
    for o in outs:
        tctx.prompt_attention_async(plan, q, k, v, o)
    assert all(torch.equal(outs[0].view(torch.int16), o.view(torch.int16)) for o in outs)


def test_on_a_stream_of_the_callers(cvs):
    """Inputs made on the stream just before, outputs used on it just after, nothing waited for in between."""
    s = torch.cuda.Stream()
    with torch.cuda.stream(s), cvs.Context(0, stream=s.cuda_stream) as c:
        plan = c.prompt_plan([600], 4, 2)
        q, k, v = (rand(50 + i, 600, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(4):
            big = big @ big * 1e-3
        q2 = q + (big[0, 0] * 0).to(q.dtype)
        out = torch.empty_like(q)
        c.prompt_attention_async(plan, q2, k, v, out)
        doubled = out * 2
        want, tol, _, _ = attention(f64(q2), f64(k), f64(v), limits_of(600, 600, True), "fp16")
        assert_within(f64(doubled) / 2, want, tol, "on the caller's stream")


def test_context_of_its_own_stream_and_device_arrays(cvs, ctx):
    """The binding's own device arrays on the context's own stream; bfloat16 as uint16."""
    rng = np.random.default_rng(3)
    q, k, v = (rng.standard_normal((77, h, 64)).astype(np.float16) for h in (4, 2, 2))
    dev = [cvs.DeviceArray.from_host(ctx, x) for x in (q, k, v)]
    out, lse = cvs.DeviceArray(ctx, q.shape, np.float16), cvs.DeviceArray(ctx, (4, 77), np.float32)
    plan = ctx.prompt_plan([77], 4, 2)
    ctx.prompt_attention_async(plan, *dev, out, lse)
    ctx.synchronize()
    want, tol, l, l_tol = attention(*(x.astype(np.float64) for x in (q, k, v)), limits_of(77, 77, True), "fp16")
    assert_within(out.to_host().astype(np.float64), want, tol, "device arrays")
    assert_within(lse.to_host().astype(np.float64), l, l_tol, "lse")
    bits = [torch.from_numpy(x.astype(np.float32)).to(torch.bfloat16) for x in (q, k, v)]
    dev = [cvs.DeviceArray.from_host(ctx, x.view(torch.int16).numpy().view(np.uint16)) for x in bits]
    out = cvs.DeviceArray(ctx, q.shape, np.uint16)
    ctx.prompt_attention_async(plan, *dev, out)
    ctx.synchronize()
    got = torch.from_numpy(out.to_host().view(np.int16)).view(torch.bfloat16).double().numpy()
    want, tol, _, _ = attention(*(f64(x) for x in bits), limits_of(77, 77, True), "bf16")
    assert_within(got, want, tol, "bfloat16 device arrays")


def test_plans_made_and_dropped(tctx):
    """A plan dropped while its call may still run, and the next ones in its memory: nothing waits, nothing mixes."""
    q, k, v = (rand(80 + i, 900, h, 64, dtype="fp16") for i, h in enumerate((8, 2, 2)))
    batches = [[900], [450, 450], [1] * 900, [300, 0, 600], [899, 1]]
    outs = []
    for lengths in batches * 4:
        outs.append(torch.zeros_like(q))
        tctx.prompt_attention_async(tctx.prompt_plan(lengths, 8, 2), q, k, v, outs[-1])
    for lengths, out in zip(batches, outs[-len(batches):]):
        kept = tctx.prompt_plan(lengths, 8, 2)
        again = torch.zeros_like(q)
        tctx.prompt_attention_async(kept, q, k, v, again)
        torch.cuda.synchronize()
        assert torch.equal(out.view(torch.int16), again.view(torch.int16)), lengths
    for i, out in enumerate(outs):
        assert torch.equal(out.view(torch.int16), outs[i % len(batches)].view(torch.int16))


def test_refusals(cvs, tctx):
    t = 16
    q, k, v = (rand(60 + i, t, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    out = torch.full_like(q, 2.0)
    plan = tctx.prompt_plan([t], 4, 2)

    def refused(match, *args, plan=plan, **kw):
        with pytest.raises(ValueError, match=match):
            tctx.prompt_attention_async(plan, *args, **kw)
        torch.cuda.synchronize()
        assert (out == 2).all(), "nothing is written by a refused call"

    refused("plan's 16 tokens", q[:15], k, v, out)
    refused("plan's 16 tokens", q, k[:15], v[:15], out)
    refused("head counts", q[:, :2], k, v, out[:, :2])
    refused("head counts", q, q, v, out)
    refused("one head_dim", q, k[..., :32], v, out)
    refused("one type", q, k.bfloat16(), v, out)
    refused("attention takes", q.float(), k, v, out)
    refused("multiple of 8", q[..., :20], k[..., :20], v[..., :20], out[..., :20])
    big = rand(1, t, 4, 136, dtype="fp16")
    refused("multiple of 8 from 8 to 128", big, big[:, :2], big[:, :2], big)
    refused("16-byte aligned", big[..., 1:65], k, v, out)
    odd = rand(1, t, 4, 68, dtype="fp16")
    refused("multiples of 8", odd[..., :64], k, v, out)
    refused("last axis", rand(1, t, 64, 4, dtype="fp16").transpose(1, 2), k, v, out)
    refused("scale", q, k, v, out, scale=-1.0)
    refused("scale", q, k, v, out, scale=float("nan"))
    refused("scale", q, k, v, out, scale=float("inf"))
    refused("lse", q, k, v, out, lse=torch.zeros(4, t + 1, device="cuda"))
    refused("context's device", q.cpu(), k, v, out)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        tctx.prompt_plan([4], 5, 2)
    with pytest.raises(ValueError, match="negative length"):
        tctx.prompt_plan([4, -1], 4, 2)
    with pytest.raises(ValueError, match="values are needed"):
        tctx.prompt_plan([4, 1], 4, 2, k_lengths=[4])
    with pytest.raises(ValueError, match="31 bits"):
        tctx.prompt_plan([1 << 31], 4, 2)
    other = cvs.Context(0)
    with pytest.raises(ValueError, match="another context"):
        other.prompt_attention_async(plan, q, k, v, out)
    other.close()


def test_plans_end_with_their_context(cvs):
    with cvs.Context(0) as c:
        plan = c.prompt_plan([4], 4, 2)
        lib = cvs.load()
        assert lib.cvs_context_destroy(c.handle) == cvs.CVS_ERR_INVALID_ARGUMENT
        assert b"plan(s)" in lib.cvs_last_error()
    assert plan.handle is None
    plan.close()


def test_lengths_beyond_any_sum(cvs, tctx):
    top = 2**63 - 1
    for q, k, heads in (([1, top], None, 2), ([1, 1], [1, top], 2), ([1, 1], [top, top], 1), ([2**62], None, 4)):
        with pytest.raises(ValueError, match="31 bits"):
            tctx.prompt_plan(q, heads, 1, k)


def test_rows_of_an_output_that_overlap(tctx):
    plan = tctx.prompt_plan([5, 4], 2, 1)
    q, k, v = (rand(i, 9, h, 16, dtype="fp16") for i, h in enumerate((2, 1, 1)))
    room = torch.zeros(9 * 64, dtype=torch.float16, device="cuda")
    for strides in ((0, 16), (32, 0), (16, 16), (8, 144), (32, 8), (16, 136)):
        with pytest.raises(ValueError, match="must not overlap"):
            tctx.prompt_attention_async(plan, q, k, v, room.as_strided((9, 2, 16), (*strides, 1)))
    want = torch.empty_like(q)
    tctx.prompt_attention_async(plan, q, k, v, want)
    for strides in ((32, 16), (48, 24), (16, 144), (64, 16), (24, 216)):  # token by token, head by head, with gaps
        out = room.zero_().as_strided((9, 2, 16), (*strides, 1))
        tctx.prompt_attention_async(plan, q, k, v, out)
        assert torch.equal(out, want), strides
