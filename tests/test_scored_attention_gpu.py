"""Attention with capped scores, a bias by distance and prefixes, over packed prompts and over a paged cache, against 64
bits.

Bounds: scored_oracle.py, derived from the number formats and the tanh's own error.
"""
import numpy as np
import pytest
import torch

from attention_oracle import TORCH, assert_within, f64
from scored_oracle import scored
from test_kv_cache_gpu import Filled, bits, rand

pytestmark = pytest.mark.gpu

KINDS = ["cap", "bias", "both"]


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def options(kind, heads, cap=20.0, steep=1.0):
    """Scores' options of a kind; slopes from steep to flat."""
    slopes = steep * 2.0 ** (-8.0 * torch.arange(heads, dtype=torch.float32) / max(heads, 2))
    return (cap if kind != "bias" else 0.0), (None if kind == "cap" else slopes.cuda())


def check(ctx, q, k, v, q_lengths, k_lengths, dtype, causal, cap, slopes, prefixes=None, scale=None, out=None):
    heads, kv = q.shape[1], k.shape[1]
    out = torch.full_like(q, 7.0) if out is None else out
    lse = torch.full((heads, q.shape[0]), 7.0, device="cuda")
    plan = ctx.prompt_plan(q_lengths, heads, kv, k_lengths, causal, prefixes)
    ctx.prompt_attention_async(plan, q, k, v, out, lse, 0.0 if scale is None else scale, cap, slopes)
    got, got_lse = f64(out), f64(lse)
    a = b = 0
    for i, (ql, kl) in enumerate(zip(q_lengths, k_lengths or q_lengths)):
        places = np.arange(ql) + kl - ql
        limits = np.full(ql, kl)
        if causal:
            limits = np.clip(np.maximum(places + 1, prefixes[i] if prefixes else 0), 0, kl)
        want, tol, l, l_tol = scored(f64(q[a:a + ql]), f64(k[b:b + kl]), f64(v[b:b + kl]), limits, dtype, scale, cap,
                                     None if slopes is None else f64(slopes), places)
        assert_within(got[a:a + ql], want, tol, f"sequence {ql}/{kl}")
        assert_within(got_lse[:, a:a + ql], l, l_tol, f"lse of {ql}/{kl}")
        a, b = a + ql, b + kl
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 128), (5, 1, 80), (3, 3, 96), (2, 1, 8), (10, 2, 72),
                                          (2, 2, 112)])
def test_ragged(tctx, dtype, kind, causal, heads, kv, dim):
    lengths = [0, 1, 2, 31, 32, 33, 0, 63, 64, 65, 130, 7, 300]
    t = sum(lengths)
    q, k, v = (rand(dim + i, t, h, dim, dtype=dtype, spread=2.0) for i, h in enumerate((heads, kv, kv)))
    check(tctx, q, k, v, lengths, None, dtype, causal, *options(kind, heads))


@pytest.mark.parametrize("dim", list(range(8, 129, 8)))
def test_every_head_size(tctx, dim):
    lengths, dtype = [70, 129, 1], "fp16" if dim % 16 else "bf16"
    q, k, v = (rand(dim + i, 200, h, dim, dtype=dtype) for i, h in enumerate((6, 2, 2)))
    for kind in KINDS:
        check(tctx, q, k, v, lengths, None, dtype, dim % 3 > 0, *options(kind, 6, cap=1.0))


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", ["none"] + KINDS)
def test_prefixes(tctx, dtype, kind):
    """Prefixes of nothing, a token, whole tiles and not, the whole sequence; keys before the queries, and too few."""
    ql = [0, 1, 70, 70, 129, 200, 90, 40, 5, 64, 30]
    kl = [3, 1, 70, 70, 129, 200, 300, 10, 0, 64, 200]
    prefixes = [2, 0, 1, 70, 64, 129, 250, 7, 0, 63, 200]
    q = rand(1, sum(ql), 8, 64, dtype=dtype)
    k, v = rand(2, sum(kl), 2, 64, dtype=dtype), rand(3, sum(kl), 2, 64, dtype=dtype)
    cap, slopes = (0.0, None) if kind == "none" else options(kind, 8, cap=2.0, steep=0.25)
    check(tctx, q, k, v, ql, kl, dtype, True, cap, slopes, prefixes)
    plain = check(tctx, q, k, v, ql, kl, dtype, True, cap, slopes, [0] * len(ql))
    same = check(tctx, q, k, v, ql, kl, dtype, True, cap, slopes)
    assert torch.equal(bits(plain), bits(same)), "a prefix of nothing"


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("steep", [0.01, 1.0, 50.0])
def test_key_lengths_of_their_own(tctx, dtype, causal, steep):
    """More keys than queries, fewer (rows before the first key, which see nothing or stand far from all), none."""
    ql, kl = [5, 70, 3, 9, 0, 1, 200, 64], [200, 30, 0, 9, 17, 1, 41, 1]
    q = rand(1, sum(ql), 8, 64, dtype=dtype)
    k, v = rand(2, sum(kl), 2, 64, dtype=dtype), rand(3, sum(kl), 2, 64, dtype=dtype)
    for kind in ("bias", "both"):
        out = check(tctx, q, k, v, ql, kl, dtype, causal, *options(kind, 8, steep=steep))
    assert not out[75:78].any(), "queries of a sequence without keys"


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("cap", [1e-3, 0.5, 5.0, 50.0, 1e4])
@pytest.mark.parametrize("spread", [1e-2, 1.0, 8.0])
def test_caps_of_any_size(tctx, dtype, cap, spread):
    """Scores far below the cap, about it, and far beyond."""
    lengths = [90, 130]
    q = rand(1, 220, 4, 64, dtype=dtype, spread=spread)
    k = rand(2, 220, 2, 64, dtype=dtype, spread=spread)
    v = rand(3, 220, 2, 64, dtype=dtype)
    check(tctx, q, k, v, lengths, None, dtype, True, cap, None)
    check(tctx, q, k, v, lengths, None, dtype, False, cap, None, scale=0.5)
    check(tctx, q, k, v, lengths, None, dtype, True, cap, torch.tensor([0.3, 0.0, 2.0, 1e-3], device="cuda"))


@pytest.mark.parametrize("cap", [1e-30, 1e-9, 1e6, 0.99e12])
@pytest.mark.parametrize("scale", [None, 1e-6, 1e4])
def test_caps_at_the_ends(tctx, cap, scale):
    """A cap that flattens every score, one that changes none."""
    q, k, v = (rand(i, 100, h, 64, dtype="bf16", spread=1.0 if scale is None or scale < 1 else 1e-2)
               for i, h in enumerate((4, 2, 2)))
    check(tctx, q, k, v, [100], None, "bf16", True, cap, None, scale=scale)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("causal", [True, False])
def test_slopes_of_any_kind(tctx, dtype, causal):
    """None, steep ones, ones that grow with the distance."""
    q, k, v = (rand(i, 700, h, 64, dtype=dtype) for i, h in enumerate((8, 2, 2)))
    slopes = torch.tensor([0.0, 1e-4, 0.05, 100.0, -0.05, -1.0, 3e4, -1e-3], device="cuda")
    check(tctx, q, k, v, [700], None, dtype, causal, 0.0, slopes)
    check(tctx, q, k, v, [699, 1], None, dtype, causal, 10.0, slopes)


def test_long_prompts(tctx):
    """Distances of thousands: the weight of what is near is not lost beside the first tile's, nor the reverse."""
    n = 5000
    for dtype, kind in (("bf16", "bias"), ("fp16", "both"), ("bf16", "cap")):
        q, k, v = (rand(i, n, h, 64, dtype=dtype) for i, h in enumerate((2, 1, 1)))
        cap, slopes = options(kind, 2, steep=0.5)
        check(tctx, q, k, v, [n], None, dtype, True, cap, slopes)
        check(tctx, q, k, v, [n], None, dtype, True, cap, slopes, prefixes=[3333])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan"), "lowest"])
def test_values_in_keys_not_seen(tctx, dtype, kind, value):
    """What stands in keys that a row does not see has no part in its result: the same bits as with zeros there."""
    x = torch.finfo(TORCH[dtype]).min if value == "lowest" else value
    lengths, heads, kv, dim = [70, 200, 5], 4, 2, 64
    t = sum(lengths)
    q, k, v = (rand(20 + i, t, h, dim, dtype=dtype) for i, h in enumerate((heads, kv, kv)))
    cap, slopes = options(kind, heads)
    plan, out = tctx.prompt_plan(lengths, heads, kv), torch.zeros_like(q)
    for at in (0, 1, 33, 69, 70, 100, 133, 134, 200, 269, 270, 274):
        end = 70 if at < 70 else 270 if at < 270 else 275
        clean = []
        for fill in (0.0, x):
            kk, vv = k.clone(), v.clone()
            kk[at], vv[at] = fill, fill
            vv[at, :, 5:] = v[at, :, 5:]
            tctx.prompt_attention_async(plan, q, kk, vv, out, cap=cap, slopes=slopes)
            clean.append(torch.cat([out[:at], out[end:]]).clone())
        assert torch.equal(bits(clean[0]), bits(clean[1])), (at, value)
        assert torch.isfinite(clean[1].float()).all()
    # Seen, they count.
    if value != "lowest":
        vv = v.clone()
        vv[103, :, 3] = x
        tctx.prompt_attention_async(plan, q, k, vv, out, cap=cap, slopes=None if slopes is None else slopes * 1e-2)
        seen = out[103:270, :, 3].float()
        assert torch.isnan(seen).all() if x != x else (seen == x).all()
        rest = torch.cat([out[:103].flatten(), out[270:].flatten(), out[103:270, :, 4:].flatten()])
        assert torch.isfinite(rest.float()).all()


@pytest.mark.parametrize("kind", ["cap", "both"])
def test_infinite_products_are_capped(tctx, kind):
    """An infinite channel makes a score of plus or minus the cap."""
    q, k, v = (rand(i, 80, h, 64, dtype="bf16") for i, h in enumerate((4, 2, 2)))
    k[11, :, 5], k[50, 1, 7] = float("inf"), float("-inf")
    q[..., 5] = q[..., 5].abs() + 0.1
    check(tctx, q, k, v, [80], None, "bf16", False, *options(kind, 4, cap=3.0))


def test_products_beyond_fp32s_squares(tctx):
    """Products whose squares are infinite are at the cap, whatever it is: they share, and those far below have nothing."""
    q = torch.full((3, 1, 64), 2.0 ** 33, dtype=torch.bfloat16, device="cuda")
    k = torch.zeros(5, 1, 64, dtype=torch.bfloat16, device="cuda")
    k[:, :, 0] = torch.tensor([1.0, 2.0 ** 40, 2.0 ** 41, -2.0 ** 41, 2.0 ** 41], device="cuda")[:, None]
    v, out = rand(1, 5, 1, 64, dtype="bf16"), torch.zeros_like(q)
    plan = tctx.prompt_plan([3], 1, 1, [5], causal=False)
    for cap, share in ((2.0 ** 55, [0, 1 / 3, 1 / 3, 0, 1 / 3]), (4.0, [1 / 3, 1 / 3, 1 / 3, 0, 0])):
        if cap == 4.0:
            k[4, :, 0] = -1.0
        tctx.prompt_attention_async(plan, q, k, v, out, cap=cap)
        # Beside them are weights of e^-8 at most (a cap of 4: every score is 4 or -4).
        want = sum(w * f64(v)[i, 0] for i, w in enumerate(share))
        assert np.abs(f64(out)[:, 0] - want).max() < 2.0 ** -7 * (1 + np.abs(f64(v)).max())


def test_rows_depend_on_themselves_alone(tctx):
    """Large scores of other rows in a wave change no bit of a row, however the others are softened."""
    q, k, v = (rand(i, 150, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    for kind in KINDS:
        cap, slopes = options(kind, 4, cap=4.0)
        plan, outs = tctx.prompt_plan([150], 4, 2), []
        for loud in (1.0, 60.0):
            q2 = q.clone()
            q2[::2] *= loud
            outs.append(torch.zeros_like(q))
            tctx.prompt_attention_async(plan, q2, k, v, outs[-1], cap=cap, slopes=slopes)
        assert torch.equal(bits(outs[0][1::2]), bits(outs[1][1::2])), kind


@pytest.mark.parametrize("dim", [64, 80, 128])
def test_strides(tctx, dim):
    lengths, heads, kv, dtype = [50, 3, 90], 6, 2, "fp16"
    t = sum(lengths)
    cap, slopes = options("both", heads)
    qkv = rand(4, t, heads + 2 * kv, dim, dtype=dtype)
    check(tctx, qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:], lengths, None, dtype, True, cap, slopes)
    q = rand(5, heads, t, dim, dtype=dtype).transpose(0, 1)
    k = rand(6, kv, t, dim, dtype=dtype).transpose(0, 1)
    v = rand(7, t, kv, dim + 24, dtype=dtype)[..., 8:8 + dim]
    wide = torch.full((t, heads, dim + 8), 5.0, dtype=TORCH[dtype], device="cuda")
    check(tctx, q, k, v, lengths, None, dtype, True, cap, slopes, out=wide[..., :dim])
    assert (wide[..., dim:] == 5).all(), "past the output's rows"


# ---- over the cache --------------------------------------------------------


def attend(f, seqs, tokens, heads, cap, slopes, layer=0, seed=50, spread=1.0, scale=None, q=None):
    """Attention of the newest tokens against 64 bits; returns the output."""
    plan, t = f.cache.plan(seqs, tokens, heads=heads), sum(tokens)
    q = rand(seed, t, heads, f.dim, dtype=f.dtype, spread=spread) if q is None else q
    out, lse = torch.full_like(q, 7.0), torch.full((heads, t), 7.0, device="cuda")
    f.cache.attention_async(plan, q, out, layer, lse, 0.0 if scale is None else scale, cap, slopes)
    got, got_lse, at = f64(out), f64(lse), 0
    for s, n in zip(seqs, tokens):
        k, v = (f64(x[layer]) for x in f.held[s])
        limits = [len(k) - n + i + 1 for i in range(n)]
        want, tol, l, l_tol = scored(f64(q[at:at + n]), k, v, limits, f.dtype, scale, cap,
                                     None if slopes is None else f64(slopes))
        assert_within(got[at:at + n], want, tol, f"sequence {s}")
        assert_within(got_lse[:, at:at + n], l, l_tol, f"lse of {s}")
        at += n
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 64, 32), (8, 2, 128, 64), (5, 1, 80, 32), (3, 3, 24, 128),
                                               (40, 2, 96, 32)])
@pytest.mark.parametrize("new", [1, 5])
def test_sequences_of_many_lengths(tctx, dtype, kind, heads, kv, dim, page, new):
    lengths = [new, new + 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 17]
    f = Filled(tctx, 2, 80, page, kv, dim, dtype, 11)
    seqs = f.new(len(lengths))
    f.append(seqs, lengths)
    attend(f, seqs, [new] * (len(seqs) - 1) + [0], heads, *options(kind, heads), layer=1, spread=2.0)
    f.cache.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("new,heads", [(1, 8), (3, 2), (40, 4)])
def test_shared_prefixes(tctx, dtype, kind, new, heads):
    """Runs that many rows share, their own tails behind them, a fork of a fork, one that shares nothing."""
    f = Filled(tctx, 1, 700, 32, 2, 64, dtype, 3)
    (root,) = f.new()
    f.append([root], [1500])
    kids = f.fork(root, 9)
    f.append(kids, [40 + 13 * i for i in range(9)])
    deep = f.fork(kids[4], 3)
    f.append(deep, [new] * 3)
    lone = f.new(1)
    f.append(lone, [777])
    attend(f, kids + deep + lone, [new] * 13, heads, *options(kind, heads, steep=0.05))
    f.cache.close()


@pytest.mark.parametrize("kind,dtype,heads", [("cap", "bf16", 8), ("bias", "fp16", 8), ("both", "bf16", 64),
                                              ("bias", "bf16", 64)])
def test_long_rows_in_parts(tctx, kind, dtype, heads):
    """More pages than a wave holds ids of, in parts that are joined; steep slopes leave most parts without weight."""
    f = Filled(tctx, 1, 400, 32, 2, 64, dtype, 5)
    (root,) = f.new()
    f.append([root], [9003])
    kids = f.fork(root, 3)
    f.append(kids, [1, 30, 70])
    for steep in (0.01, 2.0):
        attend(f, kids, [1, 2, 3], heads, *options(kind, heads, steep=steep))
    attend(f, [root], [1], heads, *options(kind, heads, steep=0.1))
    attend(f, [root], [200], heads, *options(kind, heads, steep=0.1))
    f.cache.close()


def test_one_long_page(tctx):
    f = Filled(tctx, 1, 3, 4096, 1, 32, "fp16", 5)
    (s,) = f.new()
    f.append([s], [7000])
    for kind in KINDS:
        attend(f, [s], [1], 4, *options(kind, 4, steep=0.02))
        attend(f, [s], [50], 4, *options(kind, 4, steep=0.02))
    f.cache.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", KINDS)
def test_what_pages_held_before(tctx, dtype, kind):
    """Memory past a sequence's end, where infinities and NaNs were, does not reach it."""
    f = Filled(tctx, 1, 12, 64, 2, 64, dtype, 7)
    (s,) = f.new()
    for x in (float("nan"), float("inf"), -float("inf")):
        f.append([s], [600], lambda seed, *shape: torch.full(shape, x, dtype=TORCH[dtype], device="cuda"))
        f.free([s])
        (s,) = f.new()
    f.append([s], [70])
    more = f.new(4)
    f.append(more, [1, 33, 64, 95])
    attend(f, [s] + more, [3, 1, 1, 2, 40], 8, *options(kind, 8))
    f.cache.close()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("length", [3, 64, 1500, 9000])
def test_a_key_that_only_the_last_sees(tctx, kind, value, length):
    dtype, outs = "fp16", []
    cap, slopes = options(kind, 4, steep=0.01)
    for x in (0.0, value):
        f = Filled(tctx, 1, 300, 32, 2, 64, dtype, 13)
        (s,) = f.new()
        f.append([s], [length])
        k, v = (rand(60 + i, 1, 1, 2, 64, dtype=dtype) for i in (0, 1))
        v[..., 9] = x
        f.cache.extend([s], [1])
        plan = f.cache.plan([s], [1])
        f.cache.write_async(plan, k, v)
        q, out = rand(70, 2, 4, 64, dtype=dtype), torch.zeros(2, 4, 64, dtype=torch.float16, device="cuda")
        f.cache.attention_async(f.cache.plan([s], [2], heads=4), q, out, cap=cap, slopes=slopes)
        outs.append(out)
        del plan
        f.cache.close()
    assert torch.equal(bits(outs[0][0]), bits(outs[1][0]))
    last = outs[1][1, :, 9].float()
    assert torch.isnan(last).all() if value != value else (last == value).all()
    keep = [i for i in range(64) if i != 9]
    assert torch.equal(bits(outs[0][1][:, keep]), bits(outs[1][1][:, keep]))


def test_a_prompt_and_its_cache_agree(tctx):
    """The same tokens as a prompt and as a sequence's newest ones."""
    n, heads, dtype = 300, 8, "bf16"
    f = Filled(tctx, 1, 12, 32, 2, 64, dtype, 9)
    (s,) = f.new()
    f.append([s], [n])
    k, v = (x[0] for x in f.held[s])
    q = rand(1, n, heads, 64, dtype=dtype)
    for kind in KINDS:
        cap, slopes = options(kind, heads)
        check(tctx, q, k, v, [n], None, dtype, True, cap, slopes)
        attend(f, [s], [n], heads, cap, slopes, q=q)
    f.cache.close()


# ---- calls -----------------------------------------------------------------


def test_same_bits_again_and_without_options(tctx):
    q, k, v = (rand(40 + i, 700, h, 128, dtype="bf16") for i, h in enumerate((8, 2, 2)))
    plan = tctx.prompt_plan([300, 400], 8, 2)
    for kind in KINDS:
        cap, slopes = options(kind, 8)
        outs = [torch.zeros_like(q) for _ in range(3)]
        for o in outs:
            tctx.prompt_attention_async(plan, q, k, v, o, cap=cap, slopes=slopes)
        assert all(torch.equal(bits(outs[0]), bits(o)) for o in outs)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    tctx.prompt_attention_async(plan, q, k, v, a)
    tctx.prompt_attention_async(plan, q, k, v, b, cap=0.0, slopes=None)
    assert torch.equal(bits(a), bits(b))


def test_refusals(tctx, cvs):
    q, k, v = (rand(60 + i, 16, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    out, plan = torch.full_like(q, 2.0), tctx.prompt_plan([16], 4, 2)
    f = Filled(tctx, 1, 3, 32, 2, 64, "fp16")
    (s,) = f.new()
    f.append([s], [16])
    rows = f.cache.plan([s], [16], heads=4)
    slopes = torch.ones(4, device="cuda")

    def refused(match, **kw):
        with pytest.raises(ValueError, match=match):
            tctx.prompt_attention_async(plan, q, k, v, out, **kw)
        with pytest.raises(ValueError, match=match):
            f.cache.attention_async(rows, q, out, **kw)
        torch.cuda.synchronize()
        assert (out == 2).all(), "nothing is written by a refused call"

    for cap in (-1.0, float("nan"), float("inf"), 1e-31, 3e38, 1.1e18 / 8):
        refused("cap", cap=cap)
    refused("cap", cap=1.1e12, scale=1e-6)
    refused("slopes must be 4", slopes=slopes[:2])
    refused("slopes must be 4", slopes=slopes.double())
    refused("slopes must be 4", slopes=slopes[:, None])
    refused("contiguous", slopes=torch.ones(8, device="cuda")[::2])
    refused("device", slopes=slopes.cpu())
    refused("requires grad", slopes=slopes.clone().requires_grad_())
    refused("scale", slopes=slopes, scale=-1.0)
    with pytest.raises(ValueError, match="prefixes belong to a causal plan"):
        tctx.prompt_plan([16], 4, 2, causal=False, prefixes=[3])
    for prefixes in ([17], [-1]):
        with pytest.raises(ValueError, match="prefix must lie"):
            tctx.prompt_plan([16], 4, 2, prefixes=prefixes)
    with pytest.raises(ValueError, match="values are needed"):
        tctx.prompt_plan([16], 4, 2, prefixes=[1, 2])
    del rows
    f.cache.close()


def test_null_arguments_are_refused(cvs, tctx):
    import ctypes
    lib, view, bad, h = cvs.load(), cvs.Heads(), cvs.CVS_ERR_INVALID_ARGUMENT, ctypes.c_void_p()
    one = (ctypes.c_int64 * 1)(1)
    assert lib.cvs_prompt_attention_scored_async(None, None, view, view, view, view, None, 0.0, None) == bad
    assert lib.cvs_kv_attention_scored_async(None, None, 0, view, view, None, 0.0, None) == bad
    assert lib.cvs_prompt_plan_create_prefix(None, one, None, one, 1, 1, 1, ctypes.byref(h)) == bad
    # No prefixes at all: a causal plan.
    assert lib.cvs_prompt_plan_create_prefix(tctx.handle, one, None, None, 1, 1, 1, ctypes.byref(h)) == cvs.CVS_OK
    assert lib.cvs_prompt_plan_destroy(h) == cvs.CVS_OK


def test_graphs(cvs):
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = cvs.Context(0, stream=stream.cuda_stream)
        f = Filled(ctx, 1, 900, 32, 2, 64, "bf16")
        (root,) = f.new()
        f.append([root], [9000])
        seqs = f.fork(root, 200)
        f.append(seqs, [1 + i % 5 for i in range(200)])
        q, k, v = (rand(i, 200, h, 64, dtype="bf16") for i, h in enumerate((8, 2, 2)))
        outs, slopes = [torch.empty_like(q) for _ in range(2)], options("both", 8, steep=0.01)[1]
        step, prompt = f.cache.plan(seqs, [1] * 200, heads=8), ctx.prompt_plan([3, 100, 97], 8, 2, prefixes=[0, 50, 97])

        def calls(step, prompt, outs):
            f.cache.attention_async(step, q, outs[0], cap=5.0, slopes=slopes)
            ctx.prompt_attention_async(prompt, q, k, v, outs[1], cap=5.0, slopes=slopes)

        calls(step, prompt, outs)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls(step, prompt, outs)
        del step, prompt
        for seed in (3, 6, 9):
            for i, x in enumerate((q, k, v)):
                x.copy_(rand(seed + i, *x.shape, dtype="bf16"))
            slopes.mul_(2)
            want = [torch.zeros_like(q) for _ in range(2)]
            calls(f.cache.plan(seqs, [1] * 200, heads=8), ctx.prompt_plan([3, 100, 97], 8, 2, prefixes=[0, 50, 97]), want)
            for x in outs:
                x.fill_(9.0)
            graph.replay()
            stream.synchronize()
            assert all(torch.equal(bits(x), bits(y)) for x, y in zip(outs, want)), seed
            torch.randn(1000, 1000, device="cuda").sum().item()
        f.cache.close()
        ctx.close()


def test_streams(cvs):
    """Tensors made on torch's stream behind other work, with a context on its own."""
    from test_attention_streams_gpu import slow
    q, k, v = (rand(i, 300, h, 64, dtype="fp16") for i, h in enumerate((4, 2, 2)))
    slopes = torch.tensor([1.0, 0.5, 0.25, 0.0], device="cuda")
    with cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream) as c:
        want = torch.zeros_like(q)
        c.prompt_attention_async(c.prompt_plan([300], 4, 2), q, k, v, want, cap=3.0, slopes=slopes)
        torch.cuda.synchronize()
    with cvs.Context(0) as c, torch.cuda.stream(torch.cuda.Stream()):
        out, plan = torch.zeros_like(q), c.prompt_plan([300], 4, 2)
        torch.cuda.synchronize()
        c.prompt_attention_async(plan, q, k, v, out, cap=3.0, slopes=slow(slopes))
        junk = torch.full_like(slopes, float("nan"))
        got = out * 1
        torch.cuda.synchronize()
        assert torch.equal(bits(got), bits(want))
        del junk
