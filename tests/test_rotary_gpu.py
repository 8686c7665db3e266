"""Rotations and norms of heads (cvs_rotate_async, cvs_norm_rotate_async) against 64 bits.

Bounds: rotary_oracle.py, derived from the number formats alone.
"""
import ctypes

import numpy as np
import pytest
import torch

from attention_oracle import TORCH, assert_within, f64
from rotary_oracle import pairs, ready
from test_kv_cache_gpu import bits, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def places(values):
    return torch.tensor(values, dtype=torch.int64, device="cuda")


def check(ctx, cvs, x, at, dtype, dims, interleaved=False, base=10000.0, magnitude=1.0, out=None):
    f = cvs.rotary_frequencies(dims, base)
    rotary = ctx.rotary(dims, frequencies=f, interleaved=interleaved, magnitude=magnitude)
    out = torch.full_like(x, 7.0, memory_format=torch.contiguous_format) if out is None else out
    want, tol = ready(f64(x), dtype, at.tolist(), f, interleaved, magnitude)
    rest = x[..., dims:].clone()
    ctx.rotate_async(rotary, at, x, out)
    assert_within(f64(out), want, tol, f"{dims} of {tuple(x.shape)}")
    assert torch.equal(bits(out[..., dims:].contiguous()), bits(rest.contiguous())), "channels that do not turn"
    rotary.close()
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dim,dims", [(64, 64), (128, 128), (80, 80), (80, 40), (80, 20), (128, 32), (96, 96), (96, 48),
                                      (8, 8), (8, 2), (16, 16), (40, 30), (120, 120), (72, 66), (128, 126), (24, 16)])
def test_heads(tctx, cvs, dtype, interleaved, dim, dims):
    for tokens, heads in ((1, 1), (3, 20), (67, 5), (2, 300)):
        x = rand(dim + tokens, tokens, heads, dim, dtype=dtype)
        check(tctx, cvs, x, places(list(range(7, 7 + tokens))), dtype, dims, interleaved)


@pytest.mark.parametrize("dim", list(range(8, 129, 8)))
def test_every_head_size(tctx, cvs, dim):
    dtype = "fp16" if dim % 16 else "bf16"
    x = rand(dim, 50, 3, dim, dtype=dtype)
    for dims in (dim, 2 * (dim // 4) or 2):
        for interleaved in (False, True):
            check(tctx, cvs, x, torch.arange(50, device="cuda"), dtype, dims, interleaved)


@pytest.mark.parametrize("interleaved", [False, True])
def test_positions(tctx, cvs, interleaved):
    """Far, negative, repeated and unordered positions; the inverse rotation."""
    at = places([0, 5, 5, -5, 1, 100_003, 1_000_001, 2 ** 31 - 1, -2 ** 31, 2 ** 31, 2 ** 40, 0])
    x = rand(1, len(at), 4, 64, dtype="fp16")
    check(tctx, cvs, x, at, "fp16", 64, interleaved, base=500000.0)
    out = check(tctx, cvs, x[:1].expand(len(at), 4, 64).contiguous(), at, "fp16", 64, interleaved)
    assert torch.equal(bits(out[1]), bits(out[2])) and torch.equal(bits(out[0]), bits(x[0]))


def test_frequencies_of_any_kind(tctx, cvs):
    f = np.array([0.0, 1024.0, -1.0, 2 * np.pi, -1024.0, 1e-9, np.pi / 2, 0.5])
    x = rand(1, 40, 3, 16, dtype="bf16")
    at = torch.arange(-20, 20, device="cuda")
    rotary, out = tctx.rotary(16, frequencies=f, magnitude=-1.5), torch.zeros_like(x)
    tctx.rotate_async(rotary, at, x, out)
    want, tol = ready(f64(x), "bf16", at.tolist(), f, False, -1.5)
    # A frequency of 1024 turns 163 times a position: its 64 bits have 8 less behind the point.
    assert_within(out.double().cpu().numpy(), want, tol, "frequencies")


@pytest.mark.parametrize("dim", [64, 80, 128])
def test_strides(tctx, cvs, dim):
    """Views of one projection, head-major arrays, an output in a wider array, one head for all, in place."""
    dtype, t = "bf16", 45
    at = torch.arange(100, 100 + t, device="cuda")
    qkv = rand(1, t, 9, dim, dtype=dtype)
    kept = qkv.clone()
    check(tctx, cvs, qkv[:, 2:7], at, dtype, dim)
    x = rand(2, 6, t, dim, dtype=dtype).transpose(0, 1)
    wide = torch.full((t, 6, dim + 8), 5.0, dtype=TORCH[dtype], device="cuda")
    check(tctx, cvs, x, at, dtype, dim // 2, True, out=wide[..., :dim])
    assert (wide[..., dim:] == 5).all(), "past the output's rows"
    check(tctx, cvs, rand(3, t, 1, dim, dtype=dtype).expand(t, 7, dim), at, dtype, dim)
    check(tctx, cvs, rand(3, 1, 1, dim, dtype=dtype).expand(t, 7, dim), at, dtype, dim)
    for interleaved, dims in ((False, dim), (True, dim), (False, 20)):
        qkv = kept.clone()
        apart = check(tctx, cvs, qkv[:, 2:7], at, dtype, dims, interleaved)
        check(tctx, cvs, qkv[:, 2:7], at, dtype, dims, interleaved, out=qkv[:, 2:7])
        assert torch.equal(bits(qkv[:, 2:7].contiguous()), bits(apart)), "in place"
        assert torch.equal(bits(qkv[:, :2].contiguous()), bits(kept[:, :2].contiguous())), "beside it"
        assert torch.equal(bits(qkv[:, 7:].contiguous()), bits(kept[:, 7:].contiguous())), "beside it"


@pytest.mark.parametrize("heads,kv", [(40, 8), (1, 1), (3, 0)])
@pytest.mark.parametrize("tokens", [1, 17, 700])
def test_sizes_of_a_launch(tctx, cvs, heads, kv, tokens):
    """Few and many tokens: heads of a token in several workgroups, several tokens in one; every element is written."""
    dtype, dim = "fp16", 64
    f = cvs.rotary_frequencies(dim)
    at = torch.arange(tokens, device="cuda")
    q, k = rand(1, tokens, heads, dim, dtype=dtype), rand(2, tokens, kv, dim, dtype=dtype) if kv else None
    qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0) if kv else None
    w = rand(3, dim, dtype=dtype)
    tctx.norm_rotate_async(tctx.rotary(dim), at, q, qo, k, ko, w, w if kv else None)
    for x, o in ((q, qo), (k, ko)):
        if x is not None:
            want, tol = ready(f64(x), dtype, at.tolist(), f, weight=f64(w), eps=1e-6)
            assert_within(f64(o), want, tol, "normed")


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("dim,dims,interleaved", [(128, 128, False), (80, 80, True), (80, 20, False), (64, 32, False),
                                                  (96, 96, False), (8, 4, True), (128, 0, False), (72, 0, False)])
def test_norms(tctx, cvs, dtype, dim, dims, interleaved):
    """Queries and keys with weights of their own, one of them without, weights in fp32; no rotary (dims 0)."""
    t, eps = 37, 1e-5
    q, k = rand(1, t, 6, dim, dtype=dtype, spread=3.0), rand(2, t, 2, dim, dtype=dtype, spread=0.02)
    at = torch.arange(1000, 1000 + t, device="cuda")
    f = cvs.rotary_frequencies(dims) if dims else ()
    rotary = tctx.rotary(dims, interleaved=interleaved) if dims else None
    wq, wk = rand(3, dim, dtype=dtype), rand(4, dim, dtype=dtype)
    for a, b in ((wq, wk), (wq, None), (None, wk), (wq.float(), wk), (wq, wk.float() * 1.001), (None, None)):
        qo, ko = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
        tctx.norm_rotate_async(rotary, at if dims else None, q, qo, k, ko, a, b, eps=eps)
        for x, o, w in ((q, qo, a), (k, ko, b)):
            want, tol = ready(f64(x), dtype, at.tolist(), f, interleaved, weight=None if w is None else f64(w), eps=eps)
            assert_within(f64(o), want, tol, "normed")
        only = torch.full_like(k, 7.0)
        tctx.norm_rotate_async(rotary, at if dims else None, None, None, k, only, None, b, eps=eps)
        assert torch.equal(bits(only), bits(ko)), "keys alone"


@pytest.mark.parametrize("dims,interleaved", [(64, False), (64, True), (12, False), (12, True)])
def test_infinities_stay_in_their_heads(tctx, cvs, dims, interleaved):
    """A head's infinities and NaNs reach that head alone, without a norm their own pair alone."""
    x = rand(1, 9, 5, 64, dtype="fp16")
    rotary, at = tctx.rotary(dims, interleaved=interleaved), torch.arange(1, 10, device="cuda")
    clean, out = torch.zeros_like(x), torch.zeros_like(x)
    tctx.rotate_async(rotary, at, x, clean)
    a, b = pairs(dims, interleaved)
    bad = x.clone()
    bad[4, 2, 1], bad[5, 3, 60], bad[6, 0, 63] = float("inf"), float("nan"), torch.finfo(torch.float16).min
    tctx.rotate_async(rotary, at, bad, out)
    same = torch.ones_like(x, dtype=torch.bool)
    for t, h, c in ((4, 2, 1), (5, 3, 60), (6, 0, 63)):
        same[t, h, c] = False
        for i, j in ((a, b), (b, a)):
            if c in i:
                same[t, h, int(j[list(i).index(c)])] = False
    assert torch.equal(bits(out)[same], bits(clean)[same])
    assert not torch.isfinite(out[4, 2, 1]) and not torch.isfinite(out[5, 3, 60])
    if dims == 12:
        assert out[6, 0, 63] == bad[6, 0, 63], "a channel that does not turn"
    w = rand(2, 64, dtype="fp16")
    tctx.norm_rotate_async(rotary, at, x, clean, q_weight=w)
    tctx.norm_rotate_async(rotary, at, bad, out, q_weight=w)
    whole = torch.ones(9, 5, dtype=torch.bool, device="cuda")
    for t, h in ((4, 2), (5, 3), (6, 0)):
        whole[t, h] = False
    assert torch.equal(bits(out)[whole], bits(clean)[whole])


def test_rows_of_nothing(tctx, cvs):
    """A head of zeros stays zeros; no tokens at all is no error."""
    z = torch.zeros(3, 2, 64, dtype=torch.float16, device="cuda")
    out, rotary, w = torch.full_like(z, 7.0), tctx.rotary(64), torch.ones(64, dtype=torch.float16, device="cuda")
    tctx.norm_rotate_async(rotary, torch.arange(3, device="cuda"), z, out, q_weight=w)
    assert not out.any()
    tctx.rotate_async(rotary, places([]), z[:0], out[:0])
    tctx.norm_rotate_async(rotary, places([]), z[:0], out[:0], z[:0], out[:0], w, w)


def test_refusals(tctx, cvs):
    x = rand(1, 5, 4, 64, dtype="fp16")
    out, at, rotary = torch.full_like(x, 7.0), torch.arange(5, device="cuda"), tctx.rotary(64)
    w = torch.ones(64, dtype=torch.float16, device="cuda")

    def refused(match, call):
        with pytest.raises(ValueError, match=match):
            call()
        torch.cuda.synchronize()
        assert (out == 7).all(), "a refused call wrote"

    refused("turns 128 channels", lambda: tctx.rotate_async(tctx.rotary(128), at, x, out))
    refused("one shape and type", lambda: tctx.rotate_async(rotary, at, x, out[:, :3]))
    refused("one shape and type", lambda: tctx.rotate_async(rotary, at, x, out.view(torch.bfloat16)))
    refused("positions must be 5", lambda: tctx.rotate_async(rotary, at[:4], x, out))
    refused("positions must be 5", lambda: tctx.rotate_async(rotary, at.int(), x, out))
    refused("contiguous", lambda: tctx.rotate_async(rotary, torch.arange(10, device="cuda")[::2], x, out))
    refused("device", lambda: tctx.rotate_async(rotary, at.cpu(), x, out))
    refused("must not overlap", lambda: tctx.rotate_async(rotary, at, x, out[:, :1].expand(5, 4, 64)))
    refused("same tokens", lambda: tctx.norm_rotate_async(rotary, at, x, out, x[:4], torch.zeros_like(x[:4])))
    refused("without k", lambda: tctx.norm_rotate_async(rotary, at, x, out, None, None, w, w))
    refused("needs k_out", lambda: tctx.norm_rotate_async(rotary, at, x, out, x, None))
    refused("q_weight must be 64", lambda: tctx.norm_rotate_async(rotary, at, x, out, q_weight=w[:32]))
    refused("q_weight must be 64", lambda: tctx.norm_rotate_async(rotary, at, x, out, q_weight=w.bfloat16()))
    refused("eps", lambda: tctx.norm_rotate_async(rotary, at, x, out, q_weight=w, eps=-1.0))
    refused("eps", lambda: tctx.norm_rotate_async(rotary, at, x, out, q_weight=w, eps=float("nan")))
    refused("eps", lambda: tctx.norm_rotate_async(rotary, at, x, out, q_weight=w, eps=float("inf")))
    refused("neither", lambda: tctx.norm_rotate_async(rotary, at, None, None))
    with pytest.raises(ValueError, match="requires grad"):
        tctx.rotate_async(rotary, at, x.clone().requires_grad_(), out)
    with pytest.raises(ValueError, match="frequencies"):
        tctx.rotary(64, frequencies=np.ones(31))
    for f in (np.full(32, 1025.0), np.full(32, np.nan)):
        with pytest.raises(ValueError, match="radians"):
            tctx.rotary(64, frequencies=f)
    with pytest.raises(ValueError, match="magnitude"):
        tctx.rotary(64, magnitude=float("inf"))
    with cvs.Context(0) as other:
        refused("another context", lambda: tctx.rotate_async(other.rotary(64), at, x, out))
    lib = cvs.load()
    view = cvs._heads(tctx, x, "x")[0]
    assert lib.cvs_rotate_async(tctx.handle, rotary.handle, None, view, view) == cvs.CVS_ERR_INVALID_ARGUMENT
    assert lib.cvs_rotate_async(tctx.handle, rotary.handle, at.data_ptr(), view, None) == cvs.CVS_ERR_INVALID_ARGUMENT
    hout = cvs._heads(tctx, out, "out")[0]
    assert lib.cvs_rotate_async(tctx.handle, rotary.handle, at.data_ptr() + 4, view, hout) == cvs.CVS_ERR_UNSUPPORTED
    h = ctypes.c_void_p()
    f = (ctypes.c_double * 32)()
    assert lib.cvs_rotary_create(tctx.handle, 64, 5, f, 1.0, ctypes.byref(h)) == cvs.CVS_ERR_INVALID_ARGUMENT
    held = cvs.Context(0)
    r = held.rotary(64)
    assert lib.cvs_context_destroy(held.handle) == cvs.CVS_ERR_INVALID_ARGUMENT, "a rotary is alive"
    r.close()
    held.close()


def test_device_arrays(cvs):
    """Without torch's tensors: the context's own arrays and stream."""
    rng = np.random.default_rng(5)
    x = rng.standard_normal((9, 3, 64)).astype(np.float16)
    at = np.arange(50, 59)
    with cvs.Context(0) as c:
        dx, dat, w = (cvs.DeviceArray.from_host(c, a) for a in (x, at, np.ones(64, np.float32)))
        out = cvs.DeviceArray(c, x.shape, np.float16)
        c.norm_rotate_async(c.rotary(64), dat, dx, out, q_weight=w)
        c.synchronize()
        want, tol = ready(x.astype(np.float64), "fp16", at, cvs.rotary_frequencies(64), weight=np.ones(64), eps=1e-6)
        assert_within(out.to_host().astype(np.float64), want, tol, "device arrays")


def test_streams(cvs):
    """Tensors made on torch's stream behind other work, with a context on its own."""
    from test_attention_streams_gpu import slow
    x, at = rand(1, 300, 4, 64, dtype="fp16"), torch.arange(300, device="cuda")
    with cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream) as c:
        want = torch.zeros_like(x)
        c.rotate_async(c.rotary(64), at, x, want)
    with cvs.Context(0) as c, torch.cuda.stream(torch.cuda.Stream()):
        out = torch.zeros_like(x)
        torch.cuda.synchronize()
        c.rotate_async(c.rotary(64), at * 1, slow(x), out)
        junk = torch.full_like(x, float("nan"))
        got = out * 1
        torch.cuda.synchronize()
        assert torch.equal(bits(got), bits(want))
        del junk


def test_graphs(cvs):
    """Captured calls whose rotary is dropped before the replays, with eager work between them."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        c = cvs.Context(0, stream=stream.cuda_stream)
        q, k = rand(1, 200, 8, 128, dtype="bf16"), rand(2, 200, 2, 128, dtype="bf16")
        qo, ko, at, w = torch.zeros_like(q), torch.zeros_like(k), torch.arange(200, device="cuda"), rand(3, 128, dtype="bf16")
        rotary = c.rotary(128)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            c.norm_rotate_async(rotary, at, q, qo, k, ko, w, w)
            with pytest.raises(ValueError, match="captured"):
                c.rotary(64)
        del rotary
        others = [c.rotary(128, base=3.0) for _ in range(4)]  # not in the captured one's memory
        for seed in range(3):
            q.copy_(rand(seed, 200, 8, 128, dtype="bf16"))
            at.add_(1000)
            fresh, want = c.rotary(128), [torch.zeros_like(x) for x in (q, k)]
            c.norm_rotate_async(fresh, at, q, want[0], k, want[1], w, w)
            qo.fill_(9.0), ko.fill_(9.0)
            graph.replay()
            stream.synchronize()
            assert torch.equal(bits(qo), bits(want[0])) and torch.equal(bits(ko), bits(want[1])), seed
            torch.randn(1000, 1000, device="cuda").sum().item()
        del others
        c.close()


def test_far_apart_rows(tctx, cvs):
    """Rows that span more than 4 GiB, token by token and head by head."""
    room = torch.empty(5 << 29, dtype=torch.float16, device="cuda")  # 5 GiB
    for tokens, heads, strides in ((300, 3, (1 << 23, 64)), (5, 70, (64, 36 << 20))):
        x = room.as_strided((tokens, heads, 64), (*strides, 1))
        x.copy_(rand(1, tokens, heads, 64, dtype="fp16"))
        at = torch.arange(9, 9 + tokens, device="cuda")
        for interleaved in (False, True):
            apart = check(tctx, cvs, x, at, "fp16", 64, interleaved)
            check(tctx, cvs, apart, at, "fp16", 64, interleaved, out=x)
            x.copy_(rand(1, tokens, heads, 64, dtype="fp16"))


def test_tiny_and_large_heads(tctx):
    """Norms of values whose squares leave the range of fp16, and are as small as fp32 holds; zeros keep their sign."""
    for dtype, sizes in (("fp16", (2.0 ** -24, 1e-4, 6e4)), ("bf16", (1e-17, 1e-10, 1e15))):
        for size in sizes:
            x = (rand(1, 6, 3, 64, dtype="bf16").float().sign() * size).to(TORCH[dtype])
            w, out = torch.ones(64, dtype=TORCH[dtype], device="cuda"), torch.zeros_like(x)
            tctx.norm_rotate_async(None, None, x, out, q_weight=w, eps=0.0)
            want, tol = ready(f64(x), dtype, weight=f64(w))
            assert_within(f64(out), want, tol, f"{dtype} {size}")
    x = torch.zeros(2, 1, 64, dtype=torch.float16, device="cuda")
    x[1] = -0.0
    out = torch.full_like(x, 7.0)
    tctx.rotate_async(tctx.rotary(32), places([3, 4]), x, out)
    assert torch.equal(bits(out[..., 32:]), bits(x[..., 32:]))


def test_positions_and_their_rotary(cvs, tctx):
    """A closed rotary, and positions that nothing would use, are refused rather than passed over."""
    x = rand(1, 5, 4, 64, dtype="fp16")
    out, at = torch.full_like(x, 7.0), torch.arange(5, device="cuda")
    w = torch.ones(64, dtype=torch.float16, device="cuda")
    closed = tctx.rotary(64)
    closed.close()
    cache = tctx.kv_cache(1, 4, 32, 4, 64, "fp16")
    seqs = cache.sequences(1)
    cache.extend(seqs, [5])
    plan = cache.plan(seqs, [5])
    for match, call in (
            ("null rotary", lambda: tctx.rotate_async(closed, at, x, out)),
            ("closed", lambda: tctx.norm_rotate_async(closed, at, x, out, q_weight=w)),
            ("closed", lambda: tctx.norm_rotate_async(closed, None, x, out, q_weight=w)),
            ("closed", lambda: cache.append_async(plan, x, x, rotary=closed, q=x, q_out=out)),
            ("without a rotary", lambda: tctx.norm_rotate_async(None, at, x, out, q_weight=w)),
            ("null positions", lambda: tctx.norm_rotate_async(tctx.rotary(64), None, x, out, q_weight=w))):
        with pytest.raises(ValueError, match=match):
            call()
        torch.cuda.synchronize()
        assert (out == 7).all(), "a refused call wrote"
    cache.close()
