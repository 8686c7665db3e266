"""New tokens into the cache with their norm and rotation on the way (cvs_kv_append_async): against 64 bits, and bit for
bit what the norm and rotation from array to array and a write would leave."""
import pytest
import torch

from attention_oracle import TORCH, assert_within, f64
from rotary_oracle import ready
from test_kv_cache_gpu import bits, rand

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


def filled(ctx, lengths, new, kv, dim, dtype, page=32, layers=1, prefix=0):
    """A cache whose sequences hold `lengths` tokens (forks of `prefix` shared ones and their own), `new` of them to come."""
    pages = -(-prefix // page) + sum(-(-(n + m) // page) + 2 for n, m in zip(lengths, new))
    cache = ctx.kv_cache(layers, pages, page, kv, dim, dtype)
    root = cache.sequence()
    cache.extend([root], [prefix])
    k, v = (rand(90 + i, layers, prefix, kv, dim, dtype=dtype) for i in (0, 1))
    cache.write_async(cache.plan([root], [prefix]), k, v)
    seqs = cache.fork(root, len(lengths)) if prefix else cache.sequences(len(lengths))
    cache.extend(seqs, lengths)
    total = [prefix + n for n in lengths]
    k, v = (rand(92 + i, layers, sum(lengths), kv, dim, dtype=dtype) for i in (0, 1))
    cache.write_async(cache.plan(seqs, lengths), k, v)
    cache.extend(seqs, new)
    return cache, seqs, total


def contents(cache, seqs, dtype):
    lengths = cache.lengths(seqs)
    out = [torch.full((cache.layers, sum(lengths), cache.kv_heads, cache.head_dim), 9.0, dtype=TORCH[dtype], device="cuda")
           for _ in "kv"]
    cache.read_async(cache.plan(seqs, lengths), *out)
    return out


def check(ctx, cvs, lengths, new, heads, kv, dim, dims, dtype, interleaved=False, norms=(True, True), page=32, layers=1,
          layer=0, prefix=0, positions=None, seed=1):
    t = sum(new)
    qkv = rand(seed, t, heads + 2 * kv, dim, dtype=dtype, spread=2.0)
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kv], qkv[:, heads + kv:]
    wq, wk = (rand(seed + 1 + i, dim, dtype=dtype) if n else None for i, n in enumerate(norms))
    f = cvs.rotary_frequencies(dims, 500000.0) if dims else ()
    rotary = ctx.rotary(dims, 500000.0, interleaved, magnitude=1.25) if dims else None
    args = (ctx, lengths, new, kv, dim, dtype, page, layers, prefix)
    cache, seqs, total = filled(*args)
    own = [p for n, m in zip(total, new) for p in range(n, n + m)]
    at = None if positions is None else torch.tensor(positions, device="cuda")
    places = own if positions is None else positions
    plan = cache.plan(seqs, new)
    q_out = torch.full((t, heads, dim), 7.0, dtype=TORCH[dtype], device="cuda")
    cache.append_async(plan, k, v, layer, rotary, at, wk, q, q_out, wq, eps=1e-5)

    # The new tokens against 64 bits.
    ko, vo = torch.zeros_like(k), torch.zeros_like(v)
    cache.read_async(plan, ko, vo, layer)
    for x, w, got, what in ((q, wq, q_out, "q"), (k, wk, ko, "k")):
        want, tol = ready(f64(x), dtype, places, f, interleaved, 1.25, None if w is None else f64(w), 1e-5)
        assert_within(f64(got), want, tol, what)
    assert torch.equal(bits(vo), bits(v))

    # All that the cache holds against a write of the same.
    other, others, _ = filled(*args)
    qr, kr = torch.zeros_like(q_out), torch.zeros_like(ko)
    ctx.norm_rotate_async(rotary, torch.tensor(places, device="cuda") if dims else None, q, qr, k, kr, wq, wk, eps=1e-5)
    other.write_async(other.plan(others, new), kr, v, layer)
    assert torch.equal(bits(qr), bits(q_out))
    # Layers that the call does not write hold nothing in the new tokens: of those, compare what was there.
    for a, b in zip(contents(cache, seqs, dtype), contents(other, others, dtype)):
        assert torch.equal(bits(a[layer]), bits(b[layer]))
        at0 = 0
        for n, m in zip(total, new):
            assert torch.equal(bits(a[:, at0:at0 + n]), bits(b[:, at0:at0 + n]))
            at0 += n + m
    alone, only, _ = filled(*args)
    alone.append_async(alone.plan(only, new), k, v, layer, rotary, at, wk, eps=1e-5)
    for a, b in zip(contents(cache, seqs, dtype), contents(alone, only, dtype)):
        assert torch.equal(bits(a[layer]), bits(b[layer])), "without queries"
    for c in (cache, other, alone):
        c.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("kv,dim,dims", [(2, 64, 64), (8, 128, 128), (1, 80, 80), (4, 80, 20), (3, 96, 48), (5, 8, 4),
                                         (2, 40, 32), (9, 72, 72), (1, 128, 64), (2, 120, 120), (2, 32, 32), (6, 16, 6)])
def test_heads(tctx, cvs, dtype, interleaved, kv, dim, dims):
    """Spans that begin and end inside tiles and pages, a token, whole tiles, none."""
    lengths, new = [0, 1, 31, 32, 33, 70, 64, 5], [1, 1, 1, 32, 95, 60, 0, 27]
    check(tctx, cvs, lengths, new, 2 * kv, kv, dim, dims, dtype, interleaved, page=64)


@pytest.mark.parametrize("dim", list(range(8, 129, 8)))
def test_every_head_size(tctx, cvs, dim):
    dtype = "fp16" if dim % 16 else "bf16"
    check(tctx, cvs, [3, 40], [50, 3], 3, 3, dim, dim, dtype, dim % 3 == 0)


@pytest.mark.parametrize("norms", [(True, False), (False, True), (False, False)])
@pytest.mark.parametrize("dims", [0, 64, 22])
def test_without_norms_or_rotary(tctx, cvs, norms, dims):
    check(tctx, cvs, [3, 40], [50, 3], 8, 2, 64, dims, "bf16", norms=norms)


def test_shared_pages_and_layers(tctx, cvs):
    """Forks of a prefix whose last page each has a copy of; one layer of three."""
    check(tctx, cvs, [0, 0, 3], [1, 9, 40], 4, 2, 64, 64, "fp16", layers=3, layer=1, prefix=77)
    check(tctx, cvs, [0, 1], [1, 1], 4, 2, 64, 64, "fp16", layers=3, layer=2, prefix=64)


def test_positions_of_the_callers(tctx, cvs):
    new = [4, 1, 40]
    at = [100_000 + 7 * i for i in range(44)] + [-3]
    check(tctx, cvs, [10, 0, 31], new, 4, 2, 64, 64, "fp16", positions=at)


@pytest.mark.parametrize("page", [32, 128, 4096])
def test_many_sequences(tctx, cvs, page):
    """More spans than a launch has as arguments; spans of few tokens in large pages, and of many."""
    new = [1 + i % 3 for i in range(250)]
    check(tctx, cvs, [i % 40 for i in range(250)], new, 4, 2, 16, 16, "fp16", page=page)
    check(tctx, cvs, [3, 500], [2000, 777], 5, 5, 64, 64, "bf16", page=page)


@pytest.mark.parametrize("heads,kv,dim,dims", [(40, 5, 128, 128), (32, 1, 64, 24), (63, 1, 80, 80), (24, 2, 128, 22)])
def test_query_parts(tctx, cvs, heads, kv, dim, dims):
    """Tiles whose queries several workgroups share by their tokens, tiles of fewer tokens than workgroups among them."""
    check(tctx, cvs, [0, 7, 31, 64, 3], [333, 95, 1, 3, 640], heads, kv, dim, dims, "bf16", dims == 128, page=64)


def test_a_long_sequence(tctx, cvs):
    """Positions past 100,000 from the cache's own places."""
    cache = tctx.kv_cache(1, 1001, 128, 1, 64, "bf16")
    (s,) = cache.sequences(1)
    cache.extend([s], [128_000])
    cache.extend([s], [5])
    k = rand(1, 5, 1, 64, dtype="bf16")
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    plan = cache.plan([s], [5])
    cache.append_async(plan, k, k, rotary=tctx.rotary(64, interleaved=True))
    cache.read_async(plan, ko, vo)
    want, tol = ready(f64(k), "bf16", list(range(128_000, 128_005)), cvs.rotary_frequencies(64), True)
    assert_within(f64(ko), want, tol, "keys")
    cache.close()


def test_queries_in_place_and_strides(tctx, cvs):
    cache, seqs, total = filled(tctx, [5, 60], [3, 70], 2, 64, "fp16")
    rotary, plan = tctx.rotary(64), cache.plan(seqs, [3, 70], heads=6)
    qkv = rand(5, 73, 10, 64, dtype="fp16")
    kept = qkv.clone()
    q, k, v = qkv[:, :6], qkv[:, 6:8], qkv[:, 8:]
    out = torch.zeros(73, 6, 64, dtype=torch.float16, device="cuda")
    cache.append_async(plan, k, v, rotary=rotary, q=q, q_out=out)
    cache.append_async(plan, k, v, rotary=rotary, q=q, q_out=q)
    assert torch.equal(bits(q), bits(out)) and torch.equal(bits(qkv[:, 6:]), bits(kept[:, 6:]))
    want = contents(cache, seqs, "fp16")
    kt, vt = (x.transpose(0, 1).contiguous().transpose(0, 1) for x in (k, v))
    cache.append_async(plan, kt, vt, rotary=rotary)
    one = k[:, :1].expand(73, 2, 64)
    for a, b in zip(contents(cache, seqs, "fp16"), want):
        assert torch.equal(bits(a), bits(b))
    cache.append_async(plan, one, one)
    got = torch.zeros(2, 73, 2, 64, dtype=torch.float16, device="cuda")
    cache.read_async(plan, got[0], got[1])
    assert torch.equal(bits(got[0]), bits(one)) and torch.equal(bits(got[1]), bits(one))
    cache.close()


def test_infinities_stay_in_their_rows(tctx, cvs):
    cache, seqs, _ = filled(tctx, [5], [40], 2, 80, "fp16")
    rotary, plan, w = tctx.rotary(80), cache.plan(seqs, [40]), rand(1, 80, dtype="fp16")
    k, v = rand(2, 40, 2, 80, dtype="fp16"), rand(3, 40, 2, 80, dtype="fp16")
    outs = []
    for bad in (False, True):
        if bad:
            k[7, 1, 3], k[39, 0, 70], v[20, 1, 11] = float("inf"), float("nan"), float("nan")
        cache.append_async(plan, k, v, rotary=rotary, k_weight=w)
        outs.append([torch.zeros_like(k), torch.zeros_like(v)])
        cache.read_async(plan, *outs[-1])
    same = torch.ones(40, 2, dtype=torch.bool, device="cuda")
    same[7, 1] = same[39, 0] = False
    assert torch.equal(bits(outs[0][0])[same], bits(outs[1][0])[same])
    assert torch.equal(bits(outs[1][1]), bits(v))
    cache.close()


def test_refusals(tctx, cvs):
    cache, seqs, _ = filled(tctx, [5, 60], [3, 7], 2, 64, "fp16")
    before = contents(cache, seqs, "fp16")
    rotary, plan = tctx.rotary(64), cache.plan(seqs, [3, 7], heads=4)
    q, k = rand(1, 10, 4, 64, dtype="fp16"), rand(2, 10, 2, 64, dtype="fp16")
    out, w = torch.full_like(q, 7.0), torch.ones(64, dtype=torch.float16, device="cuda")

    def refused(match, *args, **kw):
        with pytest.raises(ValueError, match=match):
            cache.append_async(*args, **kw)
        for a, b in zip(contents(cache, seqs, "fp16"), before):
            assert torch.equal(bits(a), bits(b)), "a refused call wrote"
        assert (out == 7).all(), "a refused call wrote"

    refused("10 tokens", plan, k[:9], k)
    refused("heads, head_dim and type", plan, k[:, :1], k)
    refused("heads, head_dim and type", plan, k, k.bfloat16())
    refused("layers outside", plan, k, k, layer=1)
    refused("turns 80 channels", plan, k, k, rotary=tctx.rotary(80))
    refused("positions must be 10", plan, k, k, rotary=rotary, positions=torch.arange(9, device="cuda"))
    refused("without a rotary", plan, k, k, positions=torch.arange(10, device="cuda"))
    refused("without q", plan, k, k, rotary=rotary, q_out=out)
    refused("without q", plan, k, k, rotary=rotary, q_weight=w)
    refused("needs q_out", plan, k, k, rotary=rotary, q=q)
    refused("10 tokens", plan, k, k, rotary=rotary, q=q[:9], q_out=out)
    refused("the heads of q", plan, k, k, rotary=rotary, q=q, q_out=out[:, :3])
    refused("the plan's heads", plan, k, k, rotary=rotary, q=q[:, :2], q_out=out[:, :2])
    refused("must not overlap", plan, k, k, rotary=rotary, q=q, q_out=out[:1].expand(10, 4, 64))
    refused("k_weight must be 64", plan, k, k, rotary=rotary, k_weight=w[:8])
    refused("eps", plan, k, k, rotary=rotary, k_weight=w, eps=-1.0)
    refused("requires grad", plan, k.clone().requires_grad_(), k)
    with cvs.Context(0) as ctx:
        refused("another context", plan, k, k, rotary=ctx.rotary(64))
        fork = ctx.kv_cache(1, 4, 32, 2, 64, "fp16")
        with pytest.raises(ValueError, match="another cache"):
            fork.append_async(plan, k, k)
    kid = cache.fork(seqs[0], 1)
    refused("share", plan, k, k, rotary=rotary)
    cache.free(kid)
    cache.append_async(plan, k, k, rotary=rotary, q=q, q_out=out)
    cache.extend(seqs[:1], [1])
    with pytest.raises(ValueError, match="has changed"):
        cache.append_async(plan, k, k)
    empty = cache.plan(seqs, [0, 0])
    cache.append_async(empty, k[:0], k[:0], rotary=rotary, q=q[:0], q_out=out[:0])
    lib = cvs.load()
    view = cvs._heads(tctx, k, "k")[0]
    bad = cvs.CVS_ERR_INVALID_ARGUMENT
    plan = cache.plan(seqs, [3, 7])
    assert lib.cvs_kv_append_async(cache.handle, None, 0, None, None, view, None, view, None, None, None) == bad
    assert lib.cvs_kv_append_async(cache.handle, plan.handle, 0, None, None, None, None, view, None, None, None) == bad
    assert lib.cvs_kv_append_async(cache.handle, plan.handle, 0, None, None, view, None, view, view, None, None) == bad
    del plan, empty
    cache.close()


def test_graphs(cvs):
    """Captured with its plan's spans in device memory and its rotary, both dropped before the replays."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = cvs.Context(0, stream=stream.cuda_stream)
        cache, seqs, _ = filled(ctx, [9] * 220, [1] * 220, 2, 64, "bf16")
        q, k, v = (rand(i, 220, h, 64, dtype="bf16") for i, h in enumerate((4, 2, 2)))
        out, ko, vo = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        rotary, plan = ctx.rotary(64), cache.plan(seqs, [1] * 220)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            cache.append_async(plan, k, v, rotary=rotary, q=q, q_out=out)
            cache.read_async(plan, ko, vo)
        del rotary, plan
        others = [cache.plan(seqs[i:] + seqs[:i], [1] * 220) for i in (1, 5, 100)]
        more = [ctx.rotary(64, base=2.0) for _ in range(3)]
        for seed in (3, 6, 9):
            for i, x in enumerate((q, k, v)):
                x.copy_(rand(seed + i, *x.shape, dtype="bf16"))
            want = [torch.zeros_like(x) for x in (q, k, v)]
            plan, rotary = cache.plan(seqs, [1] * 220), ctx.rotary(64)
            cache.append_async(plan, k, v, rotary=rotary, q=q, q_out=want[0])
            cache.read_async(plan, want[1], want[2])
            cache.append_async(plan, v, k)  # what the replay has to put right
            for x in (out, ko, vo):
                x.fill_(9.0)
            graph.replay()
            stream.synchronize()
            for x, y in zip((out, ko, vo), want):
                assert torch.equal(bits(x), bits(y)), seed
            torch.randn(1000, 1000, device="cuda").sum().item()
        del others, more, plan
        cache.close()
        ctx.close()


def test_past_4_gib(tctx, cvs):
    """A page whose place in the pool and whose tokens' positions are far."""
    cache = tctx.kv_cache(1, 300, 4096, 8, 128, "bf16")
    (s,) = cache.sequences(1)
    n = 299 * 4096 + 7
    cache.extend([s], [n])
    cache.extend([s], [40])
    q, k, v = (rand(i, 40, h, 128, dtype="bf16") for i, h in enumerate((16, 8, 8)))
    plan, w = cache.plan([s], [40]), rand(5, 128, dtype="bf16")
    out, ko, vo = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    cache.append_async(plan, k, v, rotary=tctx.rotary(128, 500000.0), k_weight=w, q=q, q_out=out)
    cache.read_async(plan, ko, vo)
    f, at = cvs.rotary_frequencies(128, 500000.0), list(range(n, n + 40))
    for x, got, weight in ((q, out, None), (k, ko, w)):
        want, tol = ready(f64(x), "bf16", at, f, weight=None if weight is None else f64(weight), eps=1e-6)
        assert_within(f64(got), want, tol, "past 4 GiB")
    assert torch.equal(bits(vo), bits(v))
    del plan
    cache.close()
