"""The paged cache (cvs_kv_*) and attention over it: pages against a model of
their bookkeeping, contents bit for bit, attention against 64 bits (bounds:
attention_oracle.py)."""
import random

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


def rand(seed, *shape, dtype, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * spread).to(TORCH[dtype]).cuda()


def bits(x):
    return x.contiguous().view(torch.int16)


class Filled:
    """A cache and what it should hold: each sequence's keys and values, (layers, tokens, kv_heads, dim) on the GPU."""

    def __init__(self, ctx, layers, pages, page, kv, dim, dtype, seed=0):
        self.cache = ctx.kv_cache(layers, pages, page, kv, dim, dtype)
        self.layers, self.kv, self.dim, self.dtype, self.seed = layers, kv, dim, dtype, seed
        self.held = {}

    def new(self, n=1):
        ids = self.cache.sequences(n)
        for i in ids:
            self.held[i] = [torch.zeros(self.layers, 0, self.kv, self.dim, dtype=TORCH[self.dtype], device="cuda")
                            for _ in "kv"]
        return ids

    def fork(self, parent, n, length=-1):
        ids = self.cache.fork(parent, n, length)
        for i in ids:
            self.held[i] = [x if length < 0 else x[:, :length] for x in self.held[parent]]
        return ids

    def append(self, seqs, tokens, make=None):
        """Extends and writes, in one call each."""
        self.cache.extend(seqs, tokens)
        self.seed += 2
        make = make or (lambda s, *shape: rand(s, *shape, dtype=self.dtype))
        k, v = (make(self.seed + i, self.layers, sum(tokens), self.kv, self.dim) for i in (0, 1))
        plan = self.cache.plan(seqs, tokens)
        self.cache.write_async(plan, k, v)
        at = 0
        for s, t in zip(seqs, tokens):
            self.held[s] = [torch.cat([old, new[:, at:at + t]], dim=1) for old, new in zip(self.held[s], (k, v))]
            at += t

    def check(self, seqs=None):
        """Reads everything back."""
        seqs = list(self.held) if seqs is None else seqs
        lengths = [self.held[s][0].shape[1] for s in seqs]
        assert self.cache.lengths(seqs) == lengths
        t = sum(lengths)
        k, v = (torch.full((self.layers, t, self.kv, self.dim), 9.0, dtype=TORCH[self.dtype], device="cuda")
                for _ in "kv")
        self.cache.read_async(self.cache.plan(seqs, lengths), k, v)
        at = 0
        for s, n in zip(seqs, lengths):
            for got, want in zip((k, v), self.held[s]):
                assert torch.equal(bits(got[:, at:at + n]), bits(want)), f"sequence {s}"
            at += n

    def free(self, seqs):
        self.cache.free(seqs)
        for s in seqs:
            del self.held[s]


class Model:
    """The pages' bookkeeping in a few lines: lowest free id first, copy on write, moves to the front."""

    def __init__(self, pages, page):
        self.free, self.page, self.seqs = set(range(pages)), page, {}

    def take(self):
        p = min(self.free)
        self.free.remove(p)
        return p

    def refs(self, p):
        return sum(p in pages for pages, _ in self.seqs.values())

    def need(self, n):
        return -(-n // self.page)

    def extend(self, s, t):
        pages, n = self.seqs[s]
        if t and n % self.page and self.refs(pages[-1]) > 1:
            pages[-1] = self.take()
        while len(pages) < self.need(n + t):
            pages.append(self.take())
        self.seqs[s] = (pages, n + t)

    def fork(self, s, child, n):
        self.seqs[child] = (self.seqs[s][0][:self.need(n)], n)

    def cut(self, s, n):
        pages = self.seqs[s][0]
        gone = pages[self.need(n):]
        self.seqs[s] = (pages[:self.need(n)], n)
        self.free |= {p for p in gone if not self.refs(p)}

    def drop(self, s):
        pages, _ = self.seqs.pop(s)
        self.free |= {p for p in pages if not self.refs(p)}

    def compact(self, total):
        live = total - len(self.free)
        src = sorted(set(range(live, total)) - self.free)
        to = dict(zip(src, sorted(p for p in self.free if p < live)))
        for s, (pages, n) in self.seqs.items():
            self.seqs[s] = ([to.get(p, p) for p in pages], n)
        self.free = set(range(live, total))


@pytest.mark.parametrize("page,dim,dtype,seed", [(32, 64, "fp16", 1), (32, 80, "bf16", 2), (64, 128, "bf16", 3),
                                                 (128, 24, "fp16", 4)])
def test_any_order_of_calls(tctx, cvs, page, dim, dtype, seed):
    """Random calls: page ids as the model's, contents as written, through forks, copies, cuts and compaction."""
    r = random.Random(seed)
    total = 40
    f, m = Filled(tctx, 2, total, page, 2, dim, dtype, 100 * seed), Model(total, page)
    for s in f.new(2):
        m.seqs[s] = ([], 0)
    for step in range(120):
        seqs = list(f.held)
        do = r.choice(["append", "append", "append", "fork", "cut", "free", "compact", "new"])
        if do == "new" or not seqs:
            for s in f.new(1):
                m.seqs[s] = ([], 0)
        elif do == "append":
            some = r.sample(seqs, r.randint(1, min(4, len(seqs))))
            tokens = [r.choice([0, 1, 2, page - 1, page, page + 1, r.randint(0, 3 * page)]) for _ in some]
            try:
                f.append(some, tokens)
            except RuntimeError as e:
                assert "free pages" in str(e)
                assert len(m.free) < sum(m.need(m.seqs[s][1] + t) - len(m.seqs[s][0]) + 1 for s, t in zip(some, tokens))
                continue
            for s, t in zip(some, tokens):
                m.extend(s, t)
        elif do == "fork" and len(seqs) < 12:
            p = r.choice(seqs)
            n = r.randint(0, m.seqs[p][1])
            for c in f.fork(p, 2, n):
                m.fork(p, c, n)
        elif do == "cut":
            s = r.choice(seqs)
            n = r.randint(0, m.seqs[s][1])
            f.cache.truncate(s, n)
            f.held[s] = [x[:, :n] for x in f.held[s]]
            m.cut(s, n)
        elif do == "free" and len(seqs) > 3:
            some = r.sample(seqs, 2)
            f.free(some)
            for s in some:
                m.drop(s)
        elif do == "compact":
            assert f.cache.compact() == total - len(m.free)
            m.compact(total)
        assert f.cache.free_pages() == len(m.free)
        seqs = list(f.held)
        want = [p for s in seqs for p in m.seqs[s][0]]
        assert f.cache.pages(seqs).tolist() == want, (step, do)
        if step % 10 == 9 or do == "compact":
            f.check()
    f.check()
    f.cache.close()


@pytest.mark.parametrize("dim,page", [(8, 32), (32, 64), (40, 32), (64, 128), (96, 32), (104, 64), (128, 4096)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_written_tokens_come_back(tctx, dim, page, dtype):
    """One token, tiles and pages begun in the middle, several layers at once and one at a time, strided arrays."""
    f = Filled(tctx, 3, 64 if page < 4096 else 4, page, 3, dim, dtype, 7)
    a, b = f.new(2)
    for tokens in ([1, 0], [30, 5], [2, 33], [page, 1], [7, page - 1]):
        f.append([a, b], tokens)
        f.check()
    # One layer at a time, keys and values as views of one array.
    f.cache.extend([a], [9])
    plan = f.cache.plan([a], [9])
    x = rand(5, 3, 9, 8, dim, dtype=dtype)
    for layer in range(3):
        f.cache.write_async(plan, x[layer, :, 2:5], x[layer, :, 5:], layer=layer)
    f.held[a] = [torch.cat([h, x[:, :, o:o + 3]], dim=1) for h, o in zip(f.held[a], (2, 5))]
    f.check()
    f.cache.close()


def attend(f, seqs, tokens, heads, layer=0, seed=50, spread=1.0, scale=None, q=None):
    """Attention of the newest tokens against 64 bits; returns the output."""
    plan = f.cache.plan(seqs, tokens, heads=heads)
    t = sum(tokens)
    q = rand(seed, t, heads, f.dim, dtype=f.dtype, spread=spread) if q is None else q
    out = torch.full_like(q, 7.0)
    lse = torch.full((heads, t), 7.0, device="cuda")
    f.cache.attention_async(plan, q, out, layer, lse, 0.0 if scale is None else scale)
    got, got_lse, at = f64(out), f64(lse), 0
    for s, n in zip(seqs, tokens):
        k, v = (f64(x[layer]) for x in f.held[s])
        limits = [len(k) - n + i + 1 for i in range(n)]
        want, tol, l, l_tol = attention(f64(q[at:at + n]), k, v, limits, f.dtype, scale)
        assert_within(got[at:at + n], want, tol, f"sequence {s}")
        assert_within(got_lse[:, at:at + n], l, l_tol, f"lse of {s}")
        at += n
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim,page", [(4, 4, 64, 32), (8, 2, 128, 64), (5, 1, 80, 32), (3, 3, 24, 128),
                                               (40, 2, 96, 32), (12, 4, 40, 64)])
@pytest.mark.parametrize("new", [1, 5])
def test_sequences_of_many_lengths(tctx, dtype, heads, kv, dim, page, new):
    """Lengths from the new tokens alone on, at and around ends of tiles and pages; one sequence with no new token."""
    lengths = [new, new + 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 17]
    f = Filled(tctx, 2, 80, page, kv, dim, dtype, 11)
    seqs = f.new(len(lengths))
    f.append(seqs, lengths)
    tokens = [new] * (len(seqs) - 1) + [0]
    attend(f, seqs, tokens, heads, layer=1)
    f.cache.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [1, 3, 40])
def test_shared_prefixes(tctx, dtype, new):
    """A tree of forks: of the whole, in the middle of a page and of a tile, at a page's end, two levels deep, and
    sequences of their own beside it, in an order that mixes them."""
    f = Filled(tctx, 1, 200, 32, 2, 64, dtype, 13)
    (root,) = f.new()
    f.append([root], [203])
    first = f.fork(root, 4) + f.fork(root, 2, 100) + f.fork(root, 2, 96) + f.fork(root, 1, 1)
    f.append(first, [new, new + 3, 70, new, new, 45, new, 90, new])
    second = f.fork(first[2], 3) + f.fork(first[7], 2, 100)
    f.append(second, [new, new + 1, 33 + new, new, new + 64])
    alone = f.new(2)
    f.append(alone, [new, 400])
    seqs = [second[1], alone[0], first[3], first[0], second[4], first[8], alone[1], first[5], second[0], first[1],
            second[3], first[6], first[4], second[2]]
    attend(f, seqs, [new] * len(seqs), 8)
    attend(f, seqs, [1 + i % new for i in range(len(seqs))], 8)
    # Forks that have nothing of their own: equal page lists, one a prefix of the other, a page's part.
    same = f.fork(root, 3) + f.fork(root, 1, 64) + f.fork(root, 2, 50)
    attend(f, [root] + same, [min(new, 50)] * 7, 8)
    f.check()
    f.cache.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new,heads", [(1, 8), (3, 2), (40, 4)])
def test_a_tree_of_long_prefixes(tctx, dtype, new, heads):
    """The same tree with more tokens than a small batch has: shared runs three deep, joined with what is behind them."""
    f = Filled(tctx, 1, 300, 32, 2, 64, dtype, 15)
    (root,) = f.new()
    f.append([root], [1203])
    first = f.fork(root, 4) + f.fork(root, 2, 1100) + f.fork(root, 2, 1088) + f.fork(root, 1, 1)
    f.append(first, [new, new + 3, 70, new, new, 45, new, 90, new])
    second = f.fork(first[2], 3) + f.fork(first[7], 2, 1100)
    f.append(second, [new, new + 1, 33 + new, new, new + 64])
    alone = f.new(2)
    f.append(alone, [new, 400])
    seqs = [second[1], alone[0], first[3], first[0], second[4], first[8], alone[1], first[5], second[0], first[1],
            second[3], first[6], first[4], second[2]]
    attend(f, seqs, [new] * len(seqs), heads)
    attend(f, seqs, [1 + i % new for i in range(len(seqs))], heads)
    same = f.fork(root, 3) + f.fork(root, 1, 1056) + f.fork(root, 2, 1050)
    attend(f, [root] + same, [new] * 7, heads)
    f.cache.close()


@pytest.mark.parametrize("dtype,heads", [("fp16", 8), ("bf16", 64)])
def test_long_prefix_split_over_workgroups(tctx, dtype, heads):
    """Thousands of keys for few rows: parts of a row joined, some of them empty for the rows of earlier tokens."""
    f = Filled(tctx, 1, 400, 64, 4, 64, dtype, 17)
    (root,) = f.new()
    f.append([root], [9001])
    seqs = f.fork(root, 3)
    f.append(seqs, [1, 700, 65])
    attend(f, seqs, [1, 1, 1], heads)
    attend(f, seqs, [1, 3, 2], heads, spread=6.0)
    f.cache.close()


def test_scores_of_any_size(tctx):
    for spread in (1e-3, 8.0, 40.0):
        f = Filled(tctx, 1, 40, 32, 2, 64, "bf16", 19)
        seqs = f.new(3)
        f.append(seqs, [1, 300, 77], make=lambda s, *shape: rand(s, *shape, dtype="bf16", spread=spread))
        attend(f, seqs, [1, 2, 3], 4, spread=spread)
        attend(f, seqs, [1, 2, 3], 4, spread=spread, scale=0.3)
        f.cache.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_what_pages_held_before(tctx, dtype):
    """Pages full of NaN and infinities from sequences that ended do not reach later ones, whose last pages they fill up."""
    f = Filled(tctx, 1, 24, 64, 2, 80, dtype, 23)
    for fill in (float("nan"), float("inf"), -float("inf")):
        (s,) = f.new()
        f.append([s], [24 * 64], make=lambda seed, *shape: torch.full(shape, fill, dtype=TORCH[dtype], device="cuda"))
        f.free([s])
        seqs = f.new(5)
        f.append(seqs, [1, 33, 64, 70, 100])
        out = attend(f, seqs, [1] * 5, 4)
        assert torch.isfinite(out.float()).all()
        out = attend(f, seqs, [1, 33, 5, 7, 40], 4)
        assert torch.isfinite(out.float()).all()
        kids = f.fork(seqs[4], 2, 90)  # the page's rest is the parent's
        attend(f, kids + [seqs[4]], [2, 1, 1], 4)
        f.append(kids, [1, 3])
        attend(f, kids + [seqs[4]], [2, 4, 1], 4)
        f.check()
        f.free(seqs + kids)
    f.cache.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan"), "lowest"])
def test_values_in_keys_not_seen(tctx, dtype, value):
    """Tokens before a key do not see it: the same bits whatever it holds; the tokens after it see what it holds."""
    x = torch.finfo(TORCH[dtype]).min if value == "lowest" else value
    got = {}
    for at in (70, 80, 95, 96, 108):  # of 110 tokens, the last 40 of them new
        for fill in (0.0, x):
            def make(seed, *shape):
                t = rand(seed, *shape, dtype=dtype)
                t[:, at] = fill
                return t
            f = Filled(tctx, 1, 8, 32, 2, 64, dtype, 29)
            (s,) = f.new()
            f.append([s], [110], make=make)
            plan = f.cache.plan([s], [40], heads=4)
            q, out = rand(3, 40, 4, 64, dtype=dtype), torch.zeros(40, 4, 64, dtype=TORCH[dtype], device="cuda")
            f.cache.attention_async(plan, q, out)
            got[fill] = out[:at - 70].clone()
            f.cache.close()
        assert torch.equal(bits(got[0.0]), bits(got[x])), at
        assert torch.isfinite(got[x].float()).all()
    if value == "lowest":
        return

    def one_value(seed, *shape):
        t = rand(seed, *shape, dtype=dtype)
        if seed % 2 == 0:  # Filled.append makes the values with the even seed after the keys' odd one
            t[:, 90, :, 3] = x
        return t

    f = Filled(tctx, 1, 8, 32, 2, 64, dtype, 29)
    (s,) = f.new()
    f.append([s], [110], make=one_value)
    out = torch.zeros(40, 4, 64, dtype=TORCH[dtype], device="cuda")
    f.cache.attention_async(f.cache.plan([s], [40], heads=4), rand(3, 40, 4, 64, dtype=dtype), out)
    seen = out[20:, :, 3].float()
    assert torch.isnan(seen).all() if x != x else (seen == x).all()
    assert torch.isfinite(out[:20].float()).all() and torch.isfinite(out[..., 4:].float()).all()
    f.cache.close()


@pytest.mark.parametrize("at", [0, 4000, 9000, 9003])
def test_an_infinite_value_in_one_of_many_parts(tctx, at):
    """Infinite in one column of one key that all rows see: infinite in that column of every row, finite elsewhere, in
    whichever of a long row's parts it stands (the last key of the shared run and one of a row's own among them)."""
    def make(seed, *shape):
        t = rand(seed, *shape, dtype="fp16")
        if seed % 2 == 0 and shape[1] == 9001 and at <= 9000:  # values: Filled.append makes them with the even seed
            t[:, at, :, 3] = float("inf")
        if seed % 2 == 0 and shape[1] != 9001 and at > 9000:
            t[:, :, :, 3] = float("inf")
        return t

    f = Filled(tctx, 1, 400, 64, 4, 64, "fp16", 43)
    (root,) = f.new()
    f.append([root], [9001], make=make)
    seqs = f.fork(root, 3)
    f.append(seqs, [1, 700, 65], make=make)
    q, out = rand(3, 3, 8, 64, dtype="fp16", spread=0.1), torch.zeros(3, 8, 64, dtype=torch.float16, device="cuda")
    f.cache.attention_async(f.cache.plan(seqs, [1, 1, 1], heads=8), q, out)
    assert (out[..., 3] == float("inf")).all()
    assert torch.isfinite(out[..., :3].float()).all() and torch.isfinite(out[..., 4:].float()).all()
    f.cache.close()


@pytest.mark.parametrize("dim,heads", [(64, 8), (128, 4)])
def test_a_whole_prompt_over_the_cache(tctx, dim, heads):
    """Many new tokens at once: rows in blocks whose keys end at different places, alone and behind a shared prefix,
    in one part and in several."""
    f = Filled(tctx, 1, 120, 32, 2, dim, "bf16", 47)
    (a,) = f.new()
    f.append([a], [333])
    attend(f, [a], [333], heads)
    kids = f.fork(a, 2, 301)
    f.append(kids, [150, 7])
    attend(f, kids + [a], [150, 7, 200], heads)
    f.append([a], [1500])
    attend(f, kids + [a], [151, 40, 3], heads)
    f.cache.close()


def test_rows_that_see_nothing_of_a_run(tctx):
    """New tokens that begin inside the shared run: in the runs behind it the first of them have no key."""
    f = Filled(tctx, 1, 60, 32, 2, 64, "fp16", 53)
    (a,) = f.new()
    f.append([a], [64])
    kids = f.fork(a, 3)
    f.append(kids, [100, 33, 500])
    attend(f, kids, [160, 95, 560], 16)
    f.cache.close()


def test_after_memory_runs_out(tctx):
    """A cache that does not fit is refused, and the next calls are not told of it again."""
    with pytest.raises(RuntimeError, match="memory"):
        tctx.kv_cache(1, 40_000, 4096, 8, 128)
    f = Filled(tctx, 1, 8, 32, 2, 64, "fp16", 59)
    (s,) = f.new()
    f.append([s], [50])
    attend(f, [s], [1], 4)
    f.check()
    f.cache.close()


def test_whole_numbers_of_any_kind(tctx):
    f = Filled(tctx, 1, 8, 32, 2, 64, "fp16", 61)
    seqs = np.array(f.new(2))
    f.cache.extend(seqs, torch.tensor([3, 4]))
    assert f.cache.lengths(seqs) == [3, 4]
    f.cache.free(seqs)
    f.cache.close()


def test_layers_past_4_gib(tctx):
    """Pages whose offsets pass 32 bits, in every kernel: written, copied, read and attended to."""
    page, kv, dim = 4096, 8, 128
    f = Filled(tctx, 2, 320, page, kv, dim, "bf16", 31)  # 16 MiB a page, 5 GiB a layer
    (low,) = f.new()
    f.cache.extend([low], [318 * page])
    (s,) = f.new()
    f.append([s], [100])
    assert f.cache.pages([s]).tolist() == [318]
    del f.held[low]
    (kid,) = f.fork(s, 1)
    f.append([kid], [40])
    assert f.cache.pages([kid]).tolist() == [319]
    attend(f, [s, kid], [1, 2], 16, layer=1)
    f.check()
    f.cache.free([low])
    assert f.cache.compact() == 2
    assert f.cache.pages([s, kid]).tolist() == [0, 1]
    f.check()
    attend(f, [s, kid], [1, 2], 16, layer=0)
    f.cache.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("value", [float("inf"), float("nan")])
@pytest.mark.parametrize("length", [3, 33, 64, 1500, 9000])
def test_few_rows_and_a_key_that_only_the_last_sees(tctx, dtype, value, length):
    """Three new tokens of a sequence, in one part and in several: what the last one holds does not reach the others."""
    got = []
    for fill in (0.0, value):
        def make(seed, *shape):
            t = rand(seed, *shape, dtype=dtype)
            t[:, -1] = fill
            return t
        f = Filled(tctx, 1, 300, 32, 2, 80, dtype, 67)
        (s,) = f.new()
        f.append([s], [length], make=make)
        out = torch.zeros(3, 4, 80, dtype=TORCH[dtype], device="cuda")
        f.cache.attention_async(f.cache.plan([s], [3], heads=4), rand(3, 3, 4, 80, dtype=dtype), out)
        got.append(out.clone())
        f.cache.close()
    assert torch.equal(bits(got[0][:2]), bits(got[1][:2]))
    assert torch.isfinite(got[1][:2].float()).all() and not torch.isfinite(got[1][2].float()).any()


def test_same_bits_again(tctx):
    f = Filled(tctx, 1, 200, 64, 2, 128, "bf16", 37)
    (root,) = f.new()
    f.append([root], [5000])
    seqs = f.fork(root, 5)
    f.append(seqs, [1, 20, 300, 4, 90])
    q = rand(3, 5, 16, 128, dtype="bf16")
    outs = [attend(f, seqs, [1] * 5, 16, q=q) for _ in range(3)]
    assert all(torch.equal(bits(outs[0]), bits(o)) for o in outs)
    f.cache.close()


def test_refusals(tctx, cvs):
    for bad, match in (((0, 4, 32, 2, 64), "at least one"), ((1, 0, 32, 2, 64), "at least one"),
                       ((1, 4, 48, 2, 64), "power of two"), ((1, 4, 16, 2, 64), "power of two"),
                       ((1, 4, 32, 2, 60), "multiple of 8"), ((1, 4, 32, 2, 136), "multiple of 8"),
                       ((1, 4, 4096, 512, 128), "512 MiB")):
        with pytest.raises(ValueError, match=match):
            tctx.kv_cache(*bad)
    with pytest.raises(ValueError, match="attention takes"):
        tctx.kv_cache(1, 4, 32, 2, 64, "float32")
    with pytest.raises(RuntimeError):
        tctx.kv_cache(4096, 1 << 20, 4096, 8, 128)
    f = Filled(tctx, 2, 6, 32, 2, 64, "fp16", 41)
    c = f.cache
    a, b = f.new(2)
    f.append([a, b], [40, 10])
    for call, match in ((lambda: c.extend([a, a], [1, 1]), "given twice"), (lambda: c.extend([a], [-1]), "cannot grow"),
                        (lambda: c.extend([99], [1]), "no sequence 99"), (lambda: c.extend([a], [1 << 31]), "grow"),
                        (lambda: c.fork(a, 1, 41), "fork at 41"), (lambda: c.truncate(a, 41), "truncate to 41"),
                        (lambda: c.free([a, a]), "given twice"), (lambda: c.free([99]), "no sequence"),
                        (lambda: c.plan([a], [41]), "has 40 tokens"), (lambda: c.plan([a], [-1]), "tokens"),
                        (lambda: c.plan([a, a], [1, 1]), "given twice"), (lambda: c.plan([a], [1], heads=3), "multiple"),
                        (lambda: c.plan([a], [1, 2]), "values are needed")):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match="3 free pages, 4 are needed"):
        c.extend([a, b], [60, 60])
    assert c.lengths([a, b]) == [40, 10] and c.free_pages() == 3
    k = rand(1, 40, 2, 64, dtype="fp16")
    plan = c.plan([a], [40])
    for call, match in ((lambda: c.write_async(plan, k[:39], k), "plan's 40 tokens"),
                        (lambda: c.write_async(plan, k[:, :1], k), "cache's heads"),
                        (lambda: c.write_async(plan, k.bfloat16(), k), "type"),
                        (lambda: c.write_async(plan, k, k, layer=2), "layers outside"),
                        (lambda: c.write_async(plan, k[None].expand(3, -1, -1, -1), k[None].expand(3, -1, -1, -1)),
                         "layers outside"),
                        (lambda: c.write_async(plan, k[None], k[None].expand(2, -1, -1, -1)), "same layers"),
                        (lambda: c.attention_async(plan, k, k.clone()), "without query heads")):
        with pytest.raises(ValueError, match=match):
            call()
    step = c.plan([a, b], [1, 1], heads=4)
    q = rand(2, 2, 4, 64, dtype="fp16")
    for call, match in ((lambda: c.attention_async(step, q[:1], q), "plan's 2 tokens"),
                        (lambda: c.attention_async(step, q[:, :2], q), "plan's heads"),
                        (lambda: c.attention_async(step, q, q.clone(), layer=2), "layer outside"),
                        (lambda: c.attention_async(step, q, q.clone(), scale=-1.0), "scale")):
        with pytest.raises(ValueError, match=match):
            call()
    (kid,) = f.fork(a, 1)
    with pytest.raises(ValueError, match="sequences share"):
        c.write_async(c.plan([kid], [1]), k[:1], k[:1])
    with pytest.raises(ValueError, match="sequences share"):
        c.write_async(plan, k, k)
    c.extend([a], [1])
    with pytest.raises(ValueError, match="has changed"):
        c.attention_async(step, q, q.clone())
    late = c.plan([kid], [1], heads=4)
    c.free([b, kid])
    with pytest.raises(ValueError, match="no sequence"):
        c.attention_async(late, q[:1], q[:1].clone())
    other = tctx.kv_cache(1, 4, 32, 2, 64, "fp16")
    with pytest.raises(ValueError, match="another cache"):
        other.read_async(plan, k, k)
    lib = cvs.load()
    assert lib.cvs_kv_cache_destroy(c.handle) == cvs.CVS_ERR_INVALID_ARGUMENT
    assert b"plan(s)" in lib.cvs_last_error()
    other.close()
    c.close()
    assert plan.handle is None and c.handle is None


def test_many_levels_of_shared_prefixes(tctx):
    f = Filled(tctx, 1, 601, 32, 1, 32, "bf16")
    (main,) = f.new()
    forks = []
    for _ in range(300):
        f.append([main], [32])
        forks += f.fork(main, 1)
    f.append(forks, [1] * 300)
    attend(f, forks, [1] * 300, 2)
    f.cache.close()


def test_rows_of_an_output_that_overlap(tctx):
    f = Filled(tctx, 3, 4, 32, 2, 16, "fp16")
    (s,) = f.new()
    f.append([s], [40])
    plan = f.cache.plan([s], [40], heads=2)
    room, other = (torch.zeros(3 * 40 * 64, dtype=torch.float16, device="cuda") for _ in "kv")
    good = other.as_strided((3, 40, 2, 16), (1280, 32, 16, 1))
    for strides in ((0, 32, 16), (1272, 32, 16), (16, 32, 16), (1280, 0, 16), (32, 80, 16)):
        bad = room.as_strided((3, 40, 2, 16), (*strides, 1))
        for k, v in ((bad, good), (good, bad)):
            with pytest.raises(ValueError, match="must not overlap"):
                f.cache.read_async(plan, k, v)
    for strides in ((1280, 32, 16), (32, 96, 16), (16, 96, 48), (40, 120, 16)):  # layers outermost, between, innermost
        k = room.zero_().as_strided((3, 40, 2, 16), (*strides, 1))
        f.cache.read_async(plan, k, good)
        assert torch.equal(k, f.held[s][0]) and torch.equal(good, f.held[s][1]), strides
    q = rand(3, 40, 2, 16, dtype="fp16")
    with pytest.raises(ValueError, match="must not overlap"):
        f.cache.attention_async(plan, q, room.as_strided((40, 2, 16), (16, 16, 1)), 0)
    # Inputs may: one row for all tokens and layers.
    row = rand(4, 1, 1, 1, 16, dtype="fp16").expand(3, 40, 2, 16)
    f.cache.write_async(plan, row, row)
    f.cache.read_async(plan, good, room.as_strided((3, 40, 2, 16), (1280, 32, 16, 1)))
    assert torch.equal(good, row)
    f.cache.close()


def test_captured_and_replayed(cvs):
    """A step's calls in a graph, replayed over changed inputs, against the same calls outside it, bit for bit."""
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        ctx = cvs.Context(0, stream=stream.cuda_stream)
        f = Filled(ctx, 2, 96, 32, 2, 64, "bf16")
        (root,) = f.new()
        f.append([root], [2000])
        seqs = f.fork(root, 3)
        f.append(seqs, [1, 40, 7])
        f.cache.extend(seqs, [1, 1, 1])
        step, prompt = f.cache.plan(seqs, [1, 1, 1], heads=8), ctx.prompt_plan([1, 0, 2], 8, 2)
        q, k, v = (torch.empty(3, h, 64, dtype=torch.bfloat16, device="cuda") for h in (8, 2, 2))
        outs = [torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)]

        def calls():
            f.cache.write_async(step, k, v, layer=1)
            f.cache.attention_async(step, q, outs[0], layer=1)
            ctx.prompt_attention_async(prompt, q, k, v, outs[1])
            f.cache.read_async(step, outs[2], outs[3], layer=1)

        def fill(seed):
            for i, x in enumerate((q, k, v)):
                x.copy_(rand(seed + i, *x.shape, dtype="bf16"))

        fill(1)
        calls()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            calls()
        for seed in (10, 20, 30, 40):
            fill(seed)
            calls()
            want = [x.clone() for x in outs]
            for x in outs:
                x.fill_(9.0)
            graph.replay()
            stream.synchronize()
            for x, y in zip(outs, want):
                assert torch.equal(bits(x), bits(y)), seed
        f.cache.close()
        ctx.close()
