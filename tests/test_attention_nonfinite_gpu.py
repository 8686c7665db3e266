"""Infinities and NaNs in the keys and values of attention: rows that do not see them, however many heads share a key,
rows that see several, and what they cost."""
import math

import pytest
import torch

from attention_oracle import TORCH
from test_kv_cache_gpu import Filled, bits, rand

pytestmark = pytest.mark.gpu

INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def tctx(cvs):
    c = cvs.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    c.close()


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("heads,kv", [(127, 1), (128, 1), (192, 1), (256, 2)])
@pytest.mark.parametrize("ql,kl", [(2, 2), (3, 40), (5, 64), (70, 70)])
def test_hidden_from_rows_of_one_token(tctx, dtype, value, heads, kv, ql, kl):
    """With 128 and more heads on a key, a block's rows may all be one token's, and hide the same keys."""
    q, k, v = (rand(i, n, h, 64, dtype=dtype) for i, (n, h) in enumerate(((ql, heads), (kl, kv), (kl, kv))))
    plan = tctx.prompt_plan([ql], heads, kv, [kl])
    for at in sorted({kl - 1, kl - ql + 1}):  # seen from query at - (kl - ql) on
        got = []
        for fill in (0.0, value):
            kk, vv = k.clone(), v.clone()
            kk[at], vv[at] = fill, fill
            out = torch.empty_like(q)
            tctx.prompt_attention_async(plan, q, kk, vv, out)
            got.append(out[:at - (kl - ql)])
        assert torch.equal(bits(got[0]), bits(got[1])), at
        assert torch.isfinite(got[1].float()).all()


COLUMN = 3


def check_column(out, other, limits, placed):
    """`other`: the same call with zeros in the column. Rows that see none of `placed` (key -> value) are finite there,
    the others have what their infinities and NaNs sum to; the other columns have the same bits."""
    x = out[..., COLUMN].float().cpu()
    for i, n in enumerate(limits):
        seen = [v for key, v in placed.items() if key < n]
        if not seen:
            assert torch.isfinite(x[i]).all(), i
        elif math.isnan(sum(seen)):
            assert torch.isnan(x[i]).all(), (i, seen)
        else:
            assert (x[i] == sum(seen)).all(), (i, seen)
    rest = [c for c in range(out.shape[-1]) if c != COLUMN]
    assert torch.equal(bits(out[..., rest]), bits(other[..., rest]))


PLACED = [{3: INF, 200: -INF}, {0: -INF, 64: -INF, 250: NAN}, {90: INF, 95: INF, 297: INF}, {260: NAN}, {299: -INF}]


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads,kv,dim", [(4, 4, 64), (8, 2, 80), (2, 1, 128), (130, 1, 64)])
@pytest.mark.parametrize("placed", PLACED)
def test_seen_in_prompts(tctx, dtype, heads, kv, dim, placed):
    q, k, v = (rand(i, 300, h, dim, dtype=dtype, spread=0.3) for i, h in enumerate((heads, kv, kv)))
    plan = tctx.prompt_plan([300], heads, kv)
    out, other = torch.empty_like(q), torch.empty_like(q)
    v[..., COLUMN] = 0.0
    tctx.prompt_attention_async(plan, q, k, v, other)
    for key, x in placed.items():
        v[key, :, COLUMN] = x
    tctx.prompt_attention_async(plan, q, k, v, out)
    check_column(out, other, range(1, 301), placed)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("shift", [0, 1500, 9000])
@pytest.mark.parametrize("new,heads,dim", [(5, 4, 64), (3, 2, 128), (200, 8, 80)])
@pytest.mark.parametrize("placed", PLACED)
def test_seen_in_a_cache(tctx, dtype, shift, new, heads, dim, placed):
    """The newest tokens of 300 behind `shift` others: few rows and many, in one part and in several."""
    outs = []
    for column in (False, True):
        def make(seed, *shape):
            t = rand(seed, *shape, dtype=dtype, spread=0.3)
            if seed % 2 == 0:  # the values: Filled.append makes them with the even seed
                t[..., COLUMN] = 0.0
                for key, x in placed.items() if column else ():
                    t[:, shift + key, :, COLUMN] = x
            return t
        f = Filled(tctx, 1, 300, 32, 2, dim, dtype, 71)
        (s,) = f.new()
        f.append([s], [shift + 300], make=make)
        outs.append(torch.empty(new, heads, dim, dtype=TORCH[dtype], device="cuda"))
        q = rand(3, new, heads, dim, dtype=dtype, spread=0.3)
        f.cache.attention_async(f.cache.plan([s], [new], heads=heads), q, outs[-1])
        f.cache.close()
    check_column(outs[1], outs[0], range(301 - new, 301), placed)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("heads", [4, 80])
def test_seen_by_some_sequences_of_a_run(tctx, dtype, heads):
    """Forks that keep 100, 700 and all 1,500 tokens of one sequence: a run's rows end far from each other."""
    placed = {50: INF, 690: -INF, 1400: NAN}
    lengths, outs = [100, 700, 1500], []
    for column in (False, True):
        def make(seed, *shape):
            t = rand(seed, *shape, dtype=dtype, spread=0.3)
            if seed % 2 == 0:
                t[..., COLUMN] = 0.0
                for key, x in placed.items() if column else ():
                    t[:, key, :, COLUMN] = x
            return t
        f = Filled(tctx, 1, 4, 4096, 2, 64, dtype, 73)  # one page: a run of all three
        (s,) = f.new()
        f.append([s], [1500], make=make)
        kids = [f.fork(s, 1, n)[0] for n in lengths]
        outs.append(torch.empty(3, heads, 64, dtype=TORCH[dtype], device="cuda"))
        q = rand(3, 3, heads, 64, dtype=dtype, spread=0.3)
        f.cache.attention_async(f.cache.plan(kids, [1, 1, 1], heads=heads), q, outs[-1])
        f.cache.close()
    check_column(outs[1], outs[0], lengths, placed)


@pytest.mark.parametrize("value", [INF, NAN])
def test_what_they_cost(tctx, value):
    """Values of nothing but infinities or NaNs, as a model that has diverged makes them: a row looks again at the keys
    that its block hides from some row (32 tokens of 128 rows, and up to 160 keys of the tiles at their ends), not at all
    4,096. 192 keys are 24 times 8 loads under way at once for each of 32 pairs of columns: 0.8 ms at 1 us each, one
    round of workgroups; 3 ms leaves room. All the row's keys one after another took 14 ms."""
    n = 4096
    q, k = rand(1, n, 8, 64, dtype="bf16"), rand(2, n, 2, 64, dtype="bf16")
    v, out = torch.full_like(k, value), torch.empty_like(q)
    plan = tctx.prompt_plan([n], 8, 2)
    times = []
    for _ in range(5):
        start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        tctx.prompt_attention_async(plan, q, k, v, out)
        stop.record()
        stop.synchronize()
        times.append(start.elapsed_time(stop))
    assert sorted(times)[2] < 3.0, times
    assert not torch.isfinite(out.float()).any()
