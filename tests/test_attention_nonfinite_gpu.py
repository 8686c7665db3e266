"""Infinities and NaNs in the keys and values of attention: rows that do not see them, however many heads share a key."""
import pytest
import torch

from test_kv_cache_gpu import bits, rand

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
