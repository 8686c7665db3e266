"""The example program with rotary positions and normed heads, and the checks that it makes itself."""
import pytest

from test_examples_gpu import load

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sizes", [dict(passages=200, found=8, questions=12, steps=16),
                                   dict(passages=50, found=1, questions=1, steps=3)])
def test_answer_over_passages(sizes):
    load("answer_over_passages").main(quiet=True, positions="rotary", **sizes)
