"""The example programs run, and pass the checks that they make themselves."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

EXAMPLES = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples")


def load(name):
    spec = importlib.util.spec_from_file_location(name, os.path.join(EXAMPLES, name + ".py"))
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


@pytest.mark.parametrize("sizes", [dict(passages=200, found=8, questions=12, steps=16),
                                   dict(passages=50, found=1, questions=1, steps=3)])
def test_answer_over_passages(sizes):
    load("answer_over_passages").main(quiet=True, **sizes)
