"""examples/one_page_many_answers.py: the static prefill, the pool and both attentions together."""

import importlib.util
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu


def test_one_page_many_answers(pkg, lib):
    at = Path(__file__).resolve().parents[1] / "examples" / "one_page_many_answers.py"
    spec = importlib.util.spec_from_file_location("one_page_many_answers", at)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    got = mod.run(answers=5, steps=6, prompt=600, window=200, sinks=4, page=32)
    # 18 full pages shared, one partly filled page each
    assert got["pages for the prompt and its branches"] == 19 + 5
    # each output is within one rounding of a weight (2^-8 of the mean |v|, below 1 here) and its own
    assert got["largest difference, shared prompt against each for itself"] <= 2.0**-8 * 1.5 + 2.0**-7
    assert got["their outputs unchanged by the move"]
    assert got["pages of the answers that go on"] <= got["pages through the window"]
