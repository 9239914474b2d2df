"""The example that trains, quantises, scores and draws runs, and its answers
are those of the model it trained."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "answer_quantized.py")


def test_answer_quantized_example(cuda):
    spec = importlib.util.spec_from_file_location("answer_quantized", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(m=50, d=130, n=1500, epochs=3)
    print(got)
    # Each operand is off by half a step of 1/127 of its largest entry at
    # most: about 1/254 sqrt(2) times the largest over the mean entry of a
    # Gaussian row (some 3 over 1), in the norm.
    assert got["score_error"] < 0.03
    assert got["agree_32_bits"] > 0.95
    assert abs(got["right_best"] - got["right_32_bits"]) < 0.03
    assert got["right_best"] > 0.5  # it has learnt something (2 in 100 by chance)
    assert 0 < got["mean_prob"] <= 1 and 1 <= got["mean_kept"] <= 10
