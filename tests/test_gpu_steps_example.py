"""The example that puts an MoE block together from the steps, and the steps' operators beside `experts` on the same block."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tokens,experts,top_k", [(100, 8, 2), (1, 4, 4), (700, 16, 4)])
def test_example_runs_and_its_gradients_are_those_of_the_block(tokens, experts, top_k):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "expert_steps.py")
    spec = importlib.util.spec_from_file_location("expert_steps", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    got = example.main(["--hidden", "256", "--experts", str(experts), "--top-k", str(top_k), "--tokens", str(tokens)])
    # An e4m3 rounding is off by at most 2^-4 of the value, 2^-4 / sqrt(3) = 0.036 in the 2-norm at worst; the output meets four (two products
    # of two operands), the gradient of the weights of the rows those, the others up to eight (the GLU's derivative at rounded values
    # counts as two, as both its factors change).  An integer is off by half a step of a / 127, and the largest of 256 normal
    # values is within 4.5 of their deviation, 4.5 / 254 / sqrt(3) = 0.011 in the 2-norm: four of them.
    assert got["serve"] < 4 * 0.011 + 0.01
    assert got["train"] < 4 * 0.036 and got["d_weights"] < 5 * 0.036
    for name in ("d_x", "d_gate_up", "d_down"):
        assert got[name] < 8 * 0.036, (name, got)
