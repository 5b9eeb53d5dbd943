"""The example of a layer of experts runs, and what it computes is its layer up to the roundings that it names."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.parametrize("weights", ["int8", "bf16"])
def test_experts_layer(weights):
    spec = importlib.util.spec_from_file_location("int8_experts", os.path.join(ROOT, "examples", "int8_experts.py"))
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    off = example.main(["--weights", weights, "--tokens", "1,33,300", "--hidden", "256", "--expert", "192", "--experts", "8", "--top", "3"])
    # A rounding to int8 moves a number by a step / 2 at most, / sqrt(12) of a step in the mean square; a step is 1 / 127 of its row's largest, which for 256 gaussian numbers is
    # under 5 deviations (h, a product: under 25 of its own): 5 / 127 / 3.46 = 0.0114 of a row's norm, 25 / 127 / 3.46 = 0.057. Six roundings reach y: x and the weight in gate
    # and up, h, and down's weight: 0.0114 * sqrt(5) + 0.057 < 0.09 (independent ones; h's dominates). bf16: 2^-8 at most each, of gate, up and down's weights, gate, up, h, y, and
    # torch's activation between: eight of them at most 8 * 2^-8 = 0.031.
    assert len(off) == 3 and all(o < (0.09 if weights == "int8" else 0.031) for o in off), off
