"""examples/sequence_head.py on the GPU: the head learns through the operators' gradients, rows
served as a prompt and single tokens equal whole rows, and the 8-bit norm stands for its values."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "sequence_head.py")


def test_sequence_head():
    spec = importlib.util.spec_from_file_location("sequence_head", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    r = example.main(rows=64, steps=40)
    assert r["losses"][-1] < 0.5 * r["losses"][0]
    assert r["hit"] > 0.8
    # 24 tokens of 32-bit arithmetic, twice: rounding of at most 24 * (12 + 12 * 16) ulp
    assert r["served"] <= 24 * (12 + 12 * 16) * 2.0 ** -24 * max(1.0, r["largest"])
    # half a step of 3 mantissa bits, of the group's largest value
    assert r["in_8_bits"] <= 2.0 ** -4 * (1 + 1e-3)
