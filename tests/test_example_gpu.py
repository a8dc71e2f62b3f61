"""examples/speculative_decode.py: a layer's prompts in chunks, drafted trees and
accepted tokens, its last step against 64 bits."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_speculative_decode(lib, fmt):
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "speculative_decode.py")
    spec = importlib.util.spec_from_file_location("speculative_decode", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # the result's rounding to bf16, half a step of the largest value, and a weight's to fp16 on top
    assert example.main(fmt) <= 2.0 ** -8
