"""MI355X: the example that runs the packed Linears, the append to the 4-bit
cache and the attention over it together (examples/attention_block.py)."""

import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "attention_block.py")


def test_the_attention_block(capsys):
    spec = importlib.util.spec_from_file_location("attention_block", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    # two roundings to bf16 (weights, result), 2^-8 at most of a value each, and far less on the whole
    assert example.main(steps=35) < 2.0 ** -7
    assert "verify: (12, 2048), [239, 72, 40] tokens held" in capsys.readouterr().out
