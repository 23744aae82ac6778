"""GPU: the example that trains an encoder (LayerNorm, AdamW, grad_norm) with its fixed-fan-in
output layer learns, with 8-bit states as with 32-bit ones."""
import importlib.util
import os

import pytest

pytestmark = pytest.mark.gpu
PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples",
                    "train_encoder.py")


def test_example_learns(dev):
    spec = importlib.util.spec_from_file_location("train_encoder", PATH)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    eight, full = (example.train(steps=300, state_bits=b) for b in (8, 32))
    # the first steps learn how rare labels are, the later ones which are right
    assert eight[-1] < 0.85 * eight[5] and full[-1] < 0.85 * full[5]
    assert abs(eight[-1] - full[-1]) < 0.1 * full[-1]
