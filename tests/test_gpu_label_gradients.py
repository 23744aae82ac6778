"""GPU: the logits' gradient where the probabilities themselves are next to nothing, against float64 with the bounds of
test_gpu_label_probs.py, whose logits lie closer together."""
import pytest
import torch

from test_gpu_label_probs import TYPES, check, data

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,O", [(1, 7102), (20, 5230), (260, 5001), (3, 14)])
@pytest.mark.parametrize("dt", TYPES)
@pytest.mark.parametrize("spread", [10.0, 20.0, 40.0])
def test_logits_far_below_the_largest(dev, B, O, dt, spread):
    """Probabilities around and under 2^-126 times factors of some hundreds: values that bf16 and fp32 still have."""
    for seed in range(3):
        z, labels, dlp, dent = data(B, O, 5, dt, dev, seed=seed + O, pitch=3, spread=spread)
        check(z, labels, 0, dlp, dent)
        check(z, labels, 3, None, dent * 100)
        check(z, labels, 0, dlp * 1e-3, None)
