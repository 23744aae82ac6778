"""GPU: the gated block at sizes that reach the forms of its products which test_gpu_gated_mlp.py does not: its
tolerances are derived there.  Which form a product takes (gated_mlp.hip: cut_of) depends on rows, columns and K:

  a  16-bit h and dg/du on 256 x 128 in three stages (many rows, K up to 1024), weights' gradients in parts on
     256 x 256; fp32 h, dg/du, dx and y on 256 x 256
  b  128 x 128 for y, dg/du and dx whole, for the weights' gradients in parts; fp32 weights' gradients in many parts
  c  16-bit h and dg/du on 256 x 128 of odd rows, dx in parts on 256 x 256, y in parts on 128 x 128
  d  dWd on 128 x 128 whole, y in parts on 256 x 256
  e  fp32 dWg/dWu on 256 x 256 whole, y in parts on 128 x 128
  f  dWd on 256 x 256 whole
  g  h on 128 x 128"""
import pytest
import torch

from test_gpu_gated_mlp import ACTS, TYPES, check, data, run

pytestmark = pytest.mark.gpu
SIZES = {"a": (32771, 264, 1032, 264), "a odd": (32771, 261, 1037, 259), "b": (20000, 136, 264, 136),
         "c": (7046, 11, 4018, 9), "d": (2983, 82, 4162, 790), "e": (86, 1830, 2827, 782),
         "f": (573, 816, 3968, 2094), "g": (33327, 100, 8, 202), "ragged": (4001, 301, 1003, 301)}


@pytest.mark.parametrize("name", list(SIZES))
@pytest.mark.parametrize("dt", TYPES)
def test_every_form(dev, name, dt):
    check(data(*SIZES[name], dt, dev, seed=3), ACTS[len(name) % 3])


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dt", TYPES)
def test_activations_on_large_tiles(dev, name, dt):
    """Gates from far below zero to far above it, with the epilogues of 256 x 128 (fp32: 256 x 256)."""
    d = data(33000, 64, 520, 72, dt, dev)
    d["wg"] *= 4.0
    check(d, name)


@pytest.mark.parametrize("name", ["a", "a odd", "c", "d"])
@pytest.mark.parametrize("dt", TYPES)
def test_two_runs_give_the_same_bits(dev, name, dt):
    d = data(*SIZES[name], dt, dev, seed=5)
    first = run(d)
    for _ in range(2):
        again = run(d)
        assert all(torch.equal(first[k], again[k]) for k in first)
