"""CPU: calls of the gated block's C entry points that start no kernel and say so."""
import os
import subprocess

import pytest

from haste_amd import _lib

BF16, F16, F32 = _lib.DTYPE_BF16, _lib.DTYPE_F16, _lib.DTYPE_F32


@pytest.mark.parametrize("dt", [BF16, F16, F32])
@pytest.mark.parametrize("D,H,O", [(8, 16, 8), (7, 13, 5), (64, 1003, 301)])
def test_backward_of_no_rows_takes_no_weights(dt, D, H, O):
    """With no rows neither the weights nor a workspace are looked at: none of these addresses is one.  (A kernel that
    copied the weights would fail to launch here, where there is no GPU.)"""
    L = _lib.lib()
    for aligned in (0, 1):
        assert L.haste_gated_mlp_workspace_size(0, D, H, O, dt, 1, aligned) == 0
    for weight in (None, 66):
        assert L.haste_gated_mlp_bwd(None, D, weight, D, weight, D, weight, H, None, O, None, None, None, None,
                                     None, None, 0, D, H, O, dt, None, 0, None) == _lib.HASTE_OK, _lib.last_error()


def test_how_copies_are_cut_into_launches(tmp_path):
    """The arithmetic, on the CPU: tests/native/launches_check.cpp."""
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "launches_check")
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", os.path.join(here, "native", "launches_check.cpp"),
                    "-o", exe], check=True, timeout=120)
    out = subprocess.run([exe], check=True, capture_output=True, text=True, timeout=60).stdout
    assert "launches_check OK" in out
