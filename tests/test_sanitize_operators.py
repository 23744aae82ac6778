"""The host code of the encoder's operators (layer norm, gradient norm, AdamW) under
AddressSanitizer and UndefinedBehaviorSanitizer, CPU only: `make -C haste_amd
sanitize_operators` drives their argument checks and workspace sizing
(tests/native/host_check_operators.cpp)."""
import os

import pytest

from test_sanitize import _run


def test_operators_host_code_under_asan_ubsan():
    if not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc not found")
    _run(["make", "-s", "-j8", "-C", "haste_amd", "sanitize_operators"], "host_check_operators OK", 1200)
