"""The host code of the embedding, the gated block and the label log probabilities under
AddressSanitizer and UndefinedBehaviorSanitizer, CPU only: `make -C haste_amd sanitize_encoder`
drives their argument checks and workspace sizing (tests/native/host_check_encoder.cpp)."""
import os

import pytest

from test_sanitize import _run


def test_encoder_host_code_under_asan_ubsan():
    if not os.path.exists("/opt/rocm/bin/hipcc"):
        pytest.skip("hipcc not found")
    _run(["make", "-s", "-j8", "-C", "haste_amd", "sanitize_encoder"], "host_check_encoder OK", 1800)
