"""The 4-bit linears' and their expert layer's part of the C ABI: tests/c_abi/asan_fp4_check.c, built with the host code under
AddressSanitizer and UBSan (make, in __graft_entry__.build() too), pins their signatures, runs every argument check and
counts which calls allocate."""
import os
import subprocess

import pytest

from test_c_abi import ASAN_BIN, ASAN_ENV, _asan_binary

BIN = os.path.join(os.path.dirname(ASAN_BIN), "asan_fp4_check")


def run(*args):
    r = subprocess.run([BIN, *args], capture_output=True, text=True, timeout=120, env={**os.environ, **ASAN_ENV})
    assert r.returncode == 0, r.stdout + r.stderr
    return r.stdout


@pytest.mark.skipif(not os.path.exists("/opt/rocm/llvm/bin/clang"), reason="needs the ROCm clang")
def test_null_contexts_under_address_sanitizer():
    _asan_binary()
    assert "asan_fp4_check ok" in run()


@pytest.mark.gpu
def test_validation_under_address_sanitizer_on_device():
    """Every refusal on a real context, before any launch."""
    assert os.path.exists(BIN), "build tests/c_abi/_asan/asan_fp4_check first (__graft_entry__.build())"
    assert "asan_fp4_check ok (device validation)" in run("--device")
