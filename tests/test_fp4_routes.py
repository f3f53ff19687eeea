"""Where the expert layer for a few tokens (frx_fp4_moe_ffn) finds its routes: the rule (frx_policy.hpp), built with g++
for the CPU."""
import ctypes
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_one_token_routes_inside(tmp_path):
    so = tmp_path / "fp4_routes.so"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I",
           os.path.join(ROOT, "ferrisres_amd", "csrc"), os.path.join(ROOT, "tests", "c_abi", "fp4_routes.cpp"), "-o", str(so)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    h = ctypes.CDLL(str(so))
    assert [bool(h.fp4_routes_inside_of(T)) for T in range(1, 65)] == [True] + 63 * [False]
