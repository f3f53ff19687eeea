"""The kernel rules of the 8-bit linears (frx_policy.hpp), built with g++ for the CPU: every kernel has a shape of
_fp8_engines that reaches it, so that a rule that moves takes no kernel out of the GPU tests unseen; and what holds of the
rules over many shapes."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

from _fp8_engines import DENSE, FEW, GROUPED, RING128, RING192, RING256, T64, T128

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = tmp_path_factory.mktemp("fp8") / "fp8_plan.so"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I",
           os.path.join(ROOT, "ferrisres_amd", "csrc"), os.path.join(ROOT, "tests", "c_abi", "fp8_plan.cpp"), "-o", str(so)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    h, out = ctypes.CDLL(str(so)), (ctypes.c_int * 3)()
    h.fp8_plan_of.argtypes = [ctypes.c_uint32] * 3 + [ctypes.c_int] * 3 + [ctypes.c_void_p]
    h.fp8_grouped_tile_of.argtypes = [ctypes.c_uint32] * 3 + [ctypes.c_int] * 2

    def plan(M, K, N, b_rows, pipe8, cus=CUS):
        h.fp8_plan_of(M, K, N, b_rows, pipe8, cus, out)
        return tuple(out)
    return plan, lambda R, N, E, pipe8, cus=CUS: h.fp8_grouped_tile_of(R, N, E, pipe8, cus)


@pytest.mark.parametrize("name", list(DENSE))
def test_shapes_reach_their_kernels(rules, name):
    (M, K, N, b_rows, pipe8), tile, split, row_tiles = DENSE[name]
    got, S, per = rules[0](M, K, N, b_rows, pipe8)
    steps = -(-K // 128)
    assert got == tile
    if tile == FEW:
        assert (S, per) == (1, row_tiles)
        return
    assert (S > 1) == split and K % 128 != 0
    assert (S - 1) * per < steps <= S * per
    # stages are filled again in every slice but the last; a wide 128 x 128 tile takes K in short slices only
    assert per >= 5 or name == "128-split"


@pytest.mark.parametrize("name", list(GROUPED))
def test_grouped_shapes_reach_their_kernels(rules, name):
    (sizes, behind, K, N, pipe8), tile = GROUPED[name]
    assert rules[1](sum(sizes) + behind, N, len(sizes), pipe8) == tile


def test_every_kernel_has_a_shape():
    """The instances that frx_fp8.hip launches: tile, 8-bit pipe, a scale per weight row."""
    have = {(tile, pipe8, b_rows == 1) for (_, _, _, b_rows, pipe8), tile, _, _ in DENSE.values() if tile != FEW}
    wide = {(RING128, 0, False), (RING192, 0, False), (T128, 0, False), (T128, 0, True)}
    pipe = {(RING128, 1, False), (RING192, 1, False), (RING256, 1, False), (T128, 1, False), (RING128, 1, True),
            (T128, 1, True)}
    assert have == wide | pipe
    split = {(tile, pipe8, b_rows == 1) for (_, _, _, b_rows, pipe8), tile, s, _ in DENSE.values() if s}
    assert split == have
    few = {(min(64, -(-M // 16) * 16) if M <= 64 else 64, rt) for (M, _, _, _, _), tile, _, rt in DENSE.values() if tile == FEW}
    assert {(16, rt) for rt in (1, 2, 3, 4)} <= few and {(32, rt) for rt in (1, 2, 3, 4)} <= few
    assert {(64, rt) for rt in (1, 2)} <= {(64 if m > 32 else m, rt) for m, rt in few}
    assert {t for _, t in GROUPED.values()} == {FEW, T64, RING128, RING256}


def test_rules_over_many_shapes(rules):
    """Any shape: a kernel that there is for its pipe and scales, slices that cover K and none of them empty, no more
    than 8; the sums of an f32 and a bf16 output go alike (the rules do not see the type)."""
    rng = random.Random(5)
    log = lambda a, b: int(a * (b / a) ** rng.random())  # noqa: E731
    for _ in range(20000):
        M, K, N = log(1, 1 << 17), log(1, 1 << 11) * 16, log(1, 1 << 17)
        b_rows, pipe8, cus = rng.choice((1, 128)), rng.choice((0, 1)), rng.choice((64, 228, 256, 304))
        tile, S, per = rules[0](M, K, N, b_rows, pipe8, cus)
        steps = -(-K // 128)
        if tile == FEW:
            assert S == 1 and 1 <= per <= (4 if M <= 32 else 2)
            continue
        allowed = {(0, 128): {RING128, RING192, T128}, (0, 1): {T128}, (1, 128): {RING128, RING192, RING256, T128},
                   (1, 1): {RING128, T128}}[pipe8, b_rows]
        assert M > 32 and tile in allowed
        assert 1 <= S <= 8 and (S - 1) * per < steps <= S * per
    for _ in range(5000):
        R, N, E = log(1, 1 << 20), log(1, 1 << 15), rng.randint(1, 64)
        tile = rules[1](R, N, E, rng.choice((0, 1)), 256)
        assert tile in ({FEW} if R <= 8 * E and N < 1 << 15 else {T64, RING128, RING256})
    assert rules[1](1 << 20, 4096, 4, 0, 256) == T64
