"""The kernel rules of the 4-bit linears and of the expert layer for a few tokens (frx_policy.hpp), built with g++ for the
CPU: every kernel has a shape of _fp4_kernels that reaches it, so that a rule that moves takes no kernel out of the GPU tests
unseen; and what holds of the rules over many shapes."""
import ctypes
import os
import random
import shutil
import subprocess

import pytest

from _fp4_kernels import (DOWN, FEW, GATE_UP, GRADS, GROUPED, KS, LAYERS, ROWS16, ROWS16_K, SPLIT, T128X192, T128X256, T192X256,
                          T256, T64, T64X128, TILES)

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CUS = 256

pytestmark = pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    so = tmp_path_factory.mktemp("fp4") / "fp4_plan.so"
    cmd = ["g++", "-std=c++17", "-O1", "-Wall", "-Wextra", "-Werror", "-shared", "-fPIC", "-I",
           os.path.join(ROOT, "ferrisres_amd", "csrc"), os.path.join(ROOT, "tests", "c_abi", "fp4_plan.cpp"), "-o", str(so)]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    h, out = ctypes.CDLL(str(so)), (ctypes.c_int * 4)()
    h.fp4_plan_of.argtypes = [ctypes.c_uint32] * 3 + [ctypes.c_int, ctypes.c_void_p]
    h.fp4_grouped_tile_of.argtypes = [ctypes.c_uint32] * 4 + [ctypes.c_int]
    h.fp4_grad_tile_of.argtypes = [ctypes.c_uint32] * 4 + [ctypes.c_int]
    h.fp4_few_of.argtypes = [ctypes.c_uint32] * 4 + [ctypes.c_int] * 2 + [ctypes.c_void_p]

    class Rules:
        @staticmethod
        def plan(M, K, N, cus=CUS):
            h.fp4_plan_of(M, K, N, cus, out)
            return tuple(out)[:3]

        @staticmethod
        def grouped(R, K, N, E, cus=CUS):
            return h.fp4_grouped_tile_of(R, K, N, E, cus)

        @staticmethod
        def grad(R, N, K, E, cus=CUS):
            return h.fp4_grad_tile_of(R, N, K, E, cus)

        @staticmethod
        def few(T, K, E, top_k, planes, down):
            h.fp4_few_of(T, K, E, top_k, planes, down, out)
            return tuple(out)
    return Rules


def test_every_tile_has_its_shapes(rules):
    for tile, (M, N) in TILES.items():
        for K in KS:
            assert rules.plan(M, K, N) == (tile, 1, -(-K // 256)), (tile, K)
    for M, K, N, tile in SPLIT:
        t, S, per = rules.plan(M, K, N)
        assert t == tile and S > 1 and K % 256 != 0
    assert set(TILES) == set(range(T64, T256 + 1))
    for (M, N), rt in ROWS16.items():
        for K in ROWS16_K:
            assert rules.plan(M, K, N) == (FEW, 1, rt)
    assert {rt for (M, _), rt in ROWS16.items() if M <= 16} == {1, 2, 3, 4}
    assert {rt for (M, _), rt in ROWS16.items() if M > 16} == {1, 2, 3, 4}


def test_every_grouped_tile_has_its_shape(rules):
    for sizes, behind, K, N, tile in GROUPED.values():
        assert rules.grouped(sum(sizes) + behind, K, N, len(sizes)) == tile
    assert {c[4] for c in GROUPED.values()} == {T64, T64X128, T128X256, T256}


def test_every_gradient_tile_has_its_shape(rules):
    for sizes, behind, N, K, tile in GRADS.values():
        assert rules.grad(sum(sizes) + behind, N, K, len(sizes)) == tile
    assert {c[4] for c in GRADS.values()} == {T64X128, T128X256, T256}


@pytest.mark.parametrize("planes", [1, 3])
def test_every_gate_up_kernel_has_a_layer(rules, planes):
    got = {(s, t, slices > 1) for s, t, slices, _ in (rules.few(T, H, E, k, planes, 0) for T, H, _, E, k in LAYERS)}
    assert got == (GATE_UP if planes == 1 else GATE_UP - {(4, 2, False)})


@pytest.mark.parametrize("planes", [2, 3])
def test_every_down_kernel_has_a_layer(rules, planes):
    got = {rules.few(T, i, E, k, planes, 1)[:2] for T, _, i, E, k in LAYERS}
    assert got == DOWN


def test_rules_over_many_shapes(rules):
    """Any shape: slices that cover K and none of them empty, no more than 8, from an even step on; a grouped tile that
    there is; the few tokens' slices cover K, and their steps what a wave holds."""
    rng = random.Random(5)
    log = lambda a, b: int(a * (b / a) ** rng.random())  # noqa: E731
    for _ in range(20000):
        M, K, N, cus = log(1, 1 << 20), log(1, 1 << 15) * 32, log(1, 1 << 20), rng.choice((64, 228, 256, 304))
        tile, S, per = rules.plan(M, K, N, cus)
        steps = -(-K // 256)
        if M <= 32:
            assert tile == FEW and S == 1 and 1 <= per <= 4
            continue
        assert T64 <= tile <= T256
        assert 1 <= S <= 8 and (S - 1) * per < steps <= S * per
        assert S == 1 or per % 2 == 0
    # what frx_fp4_linear accepts fits a launch, or (experts' rows, whose workgroups take tiles in turn) a count in 32 bits
    sides = {T64: (64, 64, 256), T64X128: (64, 128, 256), T128X192: (128, 192, 512), T128X256: (128, 256, 512),
             T192X256: (192, 256, 512), T256: (256, 256, 512)}
    for _ in range(20000):
        M, N, K, E = log(33, 1 << 31), log(1, (1 << 27) - 16), log(1, 1 << 18) * 32, rng.randint(1, 64)
        if (-(-M // 64) + 64) * -(-N // 128) >= 1 << 24:
            continue
        h, w, threads = sides[rules.plan(M, K, N)[0]]
        assert -(-M // h) * -(-N // w) * threads < 1 << 32
        tile = rules.grouped(M, K, N, E)
        h, w, threads = sides[tile]
        assert (-(-M // h) + E) * -(-N // w) * (threads if tile == T256 else 1) <= 0xF0000000
        h, w, threads = sides[rules.grad(K, M, N, E)]
        assert -(-M // h) * -(-N // w) * threads < 1 << 32
    for _ in range(5000):
        assert rules.grouped(log(1, 1 << 20), log(1, 4096) * 32, log(1, 1 << 16), rng.randint(1, 64)) in (
            T64, T64X128, T128X256, T256)
        T, K, E = rng.randint(1, 64), log(1, 1 << 14) * 32, rng.randint(1, 64)
        top_k, planes, kbs = rng.randint(1, 64), rng.choice((1, 2, 3)), -(-K // 128)
        for down in (0, 1):
            steps, tiles, slices, per = rules.few(T, K, E, top_k, planes, down)
            assert 2 <= steps <= 4 and 1 <= tiles <= 3
            assert (slices - 1) * per < kbs <= slices * per and per <= 8 * steps
