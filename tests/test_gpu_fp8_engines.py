"""Every kernel of the 8-bit linears on shapes that reach it (_fp8_engines; test_fp8_plan holds them to the rules): long
enough that the stages of its pipeline are filled again, K ending in a part of a block, in one slice and in several. Against
the formula in 64 bits (on the GPU: the shapes are large), with the tolerance that test_gpu_fp8 derives."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp8_engines import DENSE, GROUPED
from _gpu import DEV
from test_gpu_fp8 import E4M3, E5M2, TOP, up

pytestmark = pytest.mark.gpu

PIPE = {True: frx.FP8_SUMS_PIPE, False: frx.FP8_SUMS_F32}


@pytest.fixture
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def operand(seed, rows, k, code, tiles=False):
    """Codes, scales and the values they stand for (f64), on the GPU."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = (torch.randn((rows, k), generator=g, device=DEV) * (TOP[code] / 6)).clamp(-TOP[code], TOP[code]).to(code)
    s = torch.exp(torch.randn((up(rows, 128) // 128 if tiles else rows, up(k, 128) // 128), generator=g, device=DEV))
    return q, s / TOP[code], value(q, s / TOP[code], tiles)


def value(q, s, tiles=False):
    spread = s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    if tiles:
        spread = spread.repeat_interleave(128, 0)[:q.shape[0]]
    return q.double() * spread


def check(y, ref, mag, k, cut):
    eps = torch.finfo(y.dtype).eps / 2
    off = ((128 + 1 + up(k, 128) // 128 + 16) * 2.0 ** -24 + (2.0 ** -10 if cut else 0.0)) * mag
    tol = off + eps * (ref.abs() + off)
    y = y.double()
    assert torch.isfinite(y).all()
    if cut:
        assert (y - ref).norm() <= 2.0 ** -8 * ref.norm()
    bad = (y - ref).abs() > tol * (1 + 1e-6)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((y - ref).abs() / tol.clamp_min(1e-300)).max()):.3g} x"


def outs(pipe8):
    return [torch.bfloat16] if pipe8 else [torch.float32, torch.bfloat16]


@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("name", list(DENSE))
def test_product(ctx, name, code):
    m, k, n, b_rows, pipe8 = DENSE[name][0]
    ctx.set_fp8_sums(PIPE[bool(pipe8)])
    a, sa, av = operand(m + k, m, k, code)
    b, sb, bv = operand(n + k, n, k, E4M3, tiles=b_rows == 128)
    ref, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    for out in outs(pipe8):
        y = torch.full((m, n), float("nan"), dtype=out, device=DEV)
        ctx.fp8_linear(a, sa, b, sb, y)
        check(y, ref, mag, k, cut=pipe8)
        for _ in range(2):  # slices are added in order: the same bits again
            again = torch.full((m, n), float("nan"), dtype=out, device=DEV)
            ctx.fp8_linear(a, sa, b, sb, again)
            assert torch.equal(y, again)


@pytest.mark.parametrize("name", list(DENSE))
def test_strides_and_an_unaligned_output(ctx, name):
    """NaN codes behind every row of both sides and an output from an odd element on: nothing past a row enters a
    sum, nothing beside the output is written, and the result is that of the dense call."""
    m, k, n, b_rows, pipe8 = DENSE[name][0]
    ctx.set_fp8_sums(PIPE[bool(pipe8)])
    a, sa, _ = operand(1, m, k, E4M3)
    b, sb, _ = operand(2, n, k, E4M3, tiles=b_rows == 128)

    def strided(q, extra):
        wide = torch.full((q.shape[0], k + extra), 0x7F, dtype=torch.uint8, device=DEV)
        wide[:, :k] = q.view(torch.uint8)
        return wide.view(q.dtype)[:, :k]
    for out in outs(pipe8):
        y = torch.full((m, n), float("nan"), dtype=out, device=DEV)
        ctx.fp8_linear(a, sa, b, sb, y)
        assert torch.isfinite(y).all()
        flat = torch.full((m * n + 2,), 7.0, dtype=out, device=DEV)
        z = flat[1:-1].view(m, n)
        ctx.fp8_linear(strided(a, 48), sa, strided(b, 16), sb, z)
        assert torch.equal(y, z) and flat[0] == 7.0 and flat[-1] == 7.0


@pytest.mark.parametrize("name", list(DENSE))
def test_nan_and_infinite_scales_keep_to_their_rows(ctx, name):
    """A NaN code in the last columns and in the first, a NaN scale and an infinite one reach their row (or column) of y
    and no other."""
    m, k, n, b_rows, pipe8 = DENSE[name][0]
    ctx.set_fp8_sums(PIPE[bool(pipe8)])
    a, sa, _ = operand(3, m, k, E4M3)
    b, sb, _ = operand(4, n, k, E4M3, tiles=b_rows == 128)
    for out in outs(pipe8):
        clean, y = (torch.full((m, n), 7.0, dtype=out, device=DEV) for _ in range(2))
        ctx.fp8_linear(a, sa, b, sb, clean)
        a2, sa2, b2 = a.clone(), sa.clone(), b.clone()
        rows, cols = sorted({0, m // 2, m - 1}), [11, n - 1]
        a2.view(torch.uint8)[rows[0], k - 1] = 0x7F
        if len(rows) > 1:
            sa2[rows[1], -1] = float("nan")
        if len(rows) > 2:
            sa2[rows[2], 0] = float("inf")
        b2.view(torch.uint8)[cols[0], k - 2] = 0xFF
        b2.view(torch.uint8)[cols[1], 5] = 0x7F
        ctx.fp8_linear(a2, sa2, b2, sb, y)
        keep_r = torch.ones(m, dtype=torch.bool, device=DEV)
        keep_c = torch.ones(n, dtype=torch.bool, device=DEV)
        keep_r[rows], keep_c[cols] = False, False
        assert torch.isnan(y[rows[:2]]).all() and not torch.isfinite(y[rows]).any()
        assert torch.isnan(y[:, cols]).all()
        assert torch.equal(y[keep_r][:, keep_c], clean[keep_r][:, keep_c])


@pytest.mark.parametrize("name", [n for n in DENSE if DENSE[n][0][3] == 128])
def test_activations_quantised_inside_are_the_two_calls(ctx, name):
    m, k, n, _, pipe8 = DENSE[name][0]
    ctx.set_fp8_sums(PIPE[bool(pipe8)])
    g = torch.Generator(device=DEV).manual_seed(m)
    x = torch.randn((m, k), generator=g, device=DEV).bfloat16()
    b, sb, bv = operand(2, n, k, E4M3, tiles=True)
    q, s = torch.empty((m, k), dtype=E4M3, device=DEV), torch.empty((m, up(k, 128) // 128), device=DEV)
    ctx.fp8_quantize(x, frx.FP8_ROWS, q, s)
    av = value(q, s)
    ref, mag = av @ bv.t(), av.abs() @ bv.abs().t()
    for out in outs(pipe8):
        y, z = (torch.full((m, n), float("nan"), dtype=out, device=DEV) for _ in range(2))
        ctx.fp8_linear(q, s, b, sb, y)
        ctx.fp8_linear_act(x, b, sb, z)
        assert torch.equal(y, z)
        check(z, ref, mag, k, cut=pipe8)


@pytest.mark.parametrize("name,code", [(n, c) for n in GROUPED for c in (E4M3, E5M2)
                                       if not (GROUPED[n][0][4] and c is E5M2)])  # e5m2 rows: never the 8-bit pipe
def test_experts_rows(ctx, name, code):
    """Every expert's rows times its own weights; a row of NaN, and NaN rows behind the last expert, reach no other."""
    sizes, behind, k, n, pipe8 = GROUPED[name][0]
    ctx.set_fp8_sums(PIPE[bool(pipe8)])
    E, off = len(sizes), np.concatenate([[0], np.cumsum(sizes)])
    rows, last = int(off[-1]) + behind, int(off[-1])
    a, sa, av = operand(5, rows, k, code)
    a.view(torch.uint8)[last:] = 0x7F
    ops = [operand(7 + e, n, k, E4M3, tiles=True) for e in range(E)]
    b, sb = [o[0] for o in ops], [o[1] for o in ops]
    offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
    sick = last - 1
    for out in outs(pipe8):
        y = torch.full((rows, n), 5.0, dtype=out, device=DEV)
        ctx.fp8_linear_grouped(a, sa, b, sb, offsets, y)
        for e in range(E):
            i, j = int(off[e]), int(off[e + 1])
            if j > i:
                check(y[i:j], av[i:j] @ ops[e][2].t(), av[i:j].abs() @ ops[e][2].abs().t(), k, cut=pipe8)
        assert (y[last:] == 5.0).all()
        a2 = a.clone()
        a2.view(torch.uint8)[sick, k - 1] = 0x7F
        z = torch.full((rows, n), 5.0, dtype=out, device=DEV)
        ctx.fp8_linear_grouped(a2, sa, torch.stack([t.view(torch.uint8) for t in b]).view(E4M3), torch.stack(sb), offsets, z)
        assert torch.isnan(z[sick]).all()
        z[sick] = y[sick]
        assert torch.equal(y, z)


@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("pipe8", [False, True])
def test_experts_weight_gradients(ctx, code, pipe8):
    """Sums over 640 to 1280 rows of an expert, room for rows that is no multiple of 128; NaN codes and scales behind the
    last expert reach none."""
    ctx.set_fp8_sums(PIPE[pipe8])
    n, k, off, rows = 390, 260, [0, 640, 640, 1920, 2816], 2816 + 80
    a, sa, av = operand(1, n, rows, code)
    b, sb, bv = operand(2, k, rows, E4M3)
    for t in (a, b):
        t.view(torch.uint8)[:, off[-1]:] = 0x7F
    for s in (sa, sb):
        s[:, off[-1] // 128:] = float("nan")
    offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
    for out in outs(pipe8):
        dw = torch.full((4, n, k), float("nan"), dtype=out, device=DEV)
        ctx.fp8_grad_weight_grouped(a, sa, b, sb, offsets, dw)
        for e in range(4):
            i, j = off[e], off[e + 1]
            check(dw[e], av[:, i:j] @ bv[:, i:j].t(), av[:, i:j].abs() @ bv[:, i:j].abs().t(), j - i,
                  cut=pipe8 and j > i)
        again = torch.full_like(dw, float("nan"))
        ctx.fp8_grad_weight_grouped(a, sa, b, sb, offsets, again)
        assert torch.equal(dw, again)
