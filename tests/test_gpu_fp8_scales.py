"""Scales of very small and very large blocks in the 8-bit linears: a block's two scales may have a product outside the
f32 numbers, or so small that f32 keeps few of its bits, while the outputs are ordinary numbers. The formula in 64 bits and
the tolerance of test_gpu_fp8 hold there too. Among numbers below 2^-126 a rounding is off by half a step of the denormals
whatever the number, 2^-150 in f32 and 2^-134 in bf16: one for each block and each of up to 8 slices of K in the sum, one for
the output."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _gpu import DEV
from test_gpu_fp8 import E4M3, E5M2, check, gen, operand, up

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def check_small(y, ref, mag, k):
    blocks = up(k, 128) // 128
    off = (128 + 1 + blocks + 16) * 2.0 ** -24 * mag + (blocks + 8) * 2.0 ** -150
    tol = off + torch.finfo(y.dtype).eps / 2 * (ref.abs() + off) + (2.0 ** -134 if y.dtype == torch.bfloat16 else 2.0 ** -150)
    y = y.cpu().double()
    assert torch.isfinite(y).all()
    bad = (y - ref).abs() > tol * (1 + 1e-6)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {float(((y - ref).abs() / tol).max()):.3g} x"


def scaled(op, exponents, tiles=False):
    """The operand with every block's scale times 2^e of its own."""
    q, s, v = op
    s = s * torch.exp2(exponents.float())
    spread = s.double().repeat_interleave(128, 1)[:, :q.shape[1]]
    if tiles:
        spread = spread.repeat_interleave(128, 0)[:q.shape[0]]
    return q, s, q.double() * spread


def exponents(seed, shape, low, high):
    return torch.randint(low, high + 1, shape, generator=gen(seed))


# a few tokens (one, three and four row tiles a workgroup), groups of 64, K in slices, tiles of every height
SHAPES = [(1, 400, 300), (3, 272, 11000), (16, 272, 15001), (40, 272, 260), (300, 4112, 1100), (1600, 528, 3300),
          (2000, 656, 6000), (4100, 528, 5000)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("code,b_rows", [(E5M2, 128), (E4M3, 128), (E5M2, 1)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_products_of_scales_below_f32(ctx, m, k, n, code, b_rows, out):
    """Gradients of 1e-28 to 1e-34 against ordinary weights: products of scales from 2^-120 to below the smallest
    denormal, outputs that are normal numbers."""
    a = operand(m + k, m, k, code)
    a = scaled(a, exponents(1, a[1].shape, -96, -89))
    b = operand(n + k, n, k, E4M3, tiles=b_rows == 128)
    b = scaled(b, exponents(2, b[1].shape, -30, -12), tiles=b_rows == 128)
    assert (a[1] >= 2.0 ** -126).all() and (b[1] >= 2.0 ** -126).all()
    assert float(a[1].double().min() * b[1].double().min()) < 2.0 ** -135
    y = torch.full((m, n), float("nan"), dtype=out, device=DEV)
    ctx.fp8_linear(a[0].to(DEV), a[1].to(DEV), b[0].to(DEV), b[1].to(DEV), y)
    check_small(y, a[2] @ b[2].t(), a[2].abs() @ b[2].abs().t(), k)


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("tiles", [True, False])
def test_scales_far_apart_in_one_tile(ctx, m, k, n, tiles):
    """Large scales beside small ones, token by token and block by block: every product of the two is an ordinary
    number or far below one, and neither kind disturbs the other."""
    a, b = operand(m + k, m, k, E4M3), operand(n + k, n, k, E4M3, tiles=tiles)
    kb = up(k, 128) // 128
    sign = torch.where(torch.arange(kb) % 2 == 0, 1, -1)
    a = scaled(a, (70 * sign)[None, :] + exponents(3, a[1].shape, -20, 20))
    b = scaled(b, (-70 * sign)[None, :] + exponents(4, b[1].shape, -20, 20), tiles=tiles)
    ref, mag = a[2] @ b[2].t(), a[2].abs() @ b[2].abs().t()
    y = torch.full((m, n), float("nan"), device=DEV)
    ctx.fp8_linear(a[0].to(DEV), a[1].to(DEV), b[0].to(DEV), b[1].to(DEV), y)
    check(y, ref, mag, k)


@pytest.mark.parametrize("m", [1, 40, 700])
def test_scales_of_zero(ctx, m):
    """A scale of 0 on either side, beside the largest one on the other: the block adds nothing."""
    k, n = 656, 515
    a, b = operand(1, m, k, E4M3), operand(2, n, k, E4M3, tiles=True)
    ea, eb = torch.zeros(a[1].shape), torch.zeros(b[1].shape)
    a, b = list(scaled(a, ea)), list(scaled(b, eb, tiles=True))
    a[1][:, 0], b[1][:, 0] = 0.0, 2.0 ** 119
    a[1][:, 3], b[1][:, 3] = 2.0 ** 119, 0.0
    keep = torch.ones(k, dtype=torch.bool)
    keep[:128] = False
    keep[384:512] = False
    ref, mag = a[2][:, keep] @ b[2][:, keep].t(), a[2][:, keep].abs() @ b[2][:, keep].abs().t()
    y = torch.full((m, n), float("nan"), device=DEV)
    ctx.fp8_linear(a[0].to(DEV), a[1].to(DEV), b[0].to(DEV), b[1].to(DEV), y)
    check(y, ref, mag, k)


@pytest.mark.parametrize("sizes", [[1, 0, 3], [60, 5, 80], [300, 260]])
def test_experts_rows_of_small_scales(ctx, sizes):
    k, n = 528, 515
    off = np.concatenate([[0], np.cumsum(sizes)])
    rows = int(off[-1])
    a = operand(3, rows, k, E5M2)
    a = scaled(a, exponents(1, a[1].shape, -96, -89))
    ops = [operand(7 + e, n, k, E4M3, tiles=True) for e in range(len(sizes))]
    ops = [scaled(o, exponents(9, o[1].shape, -30, -12), tiles=True) for o in ops]
    y = torch.full((rows, n), float("nan"), device=DEV)
    ctx.fp8_linear_grouped(a[0].to(DEV), a[1].to(DEV), [o[0].to(DEV) for o in ops], [o[1].to(DEV) for o in ops],
                           torch.tensor(off, dtype=torch.int32, device=DEV), y)
    for e in range(len(sizes)):
        i, j = int(off[e]), int(off[e + 1])
        if j > i:
            check_small(y[i:j], a[2][i:j] @ ops[e][2].t(), a[2][i:j].abs() @ ops[e][2].abs().t(), k)


def test_experts_gradients_of_small_scales(ctx):
    n, k, rows = 130, 260, 768
    a = operand(1, n, rows, E5M2)
    a = scaled(a, exponents(1, a[1].shape, -96, -89))
    b = operand(2, k, rows, E4M3)
    b = scaled(b, exponents(2, b[1].shape, -30, -12))
    dw = torch.full((2, n, k), float("nan"), device=DEV)
    ctx.fp8_grad_weight_grouped(a[0].to(DEV), a[1].to(DEV), b[0].to(DEV), b[1].to(DEV),
                                torch.tensor([0, 640, 768], dtype=torch.int32, device=DEV), dw)
    for e, (i, j) in enumerate(((0, 640), (640, 768))):
        check_small(dw[e], a[2][:, i:j] @ b[2][:, i:j].t(), a[2][:, i:j].abs() @ b[2][:, i:j].abs().t(), j - i)


@pytest.mark.parametrize("size", [1e-28, 1e-30, 1e-32])
def test_small_gradients_end_to_end(ctx, size):
    """dx of gradients of this size, quantised here, against the values that the codes stand for."""
    m, n, k = 70, 384, 272
    dy = torch.randn((m, n), generator=gen(5)) * size
    w = 0.02 * torch.randn((n, k), generator=gen(6))
    new = lambda r, c, code, sr: (torch.empty((r, up(c, 16)), dtype=code, device=DEV),  # noqa: E731
                                  torch.empty((sr, up(c, 128) // 128), device=DEV))
    wq, ws = ctx.fp8_quantize(w.to(DEV), frx.FP8_TILES_T, *new(k, n, E4M3, up(k, 128) // 128))
    q, s = ctx.fp8_quantize(dy.to(DEV), frx.FP8_ROWS, *new(m, n, E5M2, m))
    y = torch.empty((m, k), device=DEV)
    ctx.fp8_linear(q, s, wq, ws, y)
    av = q.cpu().double() * s.cpu().double().repeat_interleave(128, 1)[:, :n]
    bv = wq.cpu().double() * ws.cpu().double().repeat_interleave(128, 1).repeat_interleave(128, 0)[:k, :wq.shape[1]]
    check_small(y, av @ bv[:, :n].t(), av.abs() @ bv[:, :n].abs().t(), n)


@pytest.mark.parametrize("n", [16, 4112])  # groups of 64 tokens; tiles
@pytest.mark.parametrize("code", [E4M3, E5M2])
@pytest.mark.parametrize("b_rows", [128, 1])
@pytest.mark.parametrize("sa,sb", [(1.0, 1.0), (2.0 ** -100, 2.0 ** -10), (2.0 ** -90, 2.0 ** -20), (2.0 ** 100, 2.0 ** -110),
                                   (2.0 ** -30, 2.0 ** -71)])
def test_every_code_exactly(ctx, n, code, b_rows, sa, sb):
    """One code a token, against ones: y is the code's value times the scales, exactly, whatever side of a line they
    lie on; a NaN stays one and an infinity too."""
    k = 144
    a = torch.zeros((256, k), dtype=torch.uint8)
    a[:, 130] = torch.arange(256)  # in the part of a block at the end
    b = torch.zeros((n, k), dtype=torch.uint8)
    b[:, 130] = torch.ones(1).to(E4M3).view(torch.uint8)
    y = torch.full((256, n), 5.0, device=DEV)
    ctx.fp8_linear(a.to(DEV).view(code), torch.full((256, 2), sa, device=DEV), b.to(DEV).view(E4M3),
                   torch.full((n if b_rows == 1 else up(n, 128) // 128, 2), sb, device=DEV), y)
    want = torch.arange(256, dtype=torch.uint8).view(code).double() * sa * sb
    y = y.cpu().double()
    assert torch.equal(torch.isnan(y), torch.isnan(want)[:, None].expand(256, n))
    keep = ~torch.isnan(want)
    assert torch.equal(y[keep], want[keep][:, None].expand(int(keep.sum()), n))
