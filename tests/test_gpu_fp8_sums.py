"""How the 8-bit linears add up (frx_set_fp8_sums). By default every sum is one of exact products in fp32, so that a bf16
output is the f32 output rounded once, bit for bit: the two run the same kernels over the same slices of K. Under
FP8_SUMS_PIPE bf16 outputs may come off the 8-bit pipe, within the tolerance that test_gpu_fp8 derives for its cuts."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _gpu import DEV
from test_gpu_fp8 import E4M3, E5M2, check, operand, values

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def both(call, shape):
    """The f32 and the bf16 result of a call that takes its output."""
    ys = [torch.full(shape, float("nan"), dtype=t, device=DEV) for t in (torch.float32, torch.bfloat16)]
    for y in ys:
        call(y)
    return ys


# a few tokens, groups of 64, K in slices (one of them ending in half a block), one slice, tiles of every height
SHAPES = [(1, 2064, 300), (40, 272, 260), (200, 400, 1000), (64, 5648, 640), (300, 4112, 1100), (700, 1040, 2100),
          (1600, 528, 3300), (2000, 656, 6000), (4100, 528, 5000)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("code,b_rows", [(E4M3, 128), (E5M2, 128), (E4M3, 1), (E5M2, 1)])
def test_bf16_is_the_f32_sum_rounded(ctx, m, k, n, code, b_rows):
    a, sa, _ = operand(m + k, m, k, code)
    b, sb, _ = operand(n + k, n, k, E4M3, tiles=b_rows == 128)
    a, sa, b, sb = (t.to(DEV) for t in (a, sa, b, sb))
    f, h = both(lambda y: ctx.fp8_linear(a, sa, b, sb, y), (m, n))
    assert torch.isfinite(f).all() and torch.equal(f.bfloat16(), h)


@pytest.mark.parametrize("m,k,n", [(2, 2048, 300), (40, 1040, 260), (1600, 528, 3300)])
def test_bf16_is_the_f32_sum_rounded_with_activations_quantised_inside(ctx, m, k, n):
    x = values(m, m, k, "bf16", spread=False).to(DEV)
    b, sb, _ = operand(n, n, k, E4M3, tiles=True)
    b, sb = b.to(DEV), sb.to(DEV)
    f, h = both(lambda y: ctx.fp8_linear_act(x, b, sb, y), (m, n))
    assert torch.isfinite(f).all() and torch.equal(f.bfloat16(), h)


@pytest.mark.parametrize("sizes", [[1, 0, 3], [60, 5, 80], [300, 260], [0, 900, 1], [1500, 700, 1300]])
@pytest.mark.parametrize("code", [E4M3, E5M2])
def test_experts_rows_do_not_depend_on_how_many_there_are(ctx, sizes, code):
    """bf16 rows are the f32 ones rounded, whatever the number of rows, and room behind the last one changes none."""
    k, n = 528, 515
    off = np.concatenate([[0], np.cumsum(sizes)])
    rows = int(off[-1])
    a, sa, _ = operand(3, rows + 4000, k, code)
    ops = [operand(7 + e, n, k, E4M3, tiles=True) for e in range(len(sizes))]
    a, sa = a.to(DEV), sa.to(DEV)
    b, sb = [o[0].to(DEV) for o in ops], [o[1].to(DEV) for o in ops]
    offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
    for r in (rows, rows + 4000):
        f, h = both(lambda y: ctx.fp8_linear_grouped(a[:r], sa[:r], b, sb, offsets, y), (r, n))
        assert torch.isfinite(f[:rows]).all() and torch.equal(f[:rows].bfloat16(), h[:rows])
        assert torch.isnan(f[rows:]).all() and torch.isnan(h[rows:]).all()


@pytest.mark.parametrize("sizes,n,k", [([128], 16, 40), ([0, 384, 256], 130, 260), ([1280, 0, 128], 257, 100)])
@pytest.mark.parametrize("code", [E4M3, E5M2])
def test_experts_gradients_are_rounded_once(ctx, sizes, n, k, code):
    off = np.concatenate([[0], np.cumsum(sizes)])
    rows = int(off[-1])
    a, sa, _ = operand(1, n, rows, code)
    b, sb, _ = operand(2, k, rows, E4M3)
    a, sa, b, sb = (t.to(DEV) for t in (a, sa, b, sb))
    offsets = torch.tensor(off, dtype=torch.int32, device=DEV)
    f, h = both(lambda y: ctx.fp8_grad_weight_grouped(a, sa, b, sb, offsets, y), (len(sizes), n, k))
    assert torch.isfinite(f).all() and torch.equal(f.bfloat16(), h)


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("code,b_rows", [(E4M3, 128), (E5M2, 128), (E4M3, 1), (E5M2, 1)])
def test_sums_on_the_8_bit_pipe(ctx, m, k, n, code, b_rows):
    """bf16 outputs within the pipe's tolerance, f32 ones untouched; the choice can be taken back."""
    a, sa, av = operand(m + k, m, k, code)
    b, sb, bv = operand(n + k, n, k, E4M3, tiles=b_rows == 128)
    a, sa, b, sb = (t.to(DEV) for t in (a, sa, b, sb))
    run = lambda y: ctx.fp8_linear(a, sa, b, sb, y)  # noqa: E731
    f0, h0 = both(run, (m, n))
    ctx.set_fp8_sums(frx.FP8_SUMS_PIPE)
    f1, h1 = both(run, (m, n))
    ctx.set_fp8_sums(frx.FP8_SUMS_F32)
    f2, h2 = both(run, (m, n))
    assert torch.equal(f0, f1) and torch.equal(f0, f2) and torch.equal(h0, h2)
    check(h1, av @ bv.t(), av.abs() @ bv.abs().t(), k)


@pytest.mark.parametrize("sizes,n", [([300, 260], 515), ([0, 900, 1], 132), ([1500, 700, 1300], 3001)])
def test_experts_rows_on_the_8_bit_pipe(ctx, sizes, n):
    k, behind = 656, 5
    ctx.set_fp8_sums(frx.FP8_SUMS_PIPE)
    off = np.concatenate([[0], np.cumsum(sizes)])
    rows = int(off[-1]) + behind
    a, sa, av = operand(5, rows, k, E4M3)
    ops = [operand(7 + e, n, k, E4M3, tiles=True) for e in range(len(sizes))]
    y = torch.full((rows, n), 5.0, dtype=torch.bfloat16, device=DEV)
    ctx.fp8_linear_grouped(a.to(DEV), sa.to(DEV), [o[0].to(DEV) for o in ops], [o[1].to(DEV) for o in ops],
                           torch.tensor(off, dtype=torch.int32, device=DEV), y)
    for e in range(len(sizes)):
        i, j = int(off[e]), int(off[e + 1])
        if j > i:
            check(y[i:j], av[i:j] @ ops[e][2].t(), av[i:j].abs() @ ops[e][2].abs().t(), k)
    assert (y[-behind:] == 5.0).all()


def test_experts_gradients_on_the_8_bit_pipe(ctx):
    n, k, rows = 257, 100, 768
    ctx.set_fp8_sums(frx.FP8_SUMS_PIPE)
    for code in (E4M3, E5M2):
        a, sa, av = operand(1, n, rows, code)
        b, sb, bv = operand(2, k, rows, E4M3)
        dw = torch.full((2, n, k), float("nan"), dtype=torch.bfloat16, device=DEV)
        ctx.fp8_grad_weight_grouped(a.to(DEV), sa.to(DEV), b.to(DEV), sb.to(DEV),
                                    torch.tensor([0, 640, 768], dtype=torch.int32, device=DEV), dw)
        for e, (i, j) in enumerate(((0, 640), (640, 768))):
            check(dw[e], av[:, i:j] @ bv[:, i:j].t(), av[:, i:j].abs() @ bv[:, i:j].abs().t(), j - i)


def test_a_captured_graph_keeps_its_sums(ctx):
    """The choice is made when a call is made: a graph replays what it was captured with."""
    m, k, n = 1600, 528, 3300
    a, sa, _ = operand(1, m, k, E4M3)
    b, sb, _ = operand(2, n, k, E4M3, tiles=True)
    a, sa, b, sb = (t.to(DEV) for t in (a, sa, b, sb))
    y = torch.zeros((m, n), dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    ctx.set_stream(side)
    torch.cuda.synchronize()
    want = []
    for mode in (frx.FP8_SUMS_F32, frx.FP8_SUMS_PIPE):
        ctx.set_fp8_sums(mode)
        ctx.fp8_linear(a, sa, b, sb, y)
        torch.cuda.synchronize()
        want.append(y.clone())
    ctx.set_fp8_sums(frx.FP8_SUMS_F32)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        ctx.fp8_linear(a, sa, b, sb, y)
    for mode in (frx.FP8_SUMS_PIPE, frx.FP8_SUMS_F32, frx.FP8_SUMS_PIPE):
        ctx.set_fp8_sums(mode)
        y.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want[0])
        ctx.fp8_linear(a, sa, b, sb, y)
        torch.cuda.synchronize()
        assert torch.equal(y, want[mode])
    del g


def test_unknown_sums_are_refused(ctx):
    for mode in (2, -1):
        with pytest.raises(frx.FrxError) as e:
            ctx.set_fp8_sums(mode)
        assert e.value.kind == "Unsupported"
