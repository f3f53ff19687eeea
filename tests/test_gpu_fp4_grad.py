"""Gradients of a layer of experts in 4-bit floating point (frx_fp4_grad_weight_grouped, and the grouped product for x)
against their formula in 64 bits and against differences. A product's tolerance: test_gpu_fp4.py."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp4_kernels import GRADS
from _fp4_ref import DT, HALF, up
from _gpu import DEV
from test_gpu_fp4_kernels import close, operand, values

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def new(r, c):
    return (torch.zeros((r, up(c, 32) // 2), dtype=torch.uint8, device=DEV),
            torch.zeros((r, up(c, 128) // 32), dtype=torch.uint8, device=DEV))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("name", list(GRADS))
def test_weight_gradients(ctx, name, dtype):
    """NaN scales stand behind the last segment; lists and stacked matrices."""
    sizes, behind, N, K, _ = GRADS[name]
    E, R, off = len(sizes), sum(sizes) + behind, np.concatenate([[0], np.cumsum(sizes)])
    a, b = operand(1, N, R, 16), operand(2, K, R, 48)
    va, vb = values(*a), values(*b)
    for _, s in (a, b):
        s[:, off[-1] // 32:] = 255
    o = torch.from_numpy(off).int().to(DEV)
    room = torch.full((E + 2, N, K), 7.0, dtype=DT[dtype], device=DEV)
    dw = room[1:-1]
    ctx.fp4_grad_weight_grouped(*a, *b, o, dw)
    for e in range(E):
        if sizes[e]:
            close(dw[e], va[:, off[e]:off[e + 1]], vb[:, off[e]:off[e + 1]])
        else:
            assert not bool(dw[e].any())
    assert bool((room[0] == 7).all()) and bool((room[-1] == 7).all())
    lists = [torch.full((N, K), 3.0, dtype=DT[dtype], device=DEV) for _ in range(E)]
    ctx.fp4_grad_weight_grouped(*a, *b, o, lists)
    assert all(torch.equal(x, y) for x, y in zip(lists, dw))


def test_rows_that_end_inside_a_block(ctx):
    """R is a multiple of 32: the last expert's rows end there, and experts behind it have none."""
    N, K, R = 50, 70, 288
    a, b = operand(1, N, R), operand(2, K, R)
    dw = torch.full((4, N, K), float("nan"), device=DEV)
    ctx.fp4_grad_weight_grouped(*a, *b, torch.tensor([0, 256, 288, 288, 384], dtype=torch.int32, device=DEV), dw)
    va, vb = values(*a), values(*b)
    close(dw[0], va[:, :256], vb[:, :256])
    close(dw[1], va[:, 256:], vb[:, 256:])
    assert not bool(dw[2:].any())


def test_an_odd_address(ctx):
    """dw from any element on."""
    a, b = operand(1, 70, 256), operand(2, 45, 256)
    o = torch.tensor([0, 128, 256], dtype=torch.int32, device=DEV)
    dw, odd = torch.zeros((2, 70, 45), device=DEV), torch.zeros(2 * 70 * 45 + 1, device=DEV)[1:].view(2, 70, 45)
    ctx.fp4_grad_weight_grouped(*a, *b, o, dw)
    ctx.fp4_grad_weight_grouped(*a, *b, o, odd)
    assert torch.equal(dw, odd) and bool(dw.any())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,top_k,E,H,N", [(1, 1, 3, 32, 16), (50, 2, 4, 160, 70), (300, 4, 16, 96, 130)])
def test_a_layer_backward(ctx, dtype, T, top_k, E, H, N):
    """Sort, dispatch, products, combine, and all of it backward, as a user runs it: dx and dw against the formula over the
    codes' values, and against differences of the loss sum(c * y) that those values give. The loss is linear in one row of
    a weight matrix and in one token: a difference is exact but for its rounding."""
    g = torch.Generator(device=DEV).manual_seed(T)
    rnd = lambda *d: torch.randn(d, device=DEV, generator=g)  # noqa: E731
    x, w, dy = rnd(T, H).to(DT[dtype]), rnd(E * N, H), rnd(T, N).to(DT[dtype])
    idx = torch.randint(-1, E, (T, top_k), device=DEV, generator=g).int()
    wt = torch.rand((T, top_k), device=DEV, generator=g)
    rows = frx.MoeRows.empty(T, top_k, E, align=128)
    ctx.moe_sort(idx, rows)
    xs = torch.zeros((rows.R, H), dtype=DT[dtype], device=DEV)
    ctx.moe_dispatch(x, rows, xs)
    # the combination's gradient: rows of dy times their weight
    dys, ys = torch.zeros((rows.R, N), dtype=DT[dtype], device=DEV), torch.zeros((rows.R, N), dtype=DT[dtype], device=DEV)
    ctx.moe_combine_backward(dy, ys, rows, wt, dys, torch.zeros((T, top_k), device=DEV))
    dyt, xt = ctx.fp4_quantize(dys, frx.FP4_COLS, *new(N, rows.R)), ctx.fp4_quantize(xs, frx.FP4_COLS, *new(H, rows.R))
    dw = torch.full((E, N, H), float("nan"), device=DEV)
    ctx.fp4_grad_weight_grouped(*dyt, *xt, rows.offsets, dw)
    # N may be no multiple of 32: the codes of a row of dy are padded with zeros, and so are w's along N
    dyr, wt4 = ctx.fp4_quantize(dys, frx.FP4_ROWS, *new(rows.R, N)), []
    for e in range(E):
        wt4.append(ctx.fp4_quantize(w[e * N:(e + 1) * N], frx.FP4_COLS, *new(H, N)))
    dxs, dx = torch.zeros((rows.R, H), device=DEV), torch.zeros((T, H), device=DEV)
    ctx.fp4_linear_grouped(*dyr, [q for q, _ in wt4], [s for _, s in wt4], rows.offsets, dxs)
    ctx.moe_combine(dxs, rows, None, dx)
    off = rows.offsets.tolist()
    row_of, slot = rows.row_of.cpu().numpy().astype(np.int64), idx.cpu().numpy()
    vt, vx, vr = values(*dyt), values(*xt), values(*dyr)
    for e in range(E):
        if off[e + 1] > off[e]:
            close(dw[e], vt[:, off[e]:off[e + 1]], vx[:, off[e]:off[e + 1]])
            close(dxs[off[e]:off[e + 1]], vr[off[e]:off[e + 1]], values(*wt4[e]))
        else:
            assert not bool(dw[e].any())
    # L(W) = sum over the expert's rows of dy's values times (x's values W^T): one entry's difference
    e = int(slot[slot >= 0][0]) if (slot >= 0).any() else 0
    seg = slice(off[e], off[e + 1])
    if off[e + 1] > off[e]:
        loss = lambda m: (vt[:, seg].T * (vx[:, seg].T @ m.T)).sum()  # noqa: E731
        m0 = w[e * N:(e + 1) * N].double()
        for n, k in ((0, 0), (N - 1, H - 1), (N // 2, H // 3)):
            m1 = m0.clone()
            m1[n, k] += 1.0
            step = float(loss(m1) - loss(m0))
            terms = float((vt[n, seg].abs() * vx[k, seg].abs()).sum())
            size = float((vt[:, seg].T * (vx[:, seg].T @ m0.T)).abs().sum())
            # a block of 32 rows is one f32 addition, and the output's rounding; 64-bit sums of the losses
            assert abs(step - float(dw[e, n, k])) <= ((off[e + 1] - off[e]) / 32 + 2) * 2.0 ** -24 * terms + 2.0 ** -40 * size
    # dx of one token: the sum of its routes' rows
    for t in (0, T - 1):
        want = sum((dxs[row_of[t, j]].double() for j in range(top_k) if 0 <= slot[t, j] < E), torch.zeros(H, device=DEV).double())
        mag = sum((dxs[row_of[t, j]].double().abs() for j in range(top_k) if 0 <= slot[t, j] < E), torch.zeros(H, device=DEV).double())
        assert bool(((dx[t].double() - want).abs() <= top_k * HALF[torch.float32] * mag).all())


def test_captured(ctx):
    """The first call is captured, replayed over new codes."""
    c, side = frx.Context(0), torch.cuda.Stream()
    c.set_stream(side)
    a, b = operand(1, 100, 384), operand(2, 60, 384)
    o = torch.tensor([0, 128, 128, 384], dtype=torch.int32, device=DEV)
    dw, want = torch.zeros((3, 100, 60), device=DEV), torch.zeros((3, 100, 60), device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.fp4_grad_weight_grouped(*a, *b, o, dw)
    for i in range(3):
        a[0].copy_(operand(7 + i, 100, 384)[0])
        o.copy_(torch.tensor([0, 128, 128 * (i + 1), 384], dtype=torch.int32))
        dw.fill_(float("nan"))
        ctx.fp4_grad_weight_grouped(*a, *b, o, want)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(dw, want) and bool(dw.any())
    del graph
    c.set_stream(None)
    c.close()


def test_long_gradients(ctx):
    """dw of more than 2^32 values: the last of them."""
    N, K, R = 66001, 66001, 128
    a, b = operand(1, N, R), operand(2, K, R)
    dw = torch.full((1, N, K), float("nan"), dtype=torch.bfloat16, device=DEV)
    ctx.fp4_grad_weight_grouped(*a, *b, torch.tensor([0, R], dtype=torch.int32, device=DEV), dw)
    r, c = slice(N - 70, N), slice(K - 4000, K)
    close(dw[0, r, c], values(a[0][r], a[1][r]), values(b[0][c], b[1][c]))
    assert not bool(torch.isnan(dw).any())
