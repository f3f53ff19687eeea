"""The 4-bit floating-point linears (frx_fp4_quantize, frx_fp4_dequantize, frx_fp4_linear, _act, _grouped) against their
formulas in 64 bits.

Codes and scales are exact by definition and compared bit for bit. A product's tolerance (_fp4_ref.product_bound): a block
of 32 products is a sum of multiples of 1/4 up to 36 and so exact; each block is one f32 addition, relative to the sum of
the terms' magnitudes; half a step of the output type relative to the value."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp4_ref import DT, pack, product_bound, random_codes, ref_codes, up, values
from _gpu import DEV, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def normal(seed, m, k, dtype, spread=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn((m, k), generator=g)
    if spread:
        x = x * torch.exp(2.0 * torch.randn((1, k), generator=g))
    return x.to(DT[dtype])


def room(r, c, extra=0):
    """q (row stride `extra` bytes longer than its columns, filled with 0x55) and scales of r rows of c values."""
    raw = torch.full((r, up(c, 32) // 2 + extra), 0x55, dtype=torch.uint8, device=DEV)
    return raw, raw[:, :up(c, 32) // 2], torch.full((r, up(c, 128) // 32), 0x55, dtype=torch.uint8, device=DEV)


def on_dev(code, byte, extra=0):
    """Packed codes (rows `extra` bytes apart, 0x77 there) and scales on the device."""
    q = pack(code)
    raw = np.full((q.shape[0], q.shape[1] + extra), 0x77, np.uint8)
    raw[:, :q.shape[1]] = q
    return torch.from_numpy(raw).to(DEV)[:, :q.shape[1]], torch.from_numpy(byte).to(DEV)


SHAPES = [(1, 1), (1, 32), (3, 130), (127, 128), (129, 257), (200, 288), (5, 1000), (300, 7), (33, 31)]


@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k", SHAPES)
def test_quantize_is_exact(ctx, cols, dtype, m, k):
    x = normal(m * 1000 + k, m, k, dtype)
    r, c = (k, m) if cols else (m, k)
    raw, q, s = room(r, c, extra=32)
    ctx.fp4_quantize(x.to(DEV), frx.FP4_COLS if cols else frx.FP4_ROWS, q, s)
    code, byte = ref_codes(x.t() if cols else x)
    assert np.array_equal(s.cpu().numpy(), byte)
    assert np.array_equal(q.cpu().numpy(), pack(code))
    assert (raw[:, up(c, 32) // 2:].cpu() == 0x55).all(), "bytes behind a row were written"


@pytest.mark.parametrize("cols", [False, True])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_odd_strides_and_offsets(ctx, cols, dtype):
    """Rows of a wider tensor from an odd element on: no vector loads apply. Codes as torch's own 4-bit dtype."""
    big = normal(5, 150, 301, dtype)
    x = big[1:140, 3:290]
    r, c = (287, 139) if cols else (139, 287)
    _, q, s = room(r, c)
    ctx.fp4_quantize(big.to(DEV)[1:140, 3:290], frx.FP4_COLS if cols else frx.FP4_ROWS,
                     q.view(torch.float4_e2m1fn_x2), s.view(torch.float8_e8m0fnu))
    code, byte = ref_codes(x.t() if cols else x)
    assert np.array_equal(s.cpu().numpy(), byte) and np.array_equal(q.cpu().numpy(), pack(code))


@pytest.mark.parametrize("cols", [False, True])
def test_quantize_special_values(ctx, cols):
    """Every rounding border and its neighbours, zeros of both signs, denormals, the largest numbers; a NaN and an
    infinity spoil their own block alone."""
    x = torch.zeros((256, 384))
    border = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 7.0])
    near = torch.cat([border, torch.nextafter(border, torch.tensor(0.0)), torch.nextafter(border, torch.tensor(9.0)),
                      -border])
    x[:32, :32] = near[:, None].expand(32, 32) if cols else near
    x[:, 128:256] = normal(9, 256, 128, "f32")
    x[3, 65], x[40, 70] = 1e-42, -2.0 ** -149
    x[7, 300], x[9, 340] = torch.finfo(torch.float32).max, 2.0 ** -126
    x[200, 130], x[20, 200] = float("nan"), float("-inf")
    x[100, 64] = -0.0
    r, c = (384, 256) if cols else (256, 384)
    _, q, s = room(r, c)
    ctx.fp4_quantize(x.to(DEV), frx.FP4_COLS if cols else frx.FP4_ROWS, q, s)
    code, byte = ref_codes(x.t() if cols else x)
    assert np.array_equal(s.cpu().numpy(), byte) and np.array_equal(q.cpu().numpy(), pack(code))
    assert (byte == 255).sum() == 2 and (byte == 252).any() and (byte == 0).any()
    y = torch.zeros((r, c), device=DEV)
    ctx.fp4_dequantize(q, s, y)
    assert np.array_equal(host(y).astype(np.float64), values(code, byte)[:, :c], equal_nan=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,extra", [(1, 1, 0), (3, 31, 0), (7, 96, 16), (65, 131, 5), (130, 264, 0)])
def test_dequantize_every_scale(ctx, dtype, m, k, extra):
    """All scales but the largest ones, whose values pass the type's range; rows of a wider result stay apart."""
    rng = np.random.default_rng(k)
    code, byte = random_codes(rng, m, up(k, 32), 0, 253)
    byte[0, 0] = 255
    q, s = on_dev(code, byte, extra=16)
    wide = torch.full((m, k + extra), 7.0, dtype=DT[dtype], device=DEV)
    ctx.fp4_dequantize(q, s, wide[:, :k])
    got = host(wide)
    assert np.array_equal(got[:, :k].astype(np.float64), values(code, byte)[:, :k], equal_nan=True)
    assert (got[:, k:] == 7).all()


def check_product(ctx, M, K, N, dtype, seed, lo=120, hi=132, extra=0, call=None):
    rng = np.random.default_rng(seed)
    (ca, sa), (cb, sb) = random_codes(rng, M, K, lo, hi), random_codes(rng, N, K, lo, hi)
    y = torch.full((M, N), float("nan"), dtype=DT[dtype], device=DEV)
    ctx.fp4_linear(*on_dev(ca, sa, extra), *on_dev(cb, sb, 2 * extra), y)
    a, b = values(ca, sa), values(cb, sb)
    ref = a @ b.T
    err = np.abs(host(y).astype(np.float64) - ref)
    assert (err <= product_bound(a, b, ref, DT[dtype])).all(), (err / product_bound(a, b, ref, DT[dtype])).max()


# few tokens, row tiles of one to four a workgroup; tiles of many tokens; edges on every side
PRODUCTS = [(1, 32, 1), (1, 2048, 48), (2, 96, 17), (5, 416, 100), (16, 1024, 16), (17, 352, 33), (31, 4096, 40), (32, 64, 5),
            (33, 288, 130), (64, 4128, 24), (64, 160, 70), (65, 32, 1), (65, 256, 129), (128, 512, 128), (130, 4128, 257),
            (200, 224, 300), (257, 1056, 511), (300, 992, 64), (1000, 288, 60), (12, 256, 4112), (1, 256, 8192),
            (3, 160, 12304), (40, 128, 8200)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", PRODUCTS)
def test_linear(ctx, M, K, N, dtype):
    check_product(ctx, M, K, N, dtype, M + 3 * K + 7 * N, extra=16 * (M % 3))


@pytest.mark.parametrize("M", [4, 70])
def test_linear_far_scales(ctx, M):
    """Scales whose sum is below any f32 number's exponent, or above; results down to denormal ones."""
    check_product(ctx, M, 256, 40, "f32", 1, 0, 60)        # nothing but zeros is left
    check_product(ctx, M, 256, 40, "f32", 2, 50, 70)       # denormals among the results
    rng = np.random.default_rng(3)
    (ca, sa), (cb, sb) = random_codes(rng, M, 256, 0, 8), random_codes(rng, 40, 256, 246, 253)
    y = torch.zeros((M, 40), device=DEV)
    ctx.fp4_linear(*on_dev(ca, sa), *on_dev(cb, sb), y)
    a, b = values(ca, sa), values(cb, sb)
    assert (np.abs(host(y) - a @ b.T) <= product_bound(a, b, a @ b.T, torch.float32)).all()


@pytest.mark.parametrize("M,N", [(3, 20), (20, 40), (50, 20), (70, 140)])
def test_a_nan_stays_in_its_row(ctx, M, N):
    rng = np.random.default_rng(M)
    (ca, sa), (cb, sb) = random_codes(rng, M, 416), random_codes(rng, N, 416)
    sa[1, 12] = sb[2, 0] = 255
    ca[1, 384:] = 0
    y = torch.zeros((M, N), device=DEV)
    ctx.fp4_linear(*on_dev(ca, sa), *on_dev(cb, sb), y)
    bad = np.zeros((M, N), bool)
    bad[1], bad[:, 2] = True, True
    assert np.array_equal(np.isnan(host(y)), bad)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("xt", ["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", [(1, 32, 1), (1, 2048, 70), (2, 4096, 33), (3, 96, 16), (4, 416, 130), (4, 30848, 20),
                                   (4, 32768, 20), (5, 288, 40), (64, 96, 20), (90, 352, 50)])
def test_linear_act_is_the_two_calls(ctx, M, K, N, dtype, xt):
    x = normal(K, M, K, xt).to(DEV)
    w = normal(N, N, K, "f32").to(DEV)
    _, wq, ws = room(N, K)
    ctx.fp4_quantize(w, frx.FP4_ROWS, wq, ws)
    _, q, s = room(M, K)
    ctx.fp4_quantize(x, frx.FP4_ROWS, q, s)
    y, y2 = (torch.full((M, N), float("nan"), dtype=DT[dtype], device=DEV) for _ in range(2))
    ctx.fp4_linear(q, s, wq, ws, y)
    ctx.fp4_linear_act(x, wq, ws, y2)
    assert torch.equal(y, y2) and torch.isfinite(y).all()
    odd = torch.zeros(M * K + 1, dtype=x.dtype, device=DEV)[1:].view(M, K).copy_(x)  # no vector loads
    y2.zero_()
    ctx.fp4_linear_act(odd, wq, ws, y2)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("m,k,n", [(1, 32, 64), (33, 64, 40), (130, 96, 200), (257, 384, 129)])
def test_gradients(ctx, dtype, m, k, n):
    """dx and dw from the quantiser's two layouts: the formula's values, and the slope of sum(dy y) along a random
    direction of w and of x (the product is linear, so a difference of any step is its slope)."""
    x, w, dy = normal(1, m, k, dtype), normal(2, n, k, "f32"), normal(3, m, n, dtype)
    quant = lambda t, b, r, c: (lambda o: (ctx.fp4_quantize(t.to(DEV), b, *o[1:]), o[1:])[1])(room(r, c))  # noqa: E731
    wt, dyr, dyt, xt = (quant(w, frx.FP4_COLS, k, n), quant(dy, frx.FP4_ROWS, m, n), quant(dy, frx.FP4_COLS, n, m),
                        quant(x, frx.FP4_COLS, k, m))
    if n % 32:  # the sums run over whole blocks: the quantiser's zero codes
        assert wt[0].shape[1] * 2 == up(n, 32)
    dx, dw = torch.zeros((m, k), device=DEV), torch.zeros((n, k), device=DEV)
    ctx.fp4_linear(*dyr, *wt, dx)
    ctx.fp4_linear(*dyt, *xt, dw)
    vdyr, vwt = values(*ref_codes(dy)), values(*ref_codes(w.t()))
    vdyt, vxt = values(*ref_codes(dy.t())), values(*ref_codes(x.t()))
    for got, a, b in ((dx, vdyr, vwt), (dw, vdyt, vxt)):
        ref = a @ b.T
        assert (np.abs(host(got) - ref) <= product_bound(a, b, ref, torch.float32)).all()
    rng = np.random.default_rng(4)
    step = rng.standard_normal((n, k))
    loss = lambda wv: (vdyt[:, :m].T * (vxt[:, :m].T @ wv.T)).sum()  # noqa: E731
    w0 = rng.standard_normal((n, k))
    slope, terms = loss(w0 + step) - loss(w0), np.abs(vdyt) @ np.abs(vxt).T
    assert abs((host(dw) * step).sum() - slope) <= ((m / 32 + 17) * 2.0 ** -24 * (terms * np.abs(step)).sum()
                                                   + 2.0 ** -40 * (terms * (np.abs(step) + 2 * np.abs(w0))).sum())


GROUPS = [([3, 0, 5, 1], 0, 96, 40), ([0, 0, 0], 8, 64, 20), ([17, 1, 40], 3, 416, 130), ([130, 65, 64, 0, 200], 9, 288, 257),
          ([1] * 64, 0, 64, 16), ([600], 20, 256, 300), ([2, 2, 2, 2], 0, 4128, 33)]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("stacked", [True, False])
@pytest.mark.parametrize("sizes,behind,K,N", GROUPS)
def test_grouped(ctx, sizes, behind, K, N, stacked, dtype):
    rng = np.random.default_rng(N)
    E, R = len(sizes), sum(sizes) + behind
    ca, sa = random_codes(rng, R, K)
    cb, sb = random_codes(rng, E * N, K)
    off = np.concatenate([[0], np.cumsum(sizes)])
    q, s = on_dev(cb, sb)
    q, s = q.view(E, N, -1), s.view(E, N, -1)
    y = torch.full((R, N), 7.0, dtype=DT[dtype], device=DEV)
    ctx.fp4_linear_grouped(*on_dev(ca, sa, 16), q if stacked else list(q), s if stacked else list(s),
                           torch.from_numpy(off).int().to(DEV), y)
    got, b = host(y), values(cb, sb).reshape(E, N, K)
    for e in range(E):
        a = values(ca, sa)[off[e]:off[e + 1]]
        ref = a @ b[e].T
        assert (np.abs(got[off[e]:off[e + 1]] - ref) <= product_bound(a, b[e], ref, DT[dtype])).all()
    assert (got[off[-1]:] == 7).all(), "rows behind the last expert's were written"


@pytest.mark.parametrize("T,top_k,E,H,N", [(1, 1, 1, 32, 16), (9, 2, 4, 160, 70), (70, 4, 8, 288, 40), (300, 2, 16, 64, 132)])
def test_together_with_the_sort(ctx, T, top_k, E, H, N):
    """Quantise, sort, dispatch codes and scales, product, combine: the layer's linear as a user runs it."""
    rng = np.random.default_rng(T)
    x, w = normal(T, T, H, "bf16"), normal(T + 1, E * N, H, "f32")
    idx = rng.integers(-1, E, (T, top_k)).astype(np.int32)
    wt = rng.random((T, top_k)).astype(np.float32)
    _, q, s = room(T, H)
    _, wq, ws = room(E * N, H)
    ctx.fp4_quantize(x.to(DEV), frx.FP4_ROWS, q, s)
    ctx.fp4_quantize(w.to(DEV), frx.FP4_ROWS, wq, ws)
    rows = frx.MoeRows.empty(T, top_k, E)
    ctx.moe_sort(torch.from_numpy(idx).to(DEV), rows)
    _, aq, as_ = room(rows.R, H)
    ctx.moe_dispatch(q, rows, aq)
    ctx.moe_dispatch(s, rows, as_)
    ys, y = torch.zeros((rows.R, N), device=DEV), torch.zeros((T, N), device=DEV)
    ctx.fp4_linear_grouped(aq, as_, wq.view(E, N, -1), ws.view(E, N, -1), rows.offsets, ys)
    ctx.moe_combine(ys, rows, torch.from_numpy(wt).to(DEV), y)
    a, b = values(*ref_codes(x)), values(*ref_codes(w)).reshape(E, N, -1)
    ref, bound = np.zeros((T, N)), np.zeros((T, N))
    for t in range(T):
        for j in range(top_k):
            if idx[t, j] >= 0:
                one = a[t:t + 1] @ b[idx[t, j]].T
                ref[t] += wt[t, j] * one[0]
                bound[t] += wt[t, j] * (product_bound(a[t:t + 1], b[idx[t, j]], one, torch.float32)[0]
                                        + (top_k + 1) * 2.0 ** -24 * np.abs(one[0]))
    assert (np.abs(host(y) - ref) <= bound + top_k * 2.0 ** -24 * np.abs(ref)).all()


@pytest.mark.parametrize("M", [2, 20, 90])
def test_captured_on_another_stream(M):
    """A forward and backward run in a graph on a side stream, replayed on new inputs, against eager calls."""
    c, e = frx.Context(0), frx.Context(0)
    K, N = 352, 200
    x, w, dy = normal(1, M, K, "bf16").to(DEV), normal(2, N, K, "f32").to(DEV), normal(3, M, N, "bf16").to(DEV)
    bufs = [[room(*d)[1:] for d in ((N, K), (K, N), (M, N), (N, M), (K, M))] for _ in range(2)]
    outs = [[torch.zeros(d, device=DEV) for d in ((M, N), (M, K), (N, K))] for _ in range(2)]

    def step(ctx, b, o):
        ctx.fp4_quantize(w, frx.FP4_ROWS, *b[0])
        ctx.fp4_quantize(w, frx.FP4_COLS, *b[1])
        ctx.fp4_linear_act(x, *b[0], o[0])
        ctx.fp4_quantize(dy, frx.FP4_ROWS, *b[2])
        ctx.fp4_quantize(dy, frx.FP4_COLS, *b[3])
        ctx.fp4_quantize(x, frx.FP4_COLS, *b[4])
        ctx.fp4_linear(*b[2], *b[1][:1], b[1][1], o[1])
        ctx.fp4_linear(*b[3], *b[4], o[2])

    side = torch.cuda.Stream()
    c.set_stream(side)
    torch.cuda.synchronize()
    step(c, bufs[0], outs[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step(c, bufs[0], outs[0])
    for i in range(3):
        x.copy_(normal(10 + i, M, K, "bf16"))
        w.mul_(1.25)
        step(e, bufs[1], outs[1])
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(*outs))
    del graph
    c.set_stream(None)
    c.close()
    e.close()


def test_results_repeat(ctx):
    """The same call gives the same bits."""
    x, w = normal(1, 300, 1056, "f32").to(DEV), normal(2, 200, 1056, "f32").to(DEV)
    _, q, s = room(200, 1056)
    ctx.fp4_quantize(w, frx.FP4_ROWS, q, s)
    for m in (1, 16, 60, 300):
        y, z = torch.zeros((m, 200), device=DEV), torch.zeros((m, 200), device=DEV)
        ctx.fp4_linear_act(x[:m], q, s, y)
        for _ in range(5):
            ctx.fp4_linear_act(x[:m], q, s, z)
            assert torch.equal(y, z)
