"""Every kernel of the 4-bit linears and of the expert layer for a few tokens (_fp4_kernels, which test_fp4_plan.py holds
against the rules), odd sizes on every side, and tensors past 4 GiB. Tolerances: test_gpu_fp4.py, test_gpu_fp4_moe.py."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp4_kernels import GROUPED, KS, LAYERS, ROWS16, ROWS16_K, SPLIT, TILES
from _fp4_ref import DT, HALF, TABLE, up
from _gpu import DEV
from test_gpu_fp4_moe import check, inputs, reference, routes, weights

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def operand(seed, m, k, extra=0):
    """Codes [m][k / 2] (rows `extra` bytes apart) and scales on the device; 255 behind a row's blocks."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    q = torch.randint(0, 256, (m, k // 2 + extra), dtype=torch.uint8, device=DEV, generator=g)[:, :k // 2]
    s = torch.full((m, up(k, 128) // 32), 255, dtype=torch.uint8, device=DEV)
    s[:, :k // 32] = torch.randint(120, 132, (m, k // 32), dtype=torch.uint8, device=DEV, generator=g)
    return q, s


def values(q, s):
    code = torch.stack([q & 15, q >> 4], -1).flatten(1).long()
    v = torch.from_numpy(TABLE).to(DEV)[code].view(q.shape[0], -1, 32)
    return (v * torch.exp2(s[:, :v.shape[1]].double() - 127)[..., None]).flatten(1)


def close(y, a, b, slices=16):
    ref = a @ b.T
    bound = (a.shape[1] / 32 + slices) * 2.0 ** -24 * (a.abs() @ b.abs().T) + HALF[y.dtype] * ref.abs() + 2.0 ** -133
    off = (y.double() - ref).abs()
    assert bool((off <= bound).all()), (off / bound).max()


def product(ctx, M, K, N, dtype, extra=0):
    a, b = operand(M, M, K, extra), operand(N + 1, N, K, 2 * extra)
    y = torch.full((M, N), float("nan"), dtype=DT[dtype], device=DEV)
    ctx.fp4_linear(*a, *b, y)
    close(y, values(*a), values(*b))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("K", KS)
@pytest.mark.parametrize("M,N", list(TILES.values()))
def test_tiles(ctx, M, N, K, dtype):
    product(ctx, M, K, N, dtype, extra=16 * (K % 3))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", [c[:3] for c in SPLIT])
def test_slices_of_k(ctx, M, K, N, dtype):
    product(ctx, M, K, N, dtype)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("K", ROWS16_K)
@pytest.mark.parametrize("M,N", list(ROWS16))
def test_few_tokens(ctx, M, N, K, dtype):
    product(ctx, M, K, N, dtype, extra=16 * (K % 5))


@pytest.mark.parametrize("xt", ["bf16", "f32"])
@pytest.mark.parametrize("M,K,N", [(1, 4128, 40), (4, 160, 8300), (3, 1056, 16300), (2, 12320, 5000),
                                   (16, 1024, 90), (16, 1056, 90), (9, 1760, 8300), (5, 3264, 16300), (11, 32, 20)])
def test_few_activations(ctx, M, K, N, xt):
    """The launch that makes the codes itself against the two calls, bit for bit."""
    g = torch.Generator(device=DEV).manual_seed(K)
    x = torch.randn((M, K), device=DEV, generator=g).to(DT[xt])
    b = operand(N, N, K)
    q, s = torch.zeros((M, K // 2), dtype=torch.uint8, device=DEV), torch.zeros((M, up(K, 128) // 32), dtype=torch.uint8, device=DEV)
    y, z = torch.zeros((M, N), device=DEV), torch.ones((M, N), device=DEV)
    ctx.fp4_quantize(x, frx.FP4_ROWS, q, s)
    ctx.fp4_linear(q, s, *b, y)
    ctx.fp4_linear_act(x, *b, z)
    assert torch.equal(y, z)
    close(z, values(q, s), values(*b))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("name", list(GROUPED))
def test_grouped_tiles(ctx, name, dtype):
    sizes, behind, K, N, _ = GROUPED[name]
    E, R, off = len(sizes), sum(sizes) + behind, np.concatenate([[0], np.cumsum(sizes)])
    a, b = operand(R, R, K, 16), operand(N, E * N, K)
    y = torch.full((R, N), 7.0, dtype=DT[dtype], device=DEV)
    ctx.fp4_linear_grouped(*a, b[0].view(E, N, -1), b[1].view(E, N, -1), torch.from_numpy(off).int().to(DEV), y)
    va, vb = values(*a), values(*b).view(E, N, -1)
    for e in range(E):
        if sizes[e]:
            close(y[off[e]:off[e + 1]], va[off[e]:off[e + 1]], vb[e])
    assert bool((y[off[-1]:] == 7).all()), "rows behind the last expert's were written"


@pytest.mark.parametrize("t", ["bf16", "f32"])
@pytest.mark.parametrize("T,H,I,E,top_k", LAYERS)
def test_layers(ctx, T, H, I, E, top_k, t):
    rng = np.random.default_rng(T + H + I)
    w = weights(rng, E, I, H)
    x = inputs(rng, T, H, t)
    idx, wt = routes(rng, T, E, top_k)
    idx[rng.random(idx.shape) < 0.1] = -1
    y = torch.full((T, H), float("nan"), dtype=DT[t], device=DEV)
    ctx.fp4_moe_ffn(x.to(DEV), None, *w[0][0], *w[1][0], *w[2][0], y, torch.from_numpy(idx).to(DEV),
                    torch.from_numpy(wt).to(DEV))
    check(y, *reference(x.double().numpy(), [v for _, v in w], idx, wt, frx.ACT_SILU, t))


def test_offsets_that_are_no_sort(ctx):
    """Offsets that go down, or pass the rows there are: rows of some expert or left alone, none outside y."""
    R, K, N, E = 70, 96, 40, 3
    a, b = operand(1, R, K), operand(2, E * N, K)
    for off in ([0, 40, 20, 70], [100, 200, 300, 400], [70, 0, 0, 2 ** 31 - 1], [-1, 5, -1, 60]):
        out = torch.full((R + 16, N), 7.0, device=DEV)
        ctx.fp4_linear_grouped(*a, b[0].view(E, N, -1), b[1].view(E, N, -1),
                               torch.tensor(off, dtype=torch.int32, device=DEV), out[8:R + 8])
        assert bool((out[:8] == 7).all()) and bool((out[R + 8:] == 7).all())


def test_first_calls_under_capture():
    """A product that would split K runs whole, the experts' and the small calls need nothing; a call whose codes have no
    place is refused and the capture goes on."""
    c, side = frx.Context(0), torch.cuda.Stream()
    c.set_stream(side)
    M, K, N = SPLIT[0][:3]
    a, b = operand(1, M, K), operand(2, N, K)
    x, few = torch.randn((M, K), device=DEV), torch.randn((3, K), device=DEV)
    y, z, g = torch.zeros((M, N), device=DEV), torch.zeros((3, N), device=DEV), torch.zeros((M, N), device=DEV)
    off = torch.tensor([0, M], dtype=torch.int32, device=DEV)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        c.fp4_linear(*a, *b, y)
        with pytest.raises(frx.FrxError, match="captured"):
            c.fp4_linear_act(x, *b, y)
        c.fp4_linear_act(few, *b, z)
        c.fp4_linear_grouped(*a, b[0][None], b[1][None], off, g)
    e = frx.Context(0)
    for i in range(3):
        few.normal_()
        for t in (y, z, g):
            t.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        close(y, values(*a), values(*b))
        assert torch.equal(y, g)
        want = torch.zeros_like(z)
        e.fp4_linear_act(few, *b, want)
        assert torch.equal(z, want) and bool(z.any())
        if i == 0:  # an eager call grows the workspace that the graph does without
            c.fp4_linear(*a, *b, torch.zeros((M, N), device=DEV))
            torch.cuda.synchronize()
    del graph
    c.set_stream(None)
    c.close()
    e.close()


def test_two_contexts_at_once():
    """Products, experts' rows and layers of two contexts on two streams, both queued before either is waited for, against
    the same calls alone; one operand on both sides of a product."""
    M, K, N, E, T = 300, 1120, 5010, 8, 7
    n = N // 10
    a, b = operand(1, M, K), operand(2, E * n, K)
    w = [t[None].expand(E, *t.shape).contiguous() for k in ((3, 352, K), (4, 352, K), (5, K, 352)) for t in operand(*k)]
    x, idx = torch.randn((T, K), device=DEV), torch.arange(2 * T, dtype=torch.int32, device=DEV).view(T, 2) % (E + 1)
    off = torch.linspace(0, M, E + 1, device=DEV).int()
    wt, router = torch.rand((T, 2), device=DEV), torch.randn((E, K), device=DEV)

    def calls(c, outs):
        for _ in range(3):
            c.fp4_linear(*a, *a, outs[0])
            c.fp4_linear_grouped(*a, b[0].view(E, n, -1), b[1].view(E, n, -1), off, outs[1])
            c.fp4_moe_ffn(x, None, *w, outs[2], idx, wt)
            c.fp4_moe_ffn(x, router, *w, outs[3], top_k=2)

    want, *got = [[torch.zeros(d, device=DEV) for d in ((M, M), (M, n), (T, K), (T, K))] for _ in range(3)]
    alone = frx.Context(0)
    calls(alone, want)
    torch.cuda.synchronize()
    pairs = [(frx.Context(0), torch.cuda.Stream()) for _ in range(2)]
    for c, stream in pairs:
        c.set_stream(stream)
    for (c, _), outs in zip(pairs, got):
        calls(c, outs)
    torch.cuda.synchronize()
    for outs in got:
        for u, v in zip(outs, want):
            assert torch.equal(u, v) and bool(v.any())
    close(want[0], values(*a), values(*a))
    for c in (alone, *(c for c, _ in pairs)):
        c.set_stream(None)
        c.close()


# ---- past 4 GiB ----------------------------------------------------------------------


@pytest.mark.parametrize("M,N", [(66000, 66001), (3, 1100000)])
def test_long_products(ctx, M, N):
    """y of more than 2^32 values; weights of more than 2^32 bytes."""
    K = 32 if M > 32 else 8192
    a, b = operand(1, M, K), operand(2, N, K)
    assert M * N > 1 << 32 or b[0].numel() > 1 << 32
    y = torch.full((M, N), float("nan"), dtype=torch.bfloat16, device=DEV)
    ctx.fp4_linear(*a, *b, y)
    rows, cols = [0, M // 2, M - 2, M - 1], slice(N - 4000, N)
    close(y[rows][:, cols], values(a[0][rows], a[1][rows]), values(b[0][cols], b[1][cols]))
    assert not bool(torch.isnan(y).any())


def test_long_groups(ctx):
    sizes, K, N = [40000, 0, 25999], 64, 66001
    R, off = sum(sizes) + 1, torch.tensor([0, 40000, 40000, 65999], dtype=torch.int32, device=DEV)
    a, b = operand(3, R, K), operand(4, 3 * N, K)
    y = torch.full((R, N), 7.0, dtype=torch.bfloat16, device=DEV)
    ctx.fp4_linear_grouped(*a, b[0].view(3, N, -1), b[1].view(3, N, -1), off, y)
    for e, rows in ((0, [0, 39999]), (2, [40000, 65998])):
        cols = slice(e * N + N - 3000, e * N + N)
        close(y[rows][:, -3000:], values(a[0][rows], a[1][rows]), values(b[0][cols], b[1][cols]))
    assert bool((y[-1] == 7).all())


@pytest.mark.parametrize("blocks", [frx.FP4_ROWS, frx.FP4_COLS])
def test_long_quantiser(ctx, blocks):
    """x of more than 2^32 values: its ends are what they are alone."""
    M, K = 66016, 65536 + 64
    x = torch.randn((M, K), dtype=torch.bfloat16, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    rows, cols = (M, K) if blocks == frx.FP4_ROWS else (K, M)
    make = lambda r, c: (torch.zeros((r, up(c, 32) // 2), dtype=torch.uint8, device=DEV),  # noqa: E731
                         torch.zeros((r, up(c, 128) // 32), dtype=torch.uint8, device=DEV))
    q, s = make(rows, cols)
    ctx.fp4_quantize(x, blocks, q, s)
    if blocks == frx.FP4_ROWS:
        small = x[-70:].contiguous()
    else:
        small = x[:, -70:].contiguous()
    p, t = make(70, cols)
    ctx.fp4_quantize(small, blocks, p, t)
    assert torch.equal(q[-70:], p) and torch.equal(s[-70:], t)
    if blocks == frx.FP4_ROWS:
        del small
        y = torch.zeros_like(x)
        ctx.fp4_dequantize(q, s, y)
        z = torch.zeros((70, K), dtype=torch.bfloat16, device=DEV)
        ctx.fp4_dequantize(p, t, z)
        assert torch.equal(y[-70:], z) and bool((z.double() == values(p, t)).all())


def test_a_long_expert(ctx):
    """Gate, up and down of more than 2^32 bytes each, one token; the reference by chunks of I, over which y is a sum."""
    H, n = 8192, 34400
    I = 32 * n
    x = torch.randn((1, H), device=DEV, generator=torch.Generator(device=DEV).manual_seed(2))
    gate, up_, down = operand(5, I, H), operand(6, I, H), operand(7, H, I)
    assert gate[0].numel() > 1 << 32 and down[0].numel() > 1 << 32
    y = torch.full((1, H), float("nan"), device=DEV)
    ctx.fp4_moe_ffn(x, None, *(t[None] for w in (gate, up_, down) for t in w), y,
                    torch.zeros((1, 1), dtype=torch.int32, device=DEV), torch.ones((1, 1), device=DEV))
    U, v = 2.0 ** -24, x.double().T
    ref, bound = torch.zeros((H, 1), dtype=torch.float64, device=DEV), torch.zeros((H, 1), dtype=torch.float64, device=DEV)
    for c in range(0, I, n):
        g, u = (values(w[0][c:c + n], w[1][c:c + n]) for w in (gate, up_))
        dg, du = (3 * H * U * (w.abs() @ v.abs()) for w in (g, u))
        g, u = g @ v, u @ v
        a = g / (1 + torch.exp(-g))
        da = 16 * U * a.abs() + 1.13 * dg
        h = a * u
        dh = da * u.abs() + a.abs() * du + da * du + 4 * U * h.abs()
        d = values(down[0][:, c // 2:(c + n) // 2], down[1][:, c // 32:(c + n) // 32])
        ref += d @ h
        bound += d.abs() @ (dh + 3 * I * U * h.abs())
    assert bool(((y.double().T - ref).abs() <= 1.01 * bound + HALF[torch.float32] * ref.abs() + 2.0 ** -133).all())
