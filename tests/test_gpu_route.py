"""Tokens sorted by expert and back (frx_moe_sort, _dispatch, _combine, _combine_backward) against plain loops, and one
training step of an expert layer through all of them.

The sort is integers, the dispatch copies, dys one f32 product: compared bit for bit. A combination rounds each product
and each of its top_k additions once, 2^-24 relative to the sum of the magnitudes, and then to its output type; a dot
product over H terms any order of H additions and a rounding of each product."""
import ctypes

import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _gpu import DEV
from test_gpu_fp8 import E4M3, E5M2, gen, operand, quantize, up

pytestmark = pytest.mark.gpu
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def ref_sort(idx, E, align, R):
    T, k = idx.shape
    off, row_of, slot_of = [0], np.full((T, k), -1, np.int32), np.full(R, -1, np.int32)
    for e in range(E):
        row = off[-1]
        for slot in np.nonzero(idx.reshape(-1) == e)[0]:
            row_of[slot // k, slot % k] = row
            slot_of[row] = slot
            row += 1
        off.append(up(row, align))
    return np.array(off, np.int32), row_of, slot_of


def routes(seed, T, top_k, E, how):
    rng = np.random.RandomState(seed)
    if how == "one":  # every route to one expert
        return np.full((T, top_k), E - 1, np.int32)
    if how == "none":
        return np.full((T, top_k), -1, np.int32)
    idx = rng.randint(0, E, (T, top_k)).astype(np.int32)
    if how == "holes":  # dropped routes, whole tokens of padding, indices past E
        idx[rng.rand(T, top_k) < 0.3] = -1
        idx[rng.rand(T) < 0.2] = E
        idx[rng.rand(T, top_k) < 0.05] = 2 ** 31 - 1
    if how == "twice":  # the same expert twice in a token
        idx[:, 1:] = idx[:, :1]
    return idx


def make(ctx, idx, E, align, extra=0):
    T, top_k = idx.shape
    R = frx.MoeRows.capacity(T, top_k, E, align) + extra
    new = lambda *s: torch.full(s, 0x5A5A5A5A, dtype=torch.int32, device=DEV)  # noqa: E731
    rows = frx.MoeRows(E, align, new(E + 1), new(T, top_k), new(R))
    ctx.moe_sort(torch.from_numpy(idx).to(DEV), rows)
    return rows


SORTS = [(1, 1, 1, 1, "any"), (1, 2, 8, 1, "any"), (7, 2, 16, 128, "holes"), (64, 4, 64, 16, "any"),
         (33, 4, 8, 1, "twice"), (200, 2, 5, 2, "holes"), (1000, 2, 64, 128, "holes"), (513, 8, 32, 64, "one"),
         (40, 2, 16, 32, "none"), (3000, 3, 48, 1, "holes"), (9000, 2, 64, 8, "holes"), (20000, 4, 7, 128, "any"),
         (5, 64, 64, 4, "any"), (4096, 1, 64, 1, "one")]


@pytest.mark.parametrize("T,top_k,E,align,how", SORTS)
def test_sort(ctx, T, top_k, E, align, how):
    idx = routes(T + E, T, top_k, E, how)
    rows = make(ctx, idx, E, align, extra=5)
    off, row_of, slot_of = ref_sort(idx, E, align, rows.R)
    assert np.array_equal(rows.offsets.cpu().numpy(), off)
    assert np.array_equal(rows.row_of.cpu().numpy(), row_of)
    assert np.array_equal(rows.slot_of.cpu().numpy(), slot_of)


CASES = [(1, 1, 1, 1, "any", 1), (1, 2, 8, 1, "any", 2048), (9, 2, 16, 128, "holes", 40), (33, 4, 8, 1, "twice", 129),
         (64, 2, 64, 16, "holes", 1000), (130, 8, 32, 64, "holes", 7), (40, 2, 16, 32, "none", 64),
         (300, 2, 8, 128, "holes", 2056), (50, 3, 4, 8, "one", 515), (6, 64, 16, 1, "any", 96)]


@pytest.mark.parametrize("T,top_k,E,align,how,H", CASES)
@pytest.mark.parametrize("dtype", ["f32", "bf16", "codes"])
def test_dispatch(ctx, T, top_k, E, align, how, H, dtype):
    idx = routes(T, T, top_k, E, how)
    rows = make(ctx, idx, E, align, extra=3)
    off, _, slot_of = ref_sort(idx, E, align, rows.R)
    if dtype == "codes":
        x = torch.randint(0, 255, (T, up(H, 4)), dtype=torch.uint8, generator=gen(1))
    else:
        x = torch.randn((T, up(H, 2)), generator=gen(1)).to(DT[dtype])
    xs = torch.full((rows.R, x.shape[1]), 77, dtype=x.dtype, device=DEV)
    ctx.moe_dispatch(x.to(DEV), rows, xs)
    want = torch.full(xs.shape, 77, dtype=x.dtype)
    want[:off[-1]] = 0
    for r, s in enumerate(slot_of):
        if s >= 0:
            want[r] = x[s // top_k]
    assert torch.equal(xs.cpu(), want)


def test_dispatch_unaligned(ctx):
    """Rows of no multiple of 16 bytes, from an address of none."""
    idx = routes(4, 20, 2, 8, "holes")
    rows = make(ctx, idx, 8, 16)
    flat = torch.arange(20 * 33 + 1, dtype=torch.float32)
    dev = flat.to(DEV)[1:].view(20, 33)
    out = torch.full((rows.R * 33 + 1,), -1.0, device=DEV)
    xs = out[1:].view(rows.R, 33)
    ctx.moe_dispatch(dev, rows, xs)
    x = flat[1:].view(20, 33)
    off, _, slot_of = ref_sort(idx, 8, 16, rows.R)
    for r, s in enumerate(slot_of):
        want = x[s // 2] if s >= 0 else torch.zeros(33) if r < off[-1] else torch.full((33,), -1.0)
        assert torch.equal(xs[r].cpu(), want)
    assert out[0] == -1.0


@pytest.mark.parametrize("T,top_k,E,align,how,H", CASES)
@pytest.mark.parametrize("st,yt,weights", [("f32", "f32", True), ("bf16", "bf16", True), ("bf16", "f32", False),
                                           ("f32", "bf16", True)])
def test_combine(ctx, T, top_k, E, align, how, H, st, yt, weights):
    """Routes that go nowhere add nothing, though their weight is NaN; the rows that no route has hold NaN."""
    idx = routes(T, T, top_k, E, how)
    rows = make(ctx, idx, E, align)
    _, row_of, slot_of = ref_sort(idx, E, align, rows.R)
    g = gen(T + H)
    ys = torch.randn((rows.R, H), generator=g).to(DT[st])
    ys[torch.from_numpy(slot_of < 0)] = float("nan")
    w = torch.randn((T, top_k), generator=g) if weights else None
    if weights:
        w[torch.from_numpy(row_of < 0)] = float("nan")
    y = torch.full((T, H), float("nan"), dtype=DT[yt], device=DEV)
    ctx.moe_combine(ys.to(DEV), rows, w.to(DEV) if weights else None, y)
    ref, mag = torch.zeros((T, H), dtype=torch.float64), torch.zeros((T, H), dtype=torch.float64)
    for t in range(T):
        for j in range(top_k):
            if row_of[t, j] >= 0:
                p = ys[row_of[t, j]].double() * (w[t, j].double() if weights else 1.0)
                ref[t] += p
                mag[t] += p.abs()
    tol = (top_k + 1) * 2.0 ** -24 * mag + torch.finfo(DT[yt]).eps / 2 * (ref.abs() + (top_k + 1) * 2.0 ** -24 * mag)
    assert ((y.cpu().double() - ref).abs() <= tol * (1 + 1e-6)).all()


@pytest.mark.parametrize("T,top_k,E,align,how,H", CASES)
@pytest.mark.parametrize("dt,st,weights,with_ys", [("f32", "f32", True, True), ("bf16", "bf16", True, True),
                                                   ("f32", "bf16", True, False), ("bf16", "f32", False, True)])
def test_combine_backward(ctx, T, top_k, E, align, how, H, dt, st, weights, with_ys):
    idx = routes(T, T, top_k, E, how)
    rows = make(ctx, idx, E, align, extra=3)
    off, row_of, slot_of = ref_sort(idx, E, align, rows.R)
    g = gen(T + H)
    dy = torch.randn((T, H), generator=g).to(DT[dt])
    ys = torch.randn((rows.R, H), generator=g).to(DT[st])
    ys[torch.from_numpy(slot_of < 0)] = float("nan")
    w = torch.randn((T, top_k), generator=g) if weights else None
    if weights:
        w[torch.from_numpy(row_of < 0)] = float("nan")
    dys = torch.full((rows.R, H), 7.0, dtype=DT[st], device=DEV)
    dw = torch.full((T, top_k), float("nan"), device=DEV) if with_ys else None
    ctx.moe_combine_backward(dy.to(DEV), ys.to(DEV) if with_ys else None, rows, w.to(DEV) if weights else None, dys, dw)
    want = torch.full((rows.R, H), 7.0).to(DT[st])
    want[:off[-1]] = 0
    rw, mag = torch.zeros((T, top_k), dtype=torch.float64), torch.zeros((T, top_k), dtype=torch.float64)
    for t in range(T):
        for j in range(top_k):
            r = row_of[t, j]
            if r >= 0:
                want[r] = ((w[t, j] if weights else 1.0) * dy[t].float()).to(DT[st])
                p = dy[t].double() * ys[r].double()
                rw[t, j], mag[t, j] = p.sum(), p.abs().sum()
    assert torch.equal(dys.cpu(), want)
    if with_ys:
        assert ((dw.cpu().double() - rw).abs() <= (H + 1) * 2.0 ** -24 * mag).all()


def test_gradients_against_differences(ctx):
    """<combine(dispatch(x) scaled per row), dy> against central differences in 64 bits over x and the weights: the
    map is linear in each, so a difference of any step equals the gradient up to f32 rounding."""
    T, top_k, E, H = 12, 3, 5, 24
    idx = routes(2, T, top_k, E, "holes")
    rows = make(ctx, idx, E, 4)
    _, row_of, _ = ref_sort(idx, E, 4, rows.R)
    g = gen(8)
    x, w, dy = (torch.randn(s, generator=g) for s in ((T, H), (T, top_k), (T, H)))
    xs = torch.zeros((rows.R, H), device=DEV)
    ctx.moe_dispatch(x.to(DEV), rows, xs)
    dys, dw = torch.zeros((rows.R, H), device=DEV), torch.zeros((T, top_k), device=DEV)
    ctx.moe_combine_backward(dy.to(DEV), xs, rows, w.to(DEV), dys, dw)
    dx = torch.zeros((T, H), device=DEV)
    ctx.moe_combine(dys, rows, None, dx)

    def loss(x, w):
        live = torch.from_numpy(row_of >= 0)
        return ((torch.where(live, w, 0.0).sum(1, keepdim=True) * x) * dy.double()).sum()
    for t, h in ((0, 0), (5, 7), (11, 23)):
        d = torch.zeros_like(x, dtype=torch.float64)
        d[t, h] = 0.5
        num = loss(x.double() + d, w.double()) - loss(x.double() - d, w.double())
        assert abs(float(num) - float(dx[t, h])) <= 1e-5 * (1 + abs(float(num)))
    for t, j in ((0, 0), (5, 2), (11, 1)):
        d = torch.zeros_like(w, dtype=torch.float64)
        d[t, j] = 0.5
        num = loss(x.double(), w.double() + d) - loss(x.double(), w.double() - d)
        assert abs(float(num) - float(dw[t, j])) <= 1e-5 * (1 + abs(float(num)))


def test_the_ternary_layers_routes(ctx):
    """frx_moe_ternary_ffn's routes, sorted: rows sent out and combined with its weights (which sum to one) give x
    back."""
    from ferrisres_amd import synth
    from _gpu import dev_f32, dev_u32
    T, H, I, E, k = 40, 128, 64, 8, 2
    g = gen(1)
    x = torch.randn((T, H), generator=g).to(DEV)
    router = torch.randn((E, H), generator=g).to(DEV)

    def mats(n, c, name):
        ts = [synth.ternary_uniform("route/mats", f"{name}{e}", n, c) for e in range(E)]
        return [dev_u32(synth.pack_rows_u32(t)) for t in ts], [dev_f32(np.full(n, 0.1, np.float32)) for _ in ts]
    (wg, sg), (wu, su), (wd, sd) = mats(I, H, "g"), mats(I, H, "u"), mats(H, I, "d")
    y = torch.empty((T, H), device=DEV)
    idx, w = torch.empty((T, k), dtype=torch.int32, device=DEV), torch.empty((T, k), device=DEV)
    ctx.moe_ternary_ffn(x, router, wg, sg, wu, su, wd, sd, y, top_k=k, topk_idx=idx, topk_w=w)
    rows = frx.MoeRows.empty(T, k, E, 1)
    ctx.moe_sort(idx, rows)
    xs, back = torch.empty((rows.R, H), device=DEV), torch.empty((T, H), device=DEV)
    ctx.moe_dispatch(x, rows, xs)
    ctx.moe_combine(xs, rows, w, back)
    off = rows.offsets.cpu().numpy()
    # each expert's ternary FFN over its rows, as a caller with its own experts runs it, then the combination
    ys = torch.empty((rows.R, H), device=DEV)
    for e in range(E):
        a, b = int(off[e]), int(off[e + 1])
        if b > a:
            ctx.ternary_ffn(xs[a:b], wg[e], sg[e], wu[e], su[e], wd[e], sd[e], ys[a:b])
    mine = torch.empty((T, H), device=DEV)
    ctx.moe_combine(ys, rows, w, mine)
    assert (back - x).abs().max() <= 4 * 2.0 ** -24 * x.abs().max() * 2
    # two paths of one layer, each within 1e-3 of the reference (the framework's parity bound)
    assert (mine - y).abs().max() <= 2e-3 * y.abs().max()


@pytest.mark.parametrize("T,top_k,E", [(5, 2, 4), (90, 2, 4), (300, 1, 3)])
def test_training_step_of_an_expert_layer(ctx, T, top_k, E):
    """Sort, quantise, dispatch, the experts' product, combine; then back through all of them: outputs and gradients
    against 64 bits over the values that the codes stand for."""
    H, N = 160, 96
    idx = routes(T, T, top_k, E, "holes")
    rows = make(ctx, idx, E, 128)
    off, row_of, slot_of = ref_sort(idx, E, 128, rows.R)
    g = gen(T)
    x, dy = torch.randn((T, H), generator=g), torch.randn((T, N), generator=g)
    w = torch.softmax(torch.randn((T, top_k), generator=g), 1)
    W = 0.1 * torch.randn((E, N, H), generator=g)
    X, DY, Wd = x.to(DEV), dy.to(DEV), w.to(DEV)
    wq, ws, wtq, wts = [], [], [], []
    for e in range(E):
        q, s = quantize(ctx, W[e].to(DEV), frx.FP8_TILES, E4M3)[1:3]
        qt, st = quantize(ctx, W[e].to(DEV), frx.FP8_TILES_T, E4M3)[1:3]
        wq.append(q), ws.append(s), wtq.append(qt), wts.append(st)
    new = lambda *s: torch.zeros(s, device=DEV)  # noqa: E731
    xs, ys, y = new(rows.R, H), new(rows.R, N), new(T, N)
    ctx.moe_dispatch(X, rows, xs)
    _, aq, asc, _ = quantize(ctx, xs, frx.FP8_ROWS, E4M3)
    ctx.fp8_linear_grouped(aq, asc, wq, ws, rows.offsets, ys)
    ctx.moe_combine(ys, rows, Wd, y)
    dys, dweight, dxs, dx, dw = new(rows.R, N), new(T, top_k), new(rows.R, H), new(T, H), new(E, N, H)
    ctx.moe_combine_backward(DY, ys, rows, Wd, dys, dweight)
    _, dq, dsc, _ = quantize(ctx, dys, frx.FP8_ROWS, E5M2)
    ctx.fp8_linear_grouped(dq, dsc, wtq, wts, rows.offsets, dxs)
    ctx.moe_combine(dxs, rows, None, dx)
    _, dtq, dts, _ = quantize(ctx, dys, frx.FP8_COLS, E5M2)
    _, xtq, xts, _ = quantize(ctx, xs, frx.FP8_COLS, E4M3)
    ctx.fp8_grad_weight_grouped(dtq, dts, xtq, xts, rows.offsets, dw)

    def val(q, s, tiles=False):
        q, s = q.cpu().double(), s.cpu().double().repeat_interleave(128, 1)
        if tiles:
            s = s.repeat_interleave(128, 0)[:q.shape[0]]
        return q * s[:, :q.shape[1]]
    A, D, DT_, XT = val(aq, asc), val(dq, dsc), val(dtq, dts), val(xtq, xts)
    r_ys, r_dxs = torch.zeros((rows.R, N), dtype=torch.float64), torch.zeros((rows.R, H), dtype=torch.float64)
    rel = lambda a, b: float((a.cpu().double() - b).norm() / (b.norm() + 1e-30))  # noqa: E731
    for e in range(E):
        i, j = off[e], off[e + 1]
        we = val(wq[e], ws[e], True)
        r_ys[i:j] = A[i:j] @ we.t()
        r_dxs[i:j] = D[i:j, :N] @ we[:, :H]
        assert rel(dw[e], DT_[:, i:j] @ XT[:, i:j].t()) <= 300 * 2.0 ** -24
    r_y, r_dx = torch.zeros((T, N), dtype=torch.float64), torch.zeros((T, H), dtype=torch.float64)
    r_w = torch.zeros((T, top_k), dtype=torch.float64)
    for t in range(T):
        for j in range(top_k):
            r = row_of[t, j]
            if r >= 0:
                r_y[t] += w[t, j].double() * r_ys[r]
                r_dx[t] += r_dxs[r]
                r_w[t, j] = (dy[t].double() * r_ys[r]).sum()
    # sums of at most 160 terms and three more roundings, of terms of both signs: 300 roundings in the norm
    for got, want in ((y, r_y), (dx, r_dx), (dweight, r_w)):
        assert rel(got, want) <= 300 * 2.0 ** -24


def test_captured_and_replayed(ctx):
    """Sort to combination and back in a graph, replayed on changing routes between eager calls."""
    T, top_k, E, H = 700, 4, 16, 256
    c = frx.Context(0)
    side = torch.cuda.Stream()
    c.set_stream(side)
    idxs = [torch.from_numpy(routes(s, T, top_k, E, "holes")).to(DEV) for s in range(3)]
    idx = idxs[0].clone()
    rows = frx.MoeRows.empty(T, top_k, E, 16)
    x, w = torch.randn((T, H), device=DEV), torch.rand((T, top_k), device=DEV)
    xs, y = torch.zeros((rows.R, H), device=DEV), torch.zeros((T, H), device=DEV)
    dys, dw = torch.zeros((rows.R, H), device=DEV), torch.zeros((T, top_k), device=DEV)

    def body():
        c.moe_sort(idx, rows)
        c.moe_dispatch(x, rows, xs)
        c.moe_combine(xs, rows, w, y)
        c.moe_combine_backward(x, xs, rows, w, dys, dw)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        body()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        body()
    for r in range(6):
        idx.copy_(idxs[r % 3])
        for t in (xs, y, dys, dw):
            t.fill_(-2.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (rows.offsets, rows.row_of, rows.slot_of, xs, y, dys, dw)]
        for t in (xs, y, dys, dw):
            t.fill_(-2.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            body()
        torch.cuda.synchronize()
        for a, b in zip(got, (rows.offsets, rows.row_of, rows.slot_of, xs, y, dys, dw)):
            assert torch.equal(a, b), f"replay {r}"
    del g
    c.close()


def test_first_sort_under_capture(ctx):
    """A fresh context captured at once at a size that asks for a workspace."""
    T, top_k, E = 9000, 2, 64
    idx = routes(1, T, top_k, E, "holes")
    dev = torch.from_numpy(idx).to(DEV)
    c = frx.Context(0)
    side = torch.cuda.Stream()
    c.set_stream(side)
    rows = frx.MoeRows.empty(T, top_k, E, 1)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        c.moe_sort(dev, rows)
    off, row_of, slot_of = ref_sort(idx, E, 1, rows.R)
    for _ in range(3):
        rows.row_of.fill_(5)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert np.array_equal(rows.offsets.cpu().numpy(), off)
        assert np.array_equal(rows.row_of.cpu().numpy(), row_of)
        assert np.array_equal(rows.slot_of.cpu().numpy(), slot_of)
    del g
    c.close()


def test_refusals(ctx):
    new = lambda *s: torch.zeros(s, dtype=torch.int32, device=DEV)  # noqa: E731
    with pytest.raises(frx.FrxError):
        ctx.moe_sort(new(4, 2), frx.MoeRows(8, 1, new(9), new(4, 2), new(7)))  # too few rows
    with pytest.raises(frx.FrxError):
        ctx.moe_sort(new(4, 2), frx.MoeRows(8, 3, new(9), new(4, 2), new(100)))  # align
    with pytest.raises(frx.FrxError):
        ctx.moe_sort(new(4, 2), frx.MoeRows(65, 1, new(66), new(4, 2), new(100)))
    with pytest.raises(frx.FrxError):
        frx.MoeRows(8, 1, new(8), new(4, 2), new(8))
    rows = frx.MoeRows.empty(4, 2, 8, 1)
    ctx.moe_sort(new(4, 2), rows)
    with pytest.raises(frx.FrxError):
        ctx.moe_sort(new(4, 3), rows)
    with pytest.raises(TypeError):
        ctx.moe_sort(torch.zeros((4, 2), dtype=torch.int64, device=DEV), rows)
    f = lambda *s: torch.zeros(s, device=DEV)  # noqa: E731
    for call in (lambda: ctx.moe_dispatch(f(4, 8), rows, f(7, 8)),
                 lambda: ctx.moe_dispatch(f(4, 8).to(torch.uint8)[:, :3].contiguous(), rows, f(8, 3).to(torch.uint8)),
                 lambda: ctx.moe_dispatch(f(8, 8)[::2], rows, f(8, 8)),
                 lambda: ctx.moe_combine(f(8, 8), rows, f(4, 3), f(4, 8)),
                 lambda: ctx.moe_combine(f(8, 7), rows, None, f(4, 8)),
                 lambda: ctx.moe_combine_backward(f(4, 8), f(8, 8), rows, None, f(8, 8), None)):
        with pytest.raises(frx.FrxError):
            call()
    with pytest.raises(TypeError):
        ctx.moe_combine(f(8, 8).half(), rows, None, f(4, 8))


@pytest.mark.parametrize("T,top_k,E,align,how", [(700001, 2, 5, 128, "holes"), (1048577, 1, 64, 1, "any")])
def test_sort_of_very_many(ctx, T, top_k, E, align, how):
    """More chunks of slots than workgroups that count them."""
    idx = routes(T + E, T, top_k, E, how)
    rows = make(ctx, idx, E, align, extra=1000)
    flat = np.where((idx >= 0) & (idx < E), idx, E).reshape(-1)
    order = np.argsort(flat, kind="stable")
    count = np.bincount(flat, minlength=E + 1)[:E]
    off = np.concatenate([[0], np.cumsum(-(-count // align) * align)])
    row_of, slot_of = np.full(T * top_k, -1, np.int64), np.full(rows.R, -1, np.int64)
    at = 0
    for e in range(E):
        slots = order[at:at + count[e]]
        at += count[e]
        row_of[slots] = off[e] + np.arange(count[e])
        slot_of[off[e]:off[e] + count[e]] = slots
    assert np.array_equal(rows.offsets.cpu().numpy(), off)
    assert np.array_equal(rows.row_of.cpu().numpy().reshape(-1), row_of)
    assert np.array_equal(rows.slot_of.cpu().numpy(), slot_of)


def test_sizes_past_a_launch_are_refused(ctx):
    """Rows and columns of more than a launch holds, before anything is read."""
    rows = frx.MoeRows.empty(4, 2, 3, 1, device=DEV)
    t = torch.zeros((64,), device=DEV)
    p, L, h = t.data_ptr(), frx.lib(), ctx._h
    small = rows._c
    shape = L.frx_moe_combine(h, p, 0, ctypes.byref(small), None, p, 0, 0)
    assert shape != 0
    assert L.frx_moe_combine(h, p, 0, ctypes.byref(small), None, p, 0, 1 << 24) == shape
    assert L.frx_moe_combine_backward(h, p, 0, None, 0, ctypes.byref(small), None, p, None, 1 << 24) == shape
    big = type(small).from_buffer_copy(small)
    big.T, big.R = 1 << 23, 1 << 24
    assert L.frx_moe_sort(h, p, ctypes.byref(big)) == shape
    assert L.frx_moe_dispatch(h, p, 4, ctypes.byref(big), p) == shape
    torch.cuda.synchronize()
    assert not t.any()
