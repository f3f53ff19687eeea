"""The expert layer for a few tokens (frx_fp4_moe_ffn) on inputs for which every step has one right f32 result, over the
shapes that reach each of its kernels: compared bit for bit, so that a lost plane of an activation or a lost or doubled
block of K cannot hide in a tolerance.

Both activations are the identity from 20 on: exp(-20) < 2^-28 beside 1, and tanh of 0.79 * (20 + 0.04 * 20^3) is 1."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp4_kernels import LAYERS
from _fp4_ref import DT, TABLE, pack, up
from _gpu import DEV, host

HALF_, ONE, TWO, FOUR = 1, 2, 4, 6  # code numbers of powers of two


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def layer(code, byte):
    """One matrix of all experts: (codes, scales, values) of code numbers [E][n][k], scale bytes [E][n][k / 32]; 255 behind
    the bytes of a row."""
    E, n, k = code.shape
    pad = np.full((E, n, up(k, 128) // 32), 255, np.uint8)
    pad[:, :, :k // 32] = byte
    v = TABLE[code] * np.repeat(np.ldexp(1.0, byte.astype(np.int64) - 127), 32, axis=-1)
    return pack(code.reshape(E * n, k)).reshape(E, n, k // 2), pad, v


def on_dev(w):
    return [torch.from_numpy(t).to(DEV) for code, pad, _ in w for t in (code, pad)]


def distinct(rng, T, E, top_k):
    return np.stack([rng.permutation(E)[:top_k] for _ in range(T)]).astype(np.int32)


# ---- whole numbers: every block of K decides ------------------------------------------


def whole_codes(rng, E, n, k, a_block, signed):
    """a_block codes of 1 or 2 in every block of 32, zeros elsewhere."""
    place = rng.random((E, n, k // 32, 32)).argsort(axis=-1) < a_block
    code = np.where(place, rng.choice((ONE, TWO), place.shape), 0)
    if signed:
        code = np.where(place & (rng.random(place.shape) < 0.5), code + 8, code)
    return layer(code.reshape(E, n, k).astype(np.uint8), np.full((E, n, k // 32), 127, np.uint8))


def whole_case(T, H, I, E, top_k):
    rng = np.random.default_rng(T + H + I)
    w = [whole_codes(rng, E, I, H, -(-20 // (H // 32)), False), whole_codes(rng, E, I, H, 1, True),
         whole_codes(rng, E, H, I, 1, True)]
    x = rng.integers(1, 4, (T, H)).astype(np.float64)
    idx = distinct(rng, T, E, top_k)
    wt = rng.choice((0.5, 1.0, 2.0), (T, top_k))
    return x, w, idx, wt


def whole_reference(x, wv, idx, wt):
    """y, and the sum of what its terms' magnitudes can reach."""
    y, most = np.zeros(x.shape), np.zeros(x.shape)
    for e in range(len(wv[0])):
        t, j = np.nonzero(idx == e)
        if len(t):
            g, u = x[t] @ wv[0][e].T, x[t] @ wv[1][e].T
            assert g.min() >= 20
            h = g * u * wt[t, j, None]
            np.add.at(y, t, h @ wv[2][e].T)
            np.add.at(most, t, np.abs(h) @ np.abs(wv[2][e]).T + (x[t] @ np.abs(wv[1][e]).T).max())
    return y, most


@pytest.mark.parametrize("T,H,I,E,top_k", LAYERS)
def test_a_block_left_out_shows(T, H, I, E, top_k):
    """What the next test can tell apart, on the CPU: leaving any block of a matrix out, here the first, the last and one
    between, changes the layer's result; every sum is of multiples of 1/2 below 2^23, whatever its order."""
    x, w, idx, wt = whole_case(T, H, I, E, top_k)
    wv = [v for _, _, v in w]
    y, most = whole_reference(x, wv, idx, wt)
    assert most.max() < 2 ** 23
    for m in range(3):
        n = wv[m].shape[2] // 32
        for b in sorted({0, n - 1, *np.random.default_rng(m).integers(0, n, 1)}):
            less = [v.copy() if i == m else v for i, v in enumerate(wv)]
            if m == 0:  # (what is left may be an activation's argument below 20: g as it is, then)
                less[0][:, :, 32 * b:32 * b + 32] = 0
                got = np.zeros_like(y)
                for e in range(E):
                    t, j = np.nonzero(idx == e)
                    np.add.at(got, t, (x[t] @ less[0][e].T * (x[t] @ wv[1][e].T) * wt[t, j, None]) @ wv[2][e].T)
            else:
                less[m][:, :, 32 * b:32 * b + 32] = 0
                got = whole_reference(x, less, idx, wt)[0]
            assert (got != y).any(), (m, b)


@pytest.mark.gpu
@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("T,H,I,E,top_k", LAYERS)
def test_whole_numbers(ctx, T, H, I, E, top_k, xt, yt):
    x, w, idx, wt = whole_case(T, H, I, E, top_k)
    want = torch.from_numpy(whole_reference(x, [v for _, _, v in w], idx, wt)[0]).to(DT[yt])
    y = torch.full((T, H), float("nan"), dtype=DT[yt], device=DEV)
    act = frx.ACT_GELU_TANH if T % 2 == 0 else frx.ACT_SILU
    ctx.fp4_moe_ffn(torch.from_numpy(x).to(DT[xt]).to(DEV), None, *on_dev(w), y, torch.from_numpy(idx).to(DEV),
                    torch.from_numpy(wt).float().to(DEV), act=act)
    assert torch.equal(y.cpu(), want)


# ---- 24 bits: every plane decides -----------------------------------------------------


def one_hot(rng, E, n, k, positive):
    """A code of a power of two in each row, its blocks taken in turn; scales of their own."""
    col = (np.arange(E * n) % (k // 32)) * 32 + rng.integers(0, 32, E * n)
    number = rng.choice((HALF_, ONE, TWO, FOUR), E * n)
    if not positive:
        number = number + 8 * rng.integers(0, 2, E * n)
    code = np.zeros((E * n, k), np.uint8)
    code[np.arange(E * n), col] = number
    byte = rng.integers(124, 131, (E * n, k // 32)).astype(np.uint8)
    byte[np.arange(E * n), col // 32] = rng.integers(128, 131, E * n)
    v = TABLE[number] * np.ldexp(1.0, byte[np.arange(E * n), col // 32].astype(np.int64) - 127)
    return layer(code.reshape(E, n, k), byte.reshape(E, n, -1)), col.reshape(E, n), v.reshape(E, n).astype(np.float32)


def planes_case(T, H, I, E, top_k, xt):
    rng = np.random.default_rng(T + H + I + top_k)
    mats = [one_hot(rng, E, I, H, True), one_hot(rng, E, I, H, False), one_hot(rng, E, H, I, False)]
    x = rng.integers(1 << 23, 1 << 24, (T, H)).astype(np.float32) * np.float32(2.0 ** -18)  # 24 bits from 32 to 64
    if xt == "bf16":
        x = torch.from_numpy(x).bfloat16().float().numpy()
    idx = distinct(rng, T, E, top_k)
    wt = (rng.integers(1 << 23, 1 << 24, (T, top_k)).astype(np.float32) * np.float32(2.0 ** -24))
    return x, mats, idx, wt


def planes_reference(x, mats, idx, wt, cut=lambda h: h):
    """y in f32: one product to a sum, so that what is rounded is the product of g and u, its product with the weight, and
    the sum over the routes in order."""
    y = np.zeros(x.shape, np.float32)
    (_, kg, cg), (_, ku, cu), (_, kd, cd) = mats
    for t in range(len(x)):
        for j, e in enumerate(idx[t]):
            g, u = x[t, kg[e]] * cg[e], x[t, ku[e]] * cu[e]
            h = cut(g * u * wt[t, j])
            y[t] += h[kd[e]] * cd[e]
    return y


def cut(v, bits):
    return (v.view(np.uint32) & np.uint32(0xFFFFFFFF << bits & 0xFFFFFFFF)).view(np.float32)


@pytest.mark.parametrize("T,H,I,E,top_k", LAYERS)
def test_a_plane_left_out_shows(T, H, I, E, top_k):
    """What the next test can tell apart, on the CPU: the last 8 bits of x, or of the intermediate, change the result."""
    x, mats, idx, wt = planes_case(T, H, I, E, top_k, "f32")
    y = planes_reference(x, mats, idx, wt)
    assert (y != 0).all()
    assert (planes_reference(cut(x, 8), mats, idx, wt) != y).mean() > 0.5
    assert (planes_reference(x, mats, idx, wt, cut=lambda h: cut(h, 8)) != y).mean() > 0.5


@pytest.mark.gpu
@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("T,H,I,E,top_k", LAYERS)
def test_every_bit(ctx, T, H, I, E, top_k, xt, yt):
    """All 24 bits of x, of the intermediate and of the weights reach y; a bf16 y is the f32 one, rounded once."""
    x, mats, idx, wt = planes_case(T, H, I, E, top_k, xt)
    want = torch.from_numpy(planes_reference(x, mats, idx, wt)).to(DT[yt])
    y = torch.full((T, H), float("nan"), dtype=DT[yt], device=DEV)
    act = frx.ACT_GELU_TANH if T % 2 else frx.ACT_SILU
    ctx.fp4_moe_ffn(torch.from_numpy(x).to(DT[xt]).to(DEV), None, *on_dev([m[0] for m in mats]), y,
                    torch.from_numpy(idx).to(DEV), torch.from_numpy(wt).to(DEV), act=act)
    assert torch.equal(y.cpu(), want)


@pytest.mark.gpu
@pytest.mark.parametrize("xt", ["bf16", "f32"])
@pytest.mark.parametrize("T,H,I,E,top_k", LAYERS)
def test_a_bf16_y_is_the_f32_one_rounded(ctx, T, H, I, E, top_k, xt):
    """Any values: whatever the sums round, y is rounded once more."""
    rng = np.random.default_rng(T + H)
    w = [layer(rng.integers(0, 16, (E, n, k)).astype(np.uint8), rng.integers(119, 123, (E, n, k // 32)).astype(np.uint8))
         for n, k in ((I, H), (I, H), (H, I))]
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(DT[xt]).to(DEV)
    idx, wt = torch.from_numpy(distinct(rng, T, E, top_k)).to(DEV), torch.from_numpy(rng.random((T, top_k), np.float32)).to(DEV)
    y, z = torch.zeros((T, H), device=DEV), torch.zeros((T, H), dtype=torch.bfloat16, device=DEV)
    ctx.fp4_moe_ffn(x, None, *on_dev(w), y, idx, wt)
    ctx.fp4_moe_ffn(x, None, *on_dev(w), z, idx, wt)
    assert torch.equal(z, y.bfloat16()) and y.any()


# ---- either end of the range ----------------------------------------------------------


def range_case(H, I, xt, end):
    """x [2][H] and the three matrices: gate takes column 0 of x, row i of up column i % 8 under a scale that suits it, row
    n of down row n % I of the intermediate and brings it back to an ordinary size."""
    rng = np.random.default_rng(H + I)
    m = lambda: rng.integers(1 << 23, 1 << 24, 2) * 2.0 ** -23  # noqa: E731  (24 bits, 1 to 2)
    x = np.zeros((2, H))
    if end == "small":
        x[:, 0] = 64.0
        x[:, 1] = m() * 2.0 ** 126
        x[:, 2] = rng.integers(1, 128, 2) * 2.0 ** -133  # a bf16's denormal numbers
        x[:, 3] = rng.integers(1 << 20, 1 << 23, 2) * 2.0 ** -148  # f32's
        x[:, 4], x[:, 5], x[:, 6], x[:, 7] = m() * 2.0 ** -118, m(), m() * 8, m() * 2.0 ** -100
        scale = {1: (0, 1, 2, 3), 2: (247,), 3: (247,), 4: (240, 128), 5: (2, 5), 6: (10, 127), 7: (127,)}
    else:  # the intermediate below 2^128
        x[:, 0] = 2.0 ** 64
        scale = {1: (247,), 2: (130, 160), 3: (127,), 4: (100,), 5: (70,), 6: (3,), 7: (190,)}
        for c, b in scale.items():
            x[:, c] = m() * 2.0 ** min(126, 127 - 64 - (max(b) - 127) - 2)
    t = torch.from_numpy(x).to(DT[xt])
    x = t.double().numpy()
    cols = np.arange(I) % 8
    byte = np.array([rng.choice(scale.get(c, (127,))) for c in cols])
    byte[cols == 0] = 60  # (column 0 is gate's)
    number = rng.choice((HALF_, ONE, TWO, FOUR), I)
    with np.errstate(over="raise"):
        h = (x[:, :1] * (x[:, cols] * TABLE[number] * np.ldexp(1.0, byte - 127))).astype(np.float32)
    r = np.arange(H) % I
    size = np.abs(h[0, r].astype(np.float64))
    back = np.clip(127 - np.frexp(np.where(size > 0, size, 1.0))[1], 0, 252)
    want = (h[:, r] * np.ldexp(1.0, back - 127)).astype(np.float32)

    def matrix(n, k, col, number, byte):
        code, by = np.zeros((1, n, k), np.uint8), np.full((1, n, k // 32), 127, np.uint8)
        code[0, np.arange(n), col] = number
        by[0, np.arange(n), col // 32] = byte
        return layer(code, by)

    return t, [matrix(I, H, 0 * cols, ONE, 127), matrix(I, H, cols, number, byte), matrix(H, I, r, ONE, back)], h, want


@pytest.mark.parametrize("xt", ["bf16", "f32"])
@pytest.mark.parametrize("end", ["small", "large"])
def test_what_the_range_holds(end, xt):
    """On the CPU: the intermediates reach the ends that the next test is about, and y is finite and not zero."""
    _, _, h, want = range_case(32, 32, xt, end)
    size = np.abs(h)
    assert np.isfinite(want).all() and (want != 0).all()
    assert size.max() > 2.0 ** 126 if end == "large" else size.min() < 2.0 ** -110


@pytest.mark.gpu
@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("end", ["small", "large"])
@pytest.mark.parametrize("H,I", [(32, 32), (2080, 96), (4128, 2080)])
def test_either_end_of_the_range(ctx, H, I, end, xt, yt):
    """Weights, activations and intermediates that bf16 holds as denormal numbers or not at all, and the largest
    intermediates: nothing of an f32 number is lost on the way but 2^-149."""
    x, w, _, want = range_case(H, I, xt, end)
    y = torch.full((2, H), float("nan"), dtype=DT[yt], device=DEV)
    ctx.fp4_moe_ffn(x.to(DEV), None, *on_dev(w), y, torch.zeros((2, 1), dtype=torch.int32, device=DEV),
                    torch.ones((2, 1), device=DEV))
    assert torch.equal(y.cpu(), torch.from_numpy(want).to(DT[yt]))


# ---- past 4 GiB -----------------------------------------------------------------------


@pytest.mark.gpu
@pytest.mark.parametrize("xt,yt", [("f32", "f32"), ("bf16", "bf16")])
def test_a_long_expert_bit_for_bit(ctx, xt, yt):
    """Gate, up and down of more than 2^32 bytes each, one code to a row: row i of gate and of up takes a column of x of its
    own, row n of down a column of the intermediate, the rows together one of every 135 columns. A row whose address wrapped
    at 4 GiB would take another's, a slice left out would give zeros, and no value of y is one."""
    H, I = 8192, 32 * 34400
    g = torch.Generator(device=DEV).manual_seed(3)
    draw = lambda lo, hi, n: torch.randint(lo, hi, (n,), device=DEV, generator=g)  # noqa: E731

    def matrix(n, k, col, number):
        code = torch.zeros((1, n, k // 2), dtype=torch.uint8, device=DEV)
        code[0, torch.arange(n, device=DEV), col // 2] = torch.where(col % 2 == 1, number * 16, number).to(torch.uint8)
        return code, torch.full((1, n, k // 32), 127, dtype=torch.uint8, device=DEV)

    x = (draw(1 << 23, 1 << 24, H).float() * 2.0 ** -18).to(DT[xt])  # 32 to 64
    value = torch.tensor(TABLE, device=DEV, dtype=torch.float32)
    powers = torch.tensor([ONE, TWO, FOUR], device=DEV)
    kg, ku, ng, nu = draw(0, H, I), draw(0, H, I), powers[draw(0, 3, I)], powers[draw(0, 3, I)] + 8 * draw(0, 2, I)
    part = torch.arange(H, device=DEV) * I // H
    kd, nd = torch.clamp_max(part + draw(0, I // H, H), I - 1), powers[draw(0, 3, H)]
    kd[H - 1] = I - 1
    w = [t for m in (matrix(I, H, kg, ng), matrix(I, H, ku, nu), matrix(H, I, kd, nd)) for t in m]
    assert all(w[m].numel() > 1 << 32 for m in (0, 2, 4))
    xf = x.float()
    h = (xf[kg] * value[ng]) * (xf[ku] * value[nu])  # one f32 rounding
    # what a wrapped row would give differs: rows 2^32 bytes apart, for every row past the mark
    far = (1 << 32) // (H // 2)
    assert bool((h[far:] != h[:I - far]).float().mean() > 0.99) and int((kd >= far).sum()) > 300
    want = h[kd] * value[nd]
    far = -(-(1 << 32) // (I // 2))
    assert bool((want[far:] != want[:H - far]).float().mean() > 0.99)
    assert bool((want != 0).all())
    y = torch.full((1, H), float("nan"), dtype=DT[yt], device=DEV)
    ctx.fp4_moe_ffn(x[None], None, *w, y, torch.zeros((1, 1), dtype=torch.int32, device=DEV),
                    torch.ones((1, 1), device=DEV))
    assert torch.equal(y[0], want.to(DT[yt]))
