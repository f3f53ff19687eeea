"""The expert layer for a few tokens (frx_fp4_moe_ffn) against its formula in 64 bits.

Tolerance, each step's roundings relative to what enters it (u = 2^-24). gate and up: H products in f32 sums, three
planes of an f32 x among them: 3 H u of the sum of the magnitudes. act: silu's exponential, sum and quotient within 16 u
of the value, gelu's tanh within 8 u of |g| / 2 beside the 1; both change by at most 1.13 of a change of g. h = act(g) * up *
weight: 4 u, and 2^-17 of it for a bf16 y. down: 3 I u for each route, of the sum of the magnitudes. Half a step of y."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp4_ref import DT, HALF, pack, random_codes, values
from _gpu import DEV, host

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def weights(rng, E, I, H, lo=119, hi=123):
    """[(codes, scales) on the device as stacked tensors, values in f64] of gate, up and down."""
    out = []
    for n, k in ((I, H), (I, H), (H, I)):
        code, byte = random_codes(rng, E * n, k, lo, hi)
        out.append(((torch.from_numpy(pack(code)).to(DEV).view(E, n, -1), torch.from_numpy(byte).to(DEV).view(E, n, -1)),
                    values(code, byte).reshape(E, n, k)))
    return out


def act64(g, act):
    if act == frx.ACT_SILU:
        return g / (1 + np.exp(-g)), 16 * U * np.abs(g / (1 + np.exp(-g)))
    t = 0.7978845608028654 * (g + 0.044715 * g ** 3)
    return 0.5 * g * (1 + np.tanh(t)), 16 * U * np.abs(g)


def reference(x, wv, idx, wt, act, yt):
    """(y, bound) in f64."""
    T, H = x.shape
    E, I, _ = wv[0].shape
    y, bound = np.zeros((T, H)), np.zeros((T, H))
    for t in range(T):
        for j in range(idx.shape[1]):
            e = idx[t, j]
            if not 0 <= e < E:
                continue
            g, u = wv[0][e] @ x[t], wv[1][e] @ x[t]
            dg, du = 3 * H * U * (np.abs(wv[0][e]) @ np.abs(x[t])), 3 * H * U * (np.abs(wv[1][e]) @ np.abs(x[t]))
            a, da = act64(g, act)
            da = da + 1.13 * dg
            h = a * u * wt[t, j]
            dh = (da * np.abs(u) + np.abs(a) * du + da * du) * abs(wt[t, j]) + (4 * U + (2.0 ** -17 if yt == "bf16" else 0)) * np.abs(h)
            y[t] += wv[2][e] @ h
            bound[t] += np.abs(wv[2][e]) @ (dh + 3 * I * U * np.abs(h))
    return y, 1.01 * bound + HALF[DT[yt]] * np.abs(y) + 2.0 ** -133


def routes(rng, T, E, top_k):
    idx = np.stack([rng.permutation(E)[:top_k] for _ in range(T)]).astype(np.int32)
    return idx, rng.random((T, top_k)).astype(np.float32)


def inputs(rng, T, H, xt):
    return torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(DT[xt])


def check(y, ref, bound):
    err = np.abs(host(y).astype(np.float64) - ref)
    assert (err <= bound).all(), (err / bound).max()


CASES = [(1, 32, 32, 1, 1), (1, 256, 160, 4, 2), (2, 96, 288, 8, 8), (7, 416, 96, 16, 2), (16, 128, 128, 3, 1),
         (17, 1056, 64, 5, 2), (33, 64, 1056, 64, 6), (40, 160, 352, 2, 1), (64, 288, 96, 16, 4), (64, 32, 64, 1, 1)]


@pytest.mark.parametrize("xt,yt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("T,H,I,E,top_k", CASES)
def test_given_routes(ctx, T, H, I, E, top_k, xt, yt):
    """A sixteenth of the tokens is padding, some routes are dropped."""
    rng = np.random.default_rng(T + H)
    w = weights(rng, E, I, H)
    x = inputs(rng, T, H, xt)
    idx, wt = routes(rng, T, E, top_k)
    idx[T - T // 16:] = -1
    idx[rng.random(idx.shape) < 0.1] = E
    act = frx.ACT_GELU_TANH if T % 2 == 0 else frx.ACT_SILU
    y = torch.full((T, H), float("nan"), dtype=DT[yt], device=DEV)
    ctx.fp4_moe_ffn(x.to(DEV), None, *w[0][0], *w[1][0], *w[2][0], y, torch.from_numpy(idx).to(DEV),
                    torch.from_numpy(wt).to(DEV), act=act)
    check(y, *reference(x.double().numpy(), [v for _, v in w], idx, wt, act, yt))
    none = (idx < 0).all(1) | ((idx < 0) | (idx >= E)).all(1)
    assert not host(y)[none].any()


@pytest.mark.parametrize("xt,rt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("T,H,I,E,top_k", CASES)
def test_router(ctx, T, H, I, E, top_k, xt, rt):
    """The chosen experts, in order, and their softmax; the layer goes by them. Logits are drawn far enough apart
    (2^-10 beside an f32 sum's 2^-24 H) that no rounding swaps two."""
    rng = np.random.default_rng(T * 3 + H)
    w = weights(rng, E, I, H)
    x = inputs(rng, T, H, xt)
    router = torch.from_numpy(rng.standard_normal((E, H)).astype(np.float32) * H ** -0.5).to(DT[rt])
    logits = x.double().numpy() @ router.double().numpy().T
    order = np.argsort(-logits, axis=1, kind="stable")
    ranked = np.take_along_axis(logits, order, 1)
    clear = np.ones(T, bool) if E == 1 else (-np.diff(ranked, axis=1)[:, :top_k] > 2.0 ** -10).all(1)
    assert clear.sum() * 2 >= T or T < 4
    idx, wt = torch.full((T, top_k), -9, dtype=torch.int32, device=DEV), torch.zeros((T, top_k), device=DEV)
    y = torch.zeros((T, H), device=DEV)
    ctx.fp4_moe_ffn(x.to(DEV), router.to(DEV), *w[0][0], *w[1][0], *w[2][0], y, idx, wt)
    gi, gw = idx.cpu().numpy(), host(wt)
    assert np.array_equal(gi[clear], order[clear, :top_k])
    mag = np.abs(x.double().numpy()) @ np.abs(router.double().numpy()).T
    p = np.exp(ranked[:, :top_k] - ranked[:, :1])
    p /= p.sum(1, keepdims=True)
    # each logit is off by at most H u of its magnitudes, so a weight by twice that, 64 u for the exponentials and sum
    off = p * (2.1 * H * U * mag.max(1, keepdims=True) + 64 * U)
    assert (np.abs(gw - p)[clear] <= off[clear]).all()
    check(y, *reference(x.double().numpy(), [v for _, v in w], gi, gw, frx.ACT_SILU, "f32"))
    z = torch.zeros_like(y)  # routes that nobody takes, and lists of experts
    ctx.fp4_moe_ffn(x.to(DEV), router.to(DEV), *(list(t) for m in w for t in m[0]), z, top_k=top_k)
    assert torch.equal(y, z)


def test_router_ties_and_nan(ctx):
    """Equal logits go by index, zeros of both signs are equal, a NaN logit is below -inf's neighbours; a NaN token
    takes the first experts and spoils nobody else."""
    H, I, E = 32, 32, 6
    w = weights(np.random.default_rng(1), E, I, H)
    x = torch.zeros((4, H))
    x[0, 0] = x[2, 0] = 1.0
    x[3, 5] = float("nan")
    router = torch.zeros((E, H))
    router[:, 0] = torch.tensor([0.0, 2.0, -0.0, 2.0, float("nan"), 1.0])
    router[:, 1] = torch.tensor([-0.0, 0.0, 0.0, -0.0, 0.0, 0.0])
    idx, wt = torch.zeros((4, 4), dtype=torch.int32, device=DEV), torch.zeros((4, 4), device=DEV)
    y = torch.zeros((4, H), device=DEV)
    ctx.fp4_moe_ffn(x.to(DEV), router.to(DEV), *w[0][0], *w[1][0], *w[2][0], y, idx, wt)
    gi = idx.cpu().tolist()
    assert gi[0] == gi[2] == [1, 3, 5, 0]
    assert gi[1] == [0, 1, 2, 3]  # 0 * NaN is a NaN for expert 4
    assert gi[3] == [0, 1, 2, 3]
    assert torch.isfinite(y[:3]).all() and torch.isnan(y[3]).all()
    assert torch.allclose(wt[1].cpu(), torch.full((4,), 0.25), rtol=1e-6)


def test_the_same_expert_twice(ctx):
    rng = np.random.default_rng(5)
    w = weights(rng, 3, 64, 96)
    x = inputs(rng, 5, 96, "bf16")
    idx = np.array([[1, 1, 1], [0, 2, 0], [2, 2, -1], [-1, -1, -1], [0, 1, 2]], np.int32)
    wt = rng.random((5, 3)).astype(np.float32)
    y = torch.zeros((5, 96), device=DEV)
    ctx.fp4_moe_ffn(x.to(DEV), None, *w[0][0], *w[1][0], *w[2][0], y, torch.from_numpy(idx).to(DEV),
                    torch.from_numpy(wt).to(DEV))
    check(y, *reference(x.double().numpy(), [v for _, v in w], idx, wt, frx.ACT_SILU, "f32"))
    assert not y[3].any()


def test_nothing_routed_and_weights_of_zero(ctx):
    rng = np.random.default_rng(6)
    w = weights(rng, 2, 64, 64)
    x = inputs(rng, 20, 64, "f32").to(DEV)
    idx = torch.full((20, 2), -1, dtype=torch.int32, device=DEV)
    y = torch.full((20, 64), float("nan"), device=DEV)
    args = (*w[0][0], *w[1][0], *w[2][0], y)
    ctx.fp4_moe_ffn(x, None, *args, idx, torch.ones((20, 2), device=DEV))
    assert not y.any()
    y.fill_(float("nan"))
    ctx.fp4_moe_ffn(x, None, *args, idx.fill_(1), torch.zeros((20, 2), device=DEV))
    assert not y.any()


@pytest.mark.parametrize("xt", ["bf16", "f32"])
def test_a_bad_token_is_alone(ctx, xt):
    """An infinity, a NaN, the largest numbers in some tokens, padded ones among them: the others keep their bits."""
    rng = np.random.default_rng(7)
    w = weights(rng, 4, 96, 160)
    x = inputs(rng, 24, 160, xt)
    idx, wt = routes(rng, 24, 4, 2)
    idx[20:] = -1
    args = lambda v: (v.to(DEV), None, *w[0][0], *w[1][0], *w[2][0])  # noqa: E731
    ri, rw = torch.from_numpy(idx).to(DEV), torch.from_numpy(wt).to(DEV)
    y, z = torch.zeros((24, 160), device=DEV), torch.zeros((24, 160), device=DEV)
    ctx.fp4_moe_ffn(*args(x), y, ri, rw)
    x[3, 7], x[11, 100], x[21, 3], x[22] = float("inf"), float("nan"), float("nan"), float("inf")
    ctx.fp4_moe_ffn(*args(x), z, ri, rw)
    good = [t for t in range(24) if t not in (3, 11)]
    assert torch.equal(y[good], z[good])
    assert not torch.isfinite(z[[3, 11]]).any()


def test_scales_of_either_end(ctx):
    """A NaN scale spoils the tokens of its expert alone; the smallest scales of gate with large tokens lose nothing that
    f32 holds."""
    rng = np.random.default_rng(8)
    w = weights(rng, 3, 64, 64)
    x = inputs(rng, 6, 64, "f32")
    idx = np.array([[0], [1], [2], [1], [0], [2]], np.int32)
    wt = np.ones((6, 1), np.float32)
    w[2][0][1][1, 5, 1] = 255
    y = torch.zeros((6, 64), device=DEV)
    ctx.fp4_moe_ffn(x.to(DEV), None, *w[0][0], *w[1][0], *w[2][0], y, torch.from_numpy(idx).to(DEV),
                    torch.from_numpy(wt).to(DEV))
    bad = np.zeros((6, 64), bool)
    bad[[1, 3], 5] = True
    assert np.array_equal(np.isnan(host(y)), bad)
    w = weights(rng, 1, 64, 64)
    code, byte = random_codes(rng, 64, 64, 3, 12)  # values of 2^-125 to 2^-113
    gate = (torch.from_numpy(pack(code)).to(DEV).view(1, 64, -1), torch.from_numpy(byte).to(DEV).view(1, 64, -1))
    big = x * 2.0 ** 118
    up = (w[1][0][0], torch.clamp(w[1][0][1].int() - 118, 1, 254).to(torch.uint8))
    wv = [values(code, byte).reshape(1, 64, 64), w[1][1] * 2.0 ** -118, w[2][1]]
    ctx.fp4_moe_ffn(big.to(DEV), None, *gate, *up, *w[2][0], y, torch.zeros((6, 1), dtype=torch.int32, device=DEV),
                    torch.ones((6, 1), device=DEV))
    check(y, *reference(big.double().numpy(), wv, np.zeros((6, 1), int), wt, frx.ACT_SILU, "f32"))


@pytest.mark.parametrize("yt", ["bf16", "f32"])
def test_odd_offsets(ctx, yt):
    """x, router and y from an odd element on."""
    rng = np.random.default_rng(9)
    w = weights(rng, 4, 64, 96)
    x, router = inputs(rng, 3, 96, yt).to(DEV), inputs(rng, 4, 96, yt).to(DEV)
    off = lambda t: torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)  # noqa: E731
    y = torch.zeros((3, 96), dtype=DT[yt], device=DEV)
    z = off(y)
    ctx.fp4_moe_ffn(x, router, *w[0][0], *w[1][0], *w[2][0], y, top_k=2)
    ctx.fp4_moe_ffn(off(x), off(router), *w[0][0], *w[1][0], *w[2][0], z, top_k=2)
    assert torch.equal(y, z) and y.any()


@pytest.mark.parametrize("T", [1, 20])
def test_captured(T):
    """A first call under capture is refused; a captured one replays to the eager results on new inputs."""
    rng = np.random.default_rng(10)
    c, e = frx.Context(0), frx.Context(0)
    w = weights(rng, 4, 96, 64)
    x, router = inputs(rng, T, 64, "bf16").to(DEV), inputs(rng, 4, 64, "bf16").to(DEV)
    y, z = torch.zeros((T, 64), device=DEV), torch.zeros((T, 64), device=DEV)
    call = lambda ctx, o: ctx.fp4_moe_ffn(x, router, *w[0][0], *w[1][0], *w[2][0], o, top_k=2)  # noqa: E731
    side = torch.cuda.Stream()
    c.set_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        y.add_(0.0)
        with pytest.raises(frx.FrxError, match="captured") as err:
            call(c, y)
        assert err.value.kind == "Unsupported"
    del graph
    call(c, y)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        call(c, y)
    for _ in range(3):
        x.copy_(inputs(rng, T, 64, "bf16"))
        call(e, z)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, z) and y.any()
    del graph
    c.set_stream(None)
    c.close()
    e.close()
