"""What the 8-bit linears' entry points refuse on a device, before anything is launched."""
import pytest
import torch

import ferrisres_amd as frx
from _gpu import DEV
from test_gpu_fp8 import E4M3, E5M2

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def test_gradients_of_experts_lie_apart(ctx):
    """A list with one matrix twice, or with two that overlap, is refused and nothing is written; any order of
    matrices that lie apart is not."""
    N, K, R, E = 32, 48, 256, 3
    a, b = torch.zeros((N, R), device=DEV).to(E5M2), torch.zeros((K, R), device=DEV).to(E4M3)
    sa, sb = torch.ones((N, 2), device=DEV), torch.ones((K, 2), device=DEV)
    off = torch.tensor([0, 128, 128, 256], dtype=torch.int32, device=DEV)
    buf = torch.full((4 * N * K,), 7.0, device=DEV)
    at = lambda i: buf[i:i + N * K].view(N, K)  # noqa: E731
    for dw in ([at(0), at(N * K), at(0)], [at(0), at(N * K - 4), at(2 * N * K)], [at(2 * N * K), at(N * K), at(N * K + 4)]):
        with pytest.raises(frx.FrxError) as e:
            ctx.fp8_grad_weight_grouped(a, sa, b, sb, off, dw)
        assert e.value.kind == "Shape"
    torch.cuda.synchronize()
    assert (buf == 7.0).all()
    ctx.fp8_grad_weight_grouped(a, sa, b, sb, off, [at(2 * N * K), at(0), at(N * K)])
    torch.cuda.synchronize()
    assert not buf[:E * N * K].any() and (buf[E * N * K:] == 7.0).all()


def test_a_single_row_has_any_stride(ctx):
    """One token (one weight row) out of a matrix whose rows are of no multiple of 16 apart, in every operand."""
    k = 272
    g = torch.Generator().manual_seed(1)
    wide = torch.randn((3, k + 5), generator=g).to(DEV)
    x = wide[1:2, :k]
    q, s = torch.zeros((1, k), dtype=E4M3, device=DEV), torch.zeros((1, 3), device=DEV)
    ctx.fp8_quantize(x, frx.FP8_ROWS, q, s)
    raw = torch.zeros((2 * 1000003 + k,), dtype=torch.uint8, device=DEV).view(E4M3)
    q2 = raw.as_strided((1, k), (1000003, 1))  # the codes at its start, of an odd row stride
    s2 = torch.zeros_like(s)
    ctx.fp8_quantize(x, frx.FP8_ROWS, q2, s2)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(s, s2)
    w = torch.randn((24, k), generator=g).to(DEV)
    b, sb = torch.zeros((24, k), dtype=E4M3, device=DEV), torch.zeros((1, 3), device=DEV)
    ctx.fp8_quantize(w, frx.FP8_TILES, b, sb)
    y, y2 = torch.zeros((1, 24), device=DEV), torch.zeros((1, 24), device=DEV)
    ctx.fp8_linear(q, s, b, sb, y)
    ctx.fp8_linear(q2, s, b, sb, y2)
    assert torch.equal(y, y2) and y.abs().min() > 0
    t, t2 = torch.zeros((24, 1), device=DEV), torch.zeros((24, 1), device=DEV)
    ctx.fp8_quantize(w, frx.FP8_ROWS, b, rows := torch.zeros((24, 3), device=DEV))
    ctx.fp8_linear(b, rows, q, s, t)  # the row as the one weight row
    ctx.fp8_linear(b, rows, q2, s, t2)
    assert torch.equal(t, t2) and t.abs().min() > 0


@pytest.mark.parametrize("m,k,one_launch", [(4, 15872, True), (4, 15888, False), (3, 16384, True), (1, 63488, True),
                                            (1, 63536, True), (1, 63552, False), (5, 256, False), (4, 256, True)])
def test_which_calls_need_no_workspace(ctx, m, k, one_launch):
    """frx_fp8_linear_act on a fresh context under capture: one launch where M <= 4 and M K + 4 M ceil(K / 128) <=
    65536, as the header says, a refusal otherwise."""
    assert one_launch == (m <= 4 and m * k + 4 * m * -(-k // 128) <= 65536)
    side = torch.cuda.Stream()
    ctx.set_stream(side)
    x, y = torch.ones((m, k), device=DEV), torch.zeros((m, 16), device=DEV)
    b, sb = torch.ones((16, k), device=DEV).to(E4M3), torch.ones((1, -(-k // 128)), device=DEV)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        y.add_(0.0)
        if one_launch:
            ctx.fp8_linear_act(x, b, sb, y)
        else:
            with pytest.raises(frx.FrxError, match="captured") as e:
                ctx.fp8_linear_act(x, b, sb, y)
            assert e.value.kind == "Unsupported"
    for _ in range(2):
        y.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        # ones against ones: a code of 448 and a scale of f32(1 / 448) give 1 up to two roundings, summed exactly enough
        assert ((y - (k if one_launch else 0)).abs() <= k * 2.0 ** -20).all()
    del g
