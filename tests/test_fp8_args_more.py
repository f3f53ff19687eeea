"""More arguments of the 8-bit linears' binding, without a GPU (test_fp8_args has the rest)."""
import pytest
import torch

import ferrisres_amd as frx
from test_fp8_args import E4M3, E5M2, ctx, reaches_the_library, refuses  # noqa: F401  (ctx: the fixture)


def grad_args(E, N=40, K=24, R=128):
    return (torch.zeros((N, R)).to(E5M2), torch.zeros((N, 1)), torch.zeros((K, R)).to(E4M3), torch.zeros((K, 1)),
            torch.zeros((E + 1,), dtype=torch.int32))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gradients_of_experts_lie_apart(ctx, dtype):  # noqa: F811
    """Every expert's workgroups write their own matrix at the same time: an expanded output and one whose experts
    overlap are refused, rows between the experts are not."""
    E, N, K = 3, 40, 24
    a = grad_args(E)
    refuses(frx.FrxError, lambda: ctx.fp8_grad_weight_grouped(*a, torch.zeros((N, K), dtype=dtype).expand(E, N, K)))
    buf = torch.zeros((E * N * K + 64,), dtype=dtype)
    for step in (0, K, N * K - 1):
        refuses(frx.FrxError, lambda: ctx.fp8_grad_weight_grouped(*a, buf.as_strided((E, N, K), (step, K, 1))))
    for step in (N * K, N * K + 8):
        reaches_the_library(lambda: ctx.fp8_grad_weight_grouped(*a, buf.as_strided((E, N, K), (step, K, 1))))
    one = grad_args(1)
    reaches_the_library(lambda: ctx.fp8_grad_weight_grouped(*one, buf.as_strided((1, N, K), (0, K, 1))))


def test_shared_weights_are_read(ctx):  # noqa: F811
    """What is only read may be shared: one matrix for every expert."""
    a, sa = torch.zeros((12, 256)).to(E4M3), torch.zeros((12, 2))
    b, sb, y = torch.zeros((40, 256)).to(E4M3), torch.zeros((1, 2)), torch.zeros((12, 40))
    off = torch.zeros((4,), dtype=torch.int32)
    reaches_the_library(lambda: ctx.fp8_linear_grouped(a, sa, b.expand(3, 40, 256), sb.expand(3, 1, 2), off, y))
    reaches_the_library(lambda: ctx.fp8_linear_grouped(a, sa, [b] * 3, [sb] * 3, off, y))


@pytest.mark.parametrize("n", [16, 48, 256])
def test_a_single_row_has_any_stride(ctx, n):  # noqa: F811
    """The stride of a matrix of one row leads nowhere: whatever it is, the library gets one that it takes (a multiple
    of 16 that holds the row, up to 2^23), and rows of different strides may be one list's."""
    buf = torch.zeros((64 + n,)).to(E4M3)
    one = [buf.as_strided((1, n), (stride, 1)) for stride in (0, 1, n, n + 5, n + 16, 1 << 24)]
    for t in one:
        assert frx._rows2(t, "a")[:2] == (1, n)
        ld = frx._rows2(t, "a")[2]
        assert ld % 16 == 0 and n <= ld <= 1 << 23
    at, ld = frx._per_expert(one, len(one), (1, n), E4M3, "b", rows=True)
    assert ld % 16 == 0 and n <= ld <= 1 << 23 and len(at) == len(one)
    at, ld = frx._per_expert(buf.as_strided((3, 1, n), (16, 1000003, 1)), 3, (1, n), E4M3, "b", rows=True)
    assert ld % 16 == 0 and n <= ld <= 1 << 23 and at[1] - at[0] == 16
    for rows in (2, 3):  # more rows: the stride as it is
        assert frx._rows2(buf.as_strided((rows, n), (5, 1)), "a")[2] == 5


def test_tensors_of_another_device_are_refused(ctx):  # noqa: F811
    """Host tensors (or another card's) before a context of cuda:0: a device error of the binding's own, in place of
    an address that means nothing there."""
    i32 = lambda *d: torch.zeros(d, dtype=torch.int32)  # noqa: E731
    ctx._dev = 0

    def refused(call):
        with pytest.raises(frx.FrxError, match="the context on cuda:0") as e:
            call()
        assert e.value.kind == "Device"
    a, sa = torch.zeros((4, 256)).to(E4M3), torch.zeros((4, 2))
    b, sb, y = torch.zeros((40, 256)).to(E4M3), torch.zeros((1, 2)), torch.zeros((4, 40))
    refused(lambda: ctx.fp8_quantize(torch.zeros((4, 256)), frx.FP8_ROWS, a, sa))
    refused(lambda: ctx.fp8_linear(a, sa, b, sb, y))
    refused(lambda: ctx.fp8_linear_act(torch.zeros((4, 256)), b, sb, y))
    refused(lambda: ctx.fp8_linear_grouped(a, sa, b[None], sb[None], i32(2), y))
    refused(lambda: ctx.fp8_linear_grouped(a, sa, [b], [sb], i32(2), y))
    refused(lambda: ctx.fp8_grad_weight_grouped(*grad_args(2), torch.zeros((2, 40, 24))))
    refused(lambda: ctx.fp8_grad_weight_grouped(*grad_args(1), [torch.zeros((40, 24))]))
    rows = frx.MoeRows.empty(4, 2, 3, 1, device="cpu")
    x, xs = torch.zeros((4, 8)), torch.zeros((rows.R, 8))
    refused(lambda: ctx.moe_sort(i32(4, 2), rows))
    refused(lambda: ctx.moe_dispatch(x, rows, xs))
    refused(lambda: ctx.moe_combine(xs, rows, None, x))
    refused(lambda: ctx.moe_combine(xs, rows, torch.zeros((4, 2)), x))
    refused(lambda: ctx.moe_combine_backward(x, xs, rows, None, xs.clone(), torch.zeros((4, 2))))
    meta = torch.zeros((4, 2), dtype=torch.int32, device="meta")
    with pytest.raises(frx.FrxError, match="index tensors"):
        frx.MoeRows(3, 1, i32(4), meta, i32(8))


def test_routing_shapes_are_checked(ctx):  # noqa: F811
    """What the quick checks of the routing calls let through has the right shape and is contiguous; the rest is told
    apart as before."""
    rows = frx.MoeRows.empty(4, 2, 3, 1, device="cpu")
    f = lambda *d: torch.zeros(d)  # noqa: E731
    x, xs, w = f(4, 8), f(rows.R, 8), f(4, 2)
    for call in (lambda: ctx.moe_dispatch(x, rows, xs), lambda: ctx.moe_dispatch(f(4, 2, 4), rows, f(rows.R, 2, 4)),
                 lambda: ctx.moe_dispatch(f(4), rows, f(rows.R)), lambda: ctx.moe_combine(xs, rows, w, x),
                 lambda: ctx.moe_combine_backward(x, xs, rows, w, xs.clone(), w.clone())):
        reaches_the_library(call)
    wide = f(4, 16)[:, ::2]
    for call in (lambda: ctx.moe_dispatch(f(), rows, xs), lambda: ctx.moe_dispatch(f(5, 8), rows, xs),
                 lambda: ctx.moe_dispatch(wide, rows, xs), lambda: ctx.moe_dispatch(x, rows, f(rows.R, 9)),
                 lambda: ctx.moe_combine(xs, rows, w, f(5, 8)), lambda: ctx.moe_combine(xs, rows, w, wide),
                 lambda: ctx.moe_combine(f(rows.R + 1, 8), rows, w, x), lambda: ctx.moe_combine(xs, rows, w, f(1, 4, 8)),
                 lambda: ctx.moe_combine_backward(f(5, 8), xs, rows, w, xs.clone(), w.clone()),
                 lambda: ctx.moe_combine_backward(wide, xs, rows, w, xs.clone(), w.clone()),
                 lambda: ctx.moe_combine_backward(x, xs, rows, f(4, 3), xs.clone(), w.clone()),
                 lambda: ctx.fp8_linear_grouped(f(12, 16).to(E4M3), f(12, 1), f(3, 40, 16).to(E4M3), f(3, 1, 1),
                                                torch.zeros(4, dtype=torch.int32), f(12, 80)[:, ::2])):
        refuses(frx.FrxError, call)
