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
