"""The dot products of frx_moe_combine_backward over long rows: a term goes through at most 16 + H / 512 f32 roundings, 8
fused multiply-adds of its group, the groups of its lane and the lanes of its wave."""
import pytest
import torch

import ferrisres_amd as frx
from _gpu import DEV

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


def backward(ctx, dy, ys, top_k):
    T, H = dy.shape
    rows = frx.MoeRows.empty(T, top_k, 1, 1)
    ctx.moe_sort(torch.zeros((T, top_k), dtype=torch.int32, device=DEV), rows)
    dw = torch.full((T, top_k), float("nan"), device=DEV)
    dys = torch.empty((rows.R, H), dtype=ys.dtype, device=DEV)
    ctx.moe_combine_backward(dy, ys, rows, None, dys, dw)
    want = (dy.double().repeat_interleave(top_k, 0) * ys.double()).view(T, top_k, H)
    return dw, want.sum(2), want.abs().sum(2)


@pytest.mark.parametrize("H", [1, 7, 64, 515, 4096, 8191, 8192, 65536, 65543])
@pytest.mark.parametrize("dt,st", [("f32", "f32"), ("bf16", "bf16"), ("f32", "bf16"), ("bf16", "f32")])
def test_random_rows(ctx, H, dt, st):
    t = {"f32": torch.float32, "bf16": torch.bfloat16}
    g = torch.Generator(device=DEV).manual_seed(H)
    dy, ys = (torch.randn((n, H), generator=g, device=DEV) for n in (3, 6))
    dw, ref, mag = backward(ctx, dy.to(t[dt]), ys.to(t[st]), 2)
    assert ((dw.double() - ref).abs() <= (16 + H / 512) * 2.0 ** -24 * mag).all()


@pytest.mark.parametrize("H", [65536, 65543])
def test_roundings_that_all_go_one_way(ctx, H):
    """Terms a little above 1, whose excess a sum that goes term by term drops at every step once it is large: H / 64
    such steps of a lane lose 230 times 2^-24 here."""
    excess = 0.9 * 2.0 ** -15
    dw, ref, mag = backward(ctx, torch.ones((2, H), device=DEV), torch.full((2, H), 1.0 + excess, device=DEV), 1)
    assert ((dw.double() - ref).abs() <= (16 + H / 512) * 2.0 ** -24 * mag).all()


def test_infinities_and_nan(ctx):
    """They come out as a plain sum gives them."""
    H = 4096
    dy, ys = torch.ones((4, H), device=DEV), torch.ones((4, H), device=DEV)
    ys[0, 17] = float("inf")
    ys[1, 4000], ys[1, 5] = float("inf"), float("-inf")
    ys[2, 100] = float("nan")
    dw, _, _ = backward(ctx, dy, ys, 1)
    dw = dw.flatten()
    assert dw[0] == float("inf") and torch.isnan(dw[1]) and torch.isnan(dw[2]) and dw[3] == H
