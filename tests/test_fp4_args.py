"""Arguments of the 4-bit linears and the expert layer, without a GPU: a null context is a device error and never
dereferenced, the binding refuses what does not fit before it calls the library; and the reference of the GPU tests
against borders worked out by hand."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp4_ref import ref_codes, values
from test_fp8_args import ctx, reaches_the_library, refuses  # noqa: F401

U8, F4, E8 = torch.uint8, torch.float4_e2m1fn_x2, torch.float8_e8m0fnu


def test_null_context():
    L = frx.lib()
    assert L.frx_fp4_quantize(None, None, 0, 1, 1, 1, 0, None, 16, None) == 3
    assert L.frx_fp4_dequantize(None, None, 16, None, 1, 1, None, 0, 1) == 3
    assert L.frx_fp4_linear(None, None, 16, None, None, 16, None, None, 0, 1, 32, 1) == 3
    assert L.frx_fp4_linear_act(None, None, 0, None, 16, None, None, 0, 1, 32, 1) == 3
    assert L.frx_fp4_linear_grouped(None, None, 16, None, None, 16, None, None, 1, None, 0, 1, 32, 1) == 3
    assert L.frx_fp4_grad_weight_grouped(None, None, 16, None, None, 16, None, None, 1, None, 0, 32, 1, 1) == 3
    assert L.frx_fp4_moe_ffn(None, None, 0, None, 0, None, None, None, None, None, None, 1, 32, 32, 1, 1, 0, None, 0,
                             None, None) == 3


def test_reference_borders():
    x = torch.tensor([[4.0, 0.25, 0.26, 0.75, 0.74, 1.25, 1.26, 1.75, 2.5, 2.51, 3.5, 5.0, 5.1, 7.9, -0.75, -7.0]])
    code, byte = ref_codes(x)
    assert byte[0].tolist() == [127, 0, 0, 0]
    assert code[0, :16].tolist() == [6, 0, 1, 2, 1, 2, 3, 4, 4, 5, 6, 6, 7, 7, 10, 15]
    assert values(code, byte)[0, :16].tolist() == [4, 0, .5, 1, .5, 1, 1.5, 2, 2, 3, 4, 4, 6, 6, -1, -6]
    assert ref_codes(torch.tensor([[2.0 ** -149, 2.0 ** -125]]))[1][0, 0] == 0
    assert ref_codes(torch.tensor([[3.0e38]]))[1][0, 0] == 252
    code, byte = ref_codes(torch.tensor([[float("inf"), 1.0]]))
    assert byte[0, 0] == 255 and not code.any() and np.isnan(values(code, byte)).all()


def z(*d, dt=U8):
    return torch.zeros(d, dtype=dt)


def test_binding_checks_codes_and_scales(ctx):  # noqa: F811
    a, sa, b, sb = z(4, 144), z(4, 12), z(130, 144), z(130, 12)
    y, x = torch.zeros((4, 130)), torch.zeros((4, 288))
    reaches_the_library(lambda: ctx.fp4_linear(a, sa, b, sb, y))
    reaches_the_library(lambda: ctx.fp4_linear(a.view(F4), sa.view(E8), b.view(F4), sb.view(E8), y.bfloat16()))
    reaches_the_library(lambda: ctx.fp4_linear_act(x, b, sb, y))
    reaches_the_library(lambda: ctx.fp4_dequantize(a, sa, torch.zeros((4, 270))))
    for bad in (lambda: ctx.fp4_linear(a, sa[:, :9], b, sb, y), lambda: ctx.fp4_linear(a, sa, b, sb[:129], y),
                lambda: ctx.fp4_linear(a, sa, b[:, :128], sb, y), lambda: ctx.fp4_linear(a, sa, b, sb, y[:3]),
                lambda: ctx.fp4_linear(a, sa, b, sb, torch.zeros((130, 4)).t()),
                lambda: ctx.fp4_linear(a.t().contiguous().t(), sa, b, sb, y), lambda: ctx.fp4_linear(a[0], sa, b, sb, y),
                lambda: ctx.fp4_linear(a, z(4, 24)[:, ::2], b, sb, y),
                lambda: ctx.fp4_linear_act(torch.zeros((4, 576))[:, ::2], b, sb, y),
                lambda: ctx.fp4_linear_act(x[:, :256], b, sb, y), lambda: ctx.fp4_linear_act(x, b, sb, y[:, :129]),
                lambda: ctx.fp4_dequantize(a, sa, torch.zeros((4, 256))),
                lambda: ctx.fp4_dequantize(a, sa, torch.zeros((5, 288)))):
        refuses(frx.FrxError, bad)
    for bad in (lambda: ctx.fp4_linear(a.float(), sa, b, sb, y), lambda: ctx.fp4_linear(a, sa.int(), b, sb, y),
                lambda: ctx.fp4_linear(a, sa, b.view(torch.float8_e4m3fn), sb, y),
                lambda: ctx.fp4_linear(a, sa, b, sb, y.half()), lambda: ctx.fp4_linear_act(x.half(), b, sb, y),
                lambda: ctx.fp4_dequantize(a, sa, x.double())):
        refuses(TypeError, bad)


@pytest.mark.parametrize("blocks,q,s", [(frx.FP4_ROWS, (5, 32), (5, 4)), (frx.FP4_COLS, (40, 16), (40, 4))])
def test_binding_checks_the_quantiser(ctx, blocks, q, s):  # noqa: F811
    x = torch.zeros((5, 40))
    reaches_the_library(lambda: ctx.fp4_quantize(x, blocks, z(*q), z(*s)))
    reaches_the_library(lambda: ctx.fp4_quantize(x.bfloat16(), blocks, z(*q).view(F4), z(*s).view(E8)))
    for bad in (lambda: ctx.fp4_quantize(x, blocks, z(q[0], q[1] + 16), z(*s)),
                lambda: ctx.fp4_quantize(x, blocks, z(q[0] + 1, q[1]), z(*s)),
                lambda: ctx.fp4_quantize(x, blocks, z(*q), z(s[0], 2)),
                lambda: ctx.fp4_quantize(torch.zeros((40, 5)).t(), blocks, z(*q), z(*s))):
        refuses(frx.FrxError, bad)
    refuses(TypeError, lambda: ctx.fp4_quantize(x, blocks, torch.zeros(q), z(*s)))
    refuses(TypeError, lambda: ctx.fp4_quantize(x, blocks, z(*q), torch.zeros(s)))
    refuses(TypeError, lambda: ctx.fp4_quantize(x.half(), blocks, z(*q), z(*s)))


def test_binding_checks_groups(ctx):  # noqa: F811
    i32 = lambda *d: torch.zeros(d, dtype=torch.int32)  # noqa: E731
    a, sa, b, sb, y, off = z(12, 128), z(12, 8), z(3, 40, 128), z(3, 40, 8), torch.zeros((12, 40)), i32(4)
    reaches_the_library(lambda: ctx.fp4_linear_grouped(a, sa, b, sb, off, y))
    reaches_the_library(lambda: ctx.fp4_linear_grouped(a, sa, list(b), list(sb.view(E8)), off, y))
    for bad in (lambda: ctx.fp4_linear_grouped(a, sa, b[:2], sb, off, y),
                lambda: ctx.fp4_linear_grouped(a, sa, b, sb[:, :, :4], off, y),
                lambda: ctx.fp4_linear_grouped(a, sa[:11], b, sb, off, y),
                lambda: ctx.fp4_linear_grouped(a, sa, b, sb, off, y[:, :39]),
                lambda: ctx.fp4_linear_grouped(a, sa, z(0, 40, 128), z(0, 40, 8), i32(1), y),
                lambda: ctx.fp4_linear_grouped(a, sa, [], [], i32(1), y)):
        refuses(frx.FrxError, bad)
    refuses(TypeError, lambda: ctx.fp4_linear_grouped(a, sa, b, sb, off.long(), y))
    refuses(TypeError, lambda: ctx.fp4_linear_grouped(a, sa, b.int(), sb, off, y))


def test_binding_checks_weight_gradients(ctx):  # noqa: F811
    a, sa, b, sb, off = z(40, 128), z(40, 8), z(70, 128), z(70, 8), torch.zeros(4, dtype=torch.int32)
    dw = torch.zeros((3, 40, 70))
    call = ctx.fp4_grad_weight_grouped
    reaches_the_library(lambda: call(a, sa, b, sb, off, dw))
    reaches_the_library(lambda: call(a.view(F4), sa.view(E8), b, sb, off, list(dw.bfloat16())))
    for bad in (lambda: call(a, sa, b[:, :112], sb, off, dw), lambda: call(a, sa[:39], b, sb, off, dw),
                lambda: call(a, sa, b, sb[:, :4], off, dw), lambda: call(a, sa, b, sb, off, dw[:2]),
                lambda: call(a, sa, b, sb, off, dw[:, :, :69]), lambda: call(a, sa, b, sb, off, dw[:1].expand(3, 40, 70)),
                lambda: call(a, sa, b, sb, off[:1], dw[:0])):
        refuses(frx.FrxError, bad)
    refuses(TypeError, lambda: call(a, sa, b, sb, off.long(), dw))
    refuses(TypeError, lambda: call(a, sa, b, sb, off, dw.double()))


def test_binding_checks_the_layer(ctx):  # noqa: F811
    T, H, I, E = 3, 64, 96, 4
    x, router, y = torch.zeros((T, H)), torch.zeros((E, H)), torch.zeros((T, H))
    w = [z(E, I, 32), z(E, I, 4), z(E, I, 32), z(E, I, 4), z(E, H, 48), z(E, H, 4)]
    idx, wt = torch.zeros((T, 2), dtype=torch.int32), torch.zeros((T, 2))
    reaches_the_library(lambda: ctx.fp4_moe_ffn(x, router, *w, y, top_k=2))
    reaches_the_library(lambda: ctx.fp4_moe_ffn(x, router, *w, y, idx, wt))
    reaches_the_library(lambda: ctx.fp4_moe_ffn(x.bfloat16(), None, *[list(t) for t in w], y.bfloat16(), idx, wt))
    for bad in (lambda: ctx.fp4_moe_ffn(x, router, *w, y), lambda: ctx.fp4_moe_ffn(x, None, *w, y, idx),
                lambda: ctx.fp4_moe_ffn(x, None, *w, y, topk_w=wt), lambda: ctx.fp4_moe_ffn(x, None, *w, y, top_k=2),
                lambda: ctx.fp4_moe_ffn(x, router[:3], *w, y, top_k=2),
                lambda: ctx.fp4_moe_ffn(x, router, *w, y[:2], top_k=2),
                lambda: ctx.fp4_moe_ffn(x, router, *w, y, idx, wt, top_k=3),
                lambda: ctx.fp4_moe_ffn(x, router, *w, y, idx, wt[:, :1]),
                lambda: ctx.fp4_moe_ffn(x, router, *w, y, idx[:2], wt),
                lambda: ctx.fp4_moe_ffn(torch.zeros((T, 2 * H))[:, ::2], router, *w, y, top_k=2),
                lambda: ctx.fp4_moe_ffn(x, router, *(t[:0] for t in w), y, top_k=2),
                lambda: ctx.fp4_moe_ffn(x, router, *[], *w[:4], z(E, H, 32), w[5], y, top_k=2),
                lambda: ctx.fp4_moe_ffn(x, router, w[0], w[1][:, :, :2], *w[2:], y, top_k=2),
                lambda: ctx.fp4_moe_ffn(x, router, w[0], w[1], w[2][:3], *w[3:], y, top_k=2)):
        refuses(frx.FrxError, bad)
    for bad in (lambda: ctx.fp4_moe_ffn(x, router, *w, y, idx.long(), wt),
                lambda: ctx.fp4_moe_ffn(x, router, *w, y, idx, wt.double()),
                lambda: ctx.fp4_moe_ffn(x.half(), router, *w, y, idx, wt),
                lambda: ctx.fp4_moe_ffn(x, router.half(), *w, y, idx, wt),
                lambda: ctx.fp4_moe_ffn(x, router, w[0].int(), *w[1:], y, idx, wt)):
        refuses(TypeError, bad)
