"""Arguments of the 8-bit linears and the expert sort, without a GPU: a null context is a device error and never
dereferenced, the binding refuses what does not fit before it calls the library, and the room for sorted rows."""
import ctypes

import pytest
import torch

import ferrisres_amd as frx

E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2


def test_null_context():
    L = frx.lib()
    rows = frx._MoeRowsC()
    p = ctypes.byref(rows)
    assert L.frx_fp8_quantize(None, None, 0, 1, 1, 1, 0, 0, None, 16, None) == 3
    assert L.frx_fp8_linear(None, None, 16, 0, None, None, 16, None, 128, None, 0, 1, 16, 1) == 3
    assert L.frx_fp8_linear_act(None, None, 0, None, 16, None, None, 0, 1, 16, 1) == 3
    assert L.frx_fp8_linear_grouped(None, None, 16, 0, None, None, 16, None, None, 1, None, 0, 1, 16, 1) == 3
    assert L.frx_fp8_grad_weight_grouped(None, None, 16, 0, None, None, 16, None, None, 1, None, 0, 16, 1, 1) == 3
    assert L.frx_moe_sort(None, None, p) == 3
    assert L.frx_moe_dispatch(None, None, 4, p, None) == 3
    assert L.frx_moe_combine(None, None, 0, p, None, None, 0, 1) == 3
    assert L.frx_moe_combine_backward(None, None, 0, None, 0, p, None, None, None, 1) == 3


@pytest.mark.parametrize("T,top_k,E,align", [(1, 1, 1, 1), (0, 2, 8, 128), (33, 4, 8, 16), (512, 2, 64, 128)])
def test_capacity_holds_the_worst_routing(T, top_k, E, align):
    """Every expert with a route may waste align - 1 rows, and the end is a multiple of align."""
    up = lambda n: -(-n // align) * align  # noqa: E731
    got = frx.MoeRows.capacity(T, top_k, E, align)
    slots = T * top_k
    spread = [slots // E + (e < slots % E) for e in range(E)]
    one_each = [1] * min(E - 1, slots) + [slots - min(E - 1, slots)]
    for sizes in (spread, one_each, [slots]):
        assert sum(up(n) for n in sizes) <= got
    assert got % align == 0 and got <= slots + E * align
    assert frx.MoeRows.capacity(T, top_k, E, 0) == 0


@pytest.fixture
def ctx():
    c = frx.Context.__new__(frx.Context)  # no device behind it: whatever passes the binding's checks is a device error
    c._h = None
    return c


def refuses(kind, call):
    with pytest.raises(kind) as e:
        call()
    if kind is frx.FrxError:
        assert e.value.kind == "Shape", e.value


def reaches_the_library(call):
    with pytest.raises(frx.FrxError) as e:
        call()
    assert e.value.kind == "Device"


def test_binding_checks_codes_and_scales(ctx):
    a, sa = torch.zeros((4, 272)).to(E4M3), torch.zeros((4, 3))
    b, sb = torch.zeros((130, 272)).to(E4M3), torch.zeros((2, 3))
    y, x = torch.zeros((4, 130)), torch.zeros((4, 272))
    reaches_the_library(lambda: ctx.fp8_linear(a, sa, b, sb, y))
    reaches_the_library(lambda: ctx.fp8_linear(a.to(E5M2), sa, b, torch.zeros((130, 3)), y.bfloat16()))
    reaches_the_library(lambda: ctx.fp8_linear_act(x, b, sb, y))
    for bad in (lambda: ctx.fp8_linear(a, sa[:, :2], b, sb, y), lambda: ctx.fp8_linear(a, sa, b, sb[:1], y),
                lambda: ctx.fp8_linear(a, sa, b[:, :256], sb, y), lambda: ctx.fp8_linear(a, sa, b, sb, y[:3]),
                lambda: ctx.fp8_linear(a, sa, b, sb, torch.zeros((130, 4)).t()),
                lambda: ctx.fp8_linear(a.view(torch.uint8).t().contiguous().t().view(E4M3), sa, b, sb, y),
                lambda: ctx.fp8_linear(a[0], sa, b, sb, y),
                lambda: ctx.fp8_linear_act(torch.zeros((4, 544))[:, ::2], b, sb, y),
                lambda: ctx.fp8_linear_act(x, b, sb, y[:, :129])):
        refuses(frx.FrxError, bad)
    for bad in (lambda: ctx.fp8_linear(x, sa, b, sb, y), lambda: ctx.fp8_linear(a, sa.double(), b, sb, y),
                lambda: ctx.fp8_linear(a, sa, b.to(E5M2), sb, y), lambda: ctx.fp8_linear(a, sa, b, sb, y.half()),
                lambda: ctx.fp8_linear_act(x.half(), b, sb, y)):
        refuses(TypeError, bad)


@pytest.mark.parametrize("blocks,q,s", [(frx.FP8_ROWS, (5, 48), (5, 1)), (frx.FP8_COLS, (40, 16), (40, 1)),
                                        (frx.FP8_TILES, (5, 48), (1, 1)), (frx.FP8_TILES_T, (40, 16), (1, 1))])
def test_binding_checks_the_quantiser(ctx, blocks, q, s):
    x = torch.zeros((5, 40))
    new = lambda *d: torch.zeros(d)  # noqa: E731
    reaches_the_library(lambda: ctx.fp8_quantize(x, blocks, new(*q).to(E4M3), new(*s)))
    refuses(frx.FrxError, lambda: ctx.fp8_quantize(x, blocks, new(q[0], q[1] + 16).to(E4M3), new(*s)))
    refuses(frx.FrxError, lambda: ctx.fp8_quantize(x, blocks, new(q[0] + 1, q[1]).to(E4M3), new(*s)))
    refuses(frx.FrxError, lambda: ctx.fp8_quantize(x, blocks, new(*q).to(E4M3), new(s[0], 2)))
    refuses(frx.FrxError, lambda: ctx.fp8_quantize(new(40, 5).t(), blocks, new(*q).to(E4M3), new(*s)))
    refuses(TypeError, lambda: ctx.fp8_quantize(x, blocks, new(*q), new(*s)))


def test_binding_checks_experts_and_rows(ctx):
    i32 = lambda *d: torch.zeros(d, dtype=torch.int32)  # noqa: E731
    a, sa = torch.zeros((12, 256)).to(E4M3), torch.zeros((12, 2))
    b, sb, y = torch.zeros((3, 40, 256)).to(E4M3), torch.zeros((3, 1, 2)), torch.zeros((12, 40))
    off = i32(4)
    reaches_the_library(lambda: ctx.fp8_linear_grouped(a, sa, b, sb, off, y))
    reaches_the_library(lambda: ctx.fp8_linear_grouped(a, sa, list(b), list(sb), off, y))
    refuses(frx.FrxError, lambda: ctx.fp8_linear_grouped(a, sa, b[:2], sb, off, y))
    refuses(frx.FrxError, lambda: ctx.fp8_linear_grouped(a, sa, b, sb[:, :, :1], off, y))
    refuses(TypeError, lambda: ctx.fp8_linear_grouped(a, sa, b, sb, off.long(), y))
    dy, xs = torch.zeros((40, 128)).to(E5M2), torch.zeros((24, 128)).to(E4M3)
    reaches_the_library(lambda: ctx.fp8_grad_weight_grouped(dy, torch.zeros((40, 1)), xs, torch.zeros((24, 1)), off,
                                                            torch.zeros((3, 40, 24))))
    refuses(frx.FrxError, lambda: ctx.fp8_grad_weight_grouped(dy, torch.zeros((40, 1)), xs, torch.zeros((24, 1)), off,
                                                              torch.zeros((3, 24, 40))))
    rows = frx.MoeRows.empty(4, 2, 3, 4, device="cpu")
    assert rows.R == frx.MoeRows.capacity(4, 2, 3, 4)
    reaches_the_library(lambda: ctx.moe_sort(i32(4, 2), rows))
    refuses(frx.FrxError, lambda: ctx.moe_sort(i32(4, 1), rows))
    refuses(TypeError, lambda: ctx.moe_sort(i32(4, 2).long(), rows))
    refuses(frx.FrxError, lambda: ctx.moe_dispatch(torch.zeros((5, 8)), rows, torch.zeros((rows.R, 8))))
    refuses(frx.FrxError, lambda: ctx.moe_dispatch(torch.zeros((4, 8)), rows, torch.zeros((rows.R, 9))))
    refuses(TypeError, lambda: ctx.moe_dispatch(torch.zeros((4, 8)), rows, torch.zeros((rows.R, 8)).double()))
    refuses(frx.FrxError, lambda: ctx.moe_combine(torch.zeros((rows.R, 8)), rows, torch.zeros((4, 3)), torch.zeros((4, 8))))
    refuses(frx.FrxError, lambda: ctx.moe_combine_backward(torch.zeros((4, 8)), None, rows, None,
                                                           torch.zeros((rows.R, 8)), torch.zeros((4, 2))))
    refuses(frx.FrxError, lambda: frx.MoeRows(3, 1, i32(3), i32(4, 2), i32(9)))


def test_binding_checks_nothing_to_do(ctx):
    """No experts, no tokens, a vector in a matrix' place."""
    i32 = lambda *d: torch.zeros(d, dtype=torch.int32)  # noqa: E731
    a, sa, y = torch.zeros((12, 256)).to(E4M3), torch.zeros((12, 2)), torch.zeros((12, 40))
    for b, sb in ((torch.zeros((0, 40, 256)).to(E4M3), torch.zeros((0, 1, 2))), ([], [])):
        refuses(frx.FrxError, lambda: ctx.fp8_linear_grouped(a, sa, b, sb, i32(1), y))
    dy = torch.zeros((40, 16)).to(E5M2)
    for off, dw in ((i32(1), []), (i32(1), torch.zeros((0, 40, 12))), (i32(0), [])):
        refuses(frx.FrxError, lambda: ctx.fp8_grad_weight_grouped(dy, torch.zeros((40, 1)), a[:, :16],
                                                                  torch.zeros((12, 1)), off, dw))
    b, sb = torch.zeros((40, 256)).to(E4M3), torch.zeros((1, 2))
    refuses(frx.FrxError, lambda: ctx.fp8_linear_act(torch.zeros(256), b, sb, y))
    rows = frx.MoeRows.empty(0, 2, 3, 4, device="cpu")
    reaches_the_library(lambda: ctx.moe_dispatch(torch.zeros((0, 8)), rows, torch.zeros((rows.R, 8))))
