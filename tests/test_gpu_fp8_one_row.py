"""One weight row in the 8-bit linears: its one line of scales is FP8_TILES' and FP8_ROWS' at once."""
import pytest
import torch

import ferrisres_amd as frx
from _gpu import DEV
from test_gpu_fp8 import E4M3, check, operand, quantize, values

pytestmark = pytest.mark.gpu


@pytest.fixture
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("m,k", [(1, 2048), (5, 272), (40, 8192), (100, 8192), (3000, 5392), (20000, 8192)])
@pytest.mark.parametrize("out", [torch.float32, torch.bfloat16])
def test_activations_quantised_inside_are_the_two_calls(ctx, m, k, out):
    x = values(m + k, m, k, "bf16", spread=False).to(DEV)
    b, sb, bv = operand(1, 1, k, E4M3, tiles=True)
    b, sb = b.to(DEV), sb.to(DEV)
    _, q, s, _ = quantize(ctx, x, frx.FP8_ROWS, E4M3)
    y, y2 = (torch.full((m, 1), float("nan"), dtype=out, device=DEV) for _ in range(2))
    ctx.fp8_linear(q, s, b, sb, y)
    ctx.fp8_linear_act(x, b, sb, y2)
    assert torch.equal(y, y2)
    if out == torch.float32:
        av = q.cpu().double() * s.cpu().double().repeat_interleave(128, 1)[:, :k]
        check(y, av @ bv.t(), av.abs() @ bv.abs().t(), k)
