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
