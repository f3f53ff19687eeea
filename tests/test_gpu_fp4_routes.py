"""The expert layer's router (frx_fp4_moe_ffn): a single token's routes are found inside gate and up, in each kernel of
theirs, two tokens' in a launch of its own. Against 64 bits, and against a call that is given the routes."""
import numpy as np
import pytest
import torch

import ferrisres_amd as frx
from _fp4_ref import DT
from _gpu import DEV, host

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    assert torch.cuda.is_available(), "GPU tests need a gfx950 device"
    c = frx.Context(0)
    yield c
    c.close()


@pytest.mark.parametrize("T", [1, 2])
@pytest.mark.parametrize("xt,rt", [("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32"), ("f32", "bf16")])
@pytest.mark.parametrize("H", [64, 2080, 4128])  # gate and up with 2 and 4 steps a wave, and K in chunks
@pytest.mark.parametrize("E,top_k", [(32, 2), (33, 3), (64, 64)])
def test_routes_of_few_tokens(ctx, E, top_k, H, xt, rt, T):
    """The experts in order, their weights, and the layer's bits with the same routes given. Logits are planted 3/32 apart:
    router rows are x times what gives them, over x's square, and a bf16 row is off by 2^-8 of 3 at most."""
    rng = np.random.default_rng(E + H)
    x = torch.from_numpy(rng.standard_normal((T, H)).astype(np.float32)).to(DT[xt])
    x[1:] = x[:1]  # (the router fits one token)
    v = x[0].double().numpy()
    planted = (rng.permutation(E) - E / 2) * (3 / 32)
    router = torch.from_numpy((planted[:, None] * v / (v @ v)).astype(np.float32)).to(DT[rt])
    logits = router.double().numpy() @ v
    order = np.argsort(-logits)[:top_k]
    assert np.abs(np.diff(np.sort(logits))).min() > 1 / 32
    g = torch.Generator(device=DEV).manual_seed(H)
    codes = lambda n, k: (torch.randint(0, 256, (E, n, k // 2), dtype=torch.uint8, device=DEV, generator=g),  # noqa: E731
                          torch.randint(118, 123, (E, n, -(-k // 128) * 4), dtype=torch.uint8, device=DEV, generator=g))
    w = [t for m in (codes(32, H), codes(32, H), codes(H, 32)) for t in m]
    idx, wt = torch.full((T, top_k), -9, dtype=torch.int32, device=DEV), torch.zeros((T, top_k), device=DEV)
    y, z, taken = (torch.full((T, H), float("nan"), device=DEV) for _ in range(3))
    ctx.fp4_moe_ffn(x.to(DEV), router.to(DEV), *w, y, idx, wt)
    assert (idx.cpu().numpy() == order).all()
    p = np.exp(logits[order] - logits[order[0]])
    p /= p.sum()
    # a logit is off by H u of its magnitudes, which differ by that from the largest's; 64 u for exponentials and sum
    off = 2.1 * H * 2.0 ** -24 * (np.abs(router.double().numpy()) @ np.abs(v)).max() + 64 * 2.0 ** -24
    assert (np.abs(host(wt) - p) <= off * p).all()
    ctx.fp4_moe_ffn(x.to(DEV), None, *w, z, idx, wt)
    ctx.fp4_moe_ffn(x.to(DEV), router.to(DEV), *w, taken, top_k=top_k)
    assert torch.isfinite(y).all() and y.any()
    assert torch.equal(y, z) and torch.equal(y, taken)
