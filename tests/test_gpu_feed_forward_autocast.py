"""``gated_feed_forward`` inside an autocast region: the region's type, as three linear layers would have it; float32 weights train."""

from __future__ import annotations

import pytest
import torch

import gdn2_tilelang_b200 as gdn2
from gdn2_tilelang_b200 import _cabi
from tests.test_gpu_feed_forward import BF, F16

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"], autouse=True)
def way(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(_cabi.kernels(), "host", None)


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("T", [5, 300])
def test_float32_weights(T, dtype):
    """The same bits as the call on operands cast by hand; gradients come back in float32."""
    torch.manual_seed(T)
    mlp = gdn2.GatedFeedForward(72, 136).cuda()
    x = torch.randn(T, 72, device="cuda", requires_grad=True)
    weights = [mlp.gate_proj.weight, mlp.up_proj.weight, mlp.down_proj.weight]
    with torch.autocast("cuda", dtype=dtype):
        y = mlp(x)
        linear = mlp.down_proj(torch.nn.functional.silu(mlp.gate_proj(x)) * mlp.up_proj(x))
    assert y.dtype == linear.dtype == dtype
    cast = [t.detach().to(dtype).requires_grad_() for t in (x, *weights)]
    want = gdn2.gated_feed_forward(*cast)
    assert torch.equal(y, want)
    dy = torch.randn_like(y)
    for got, ref in zip(torch.autograd.grad(y, [x, *weights], dy), torch.autograd.grad(want, cast, dy)):
        assert got.dtype == torch.float32 and torch.equal(got, ref.float())


def test_operands_of_another_type_than_the_regions():
    x, wg, wu, wd = (torch.randn(*s, device="cuda").to(F16) for s in ((9, 72), (40, 72), (40, 72), (24, 40)))
    with torch.autocast("cuda", dtype=BF):
        y = gdn2.gated_feed_forward(x, wg.float(), wu, wd.to(BF))
    assert y.dtype == BF and torch.equal(y, gdn2.gated_feed_forward(*(t.to(BF) for t in (x, wg, wu, wd))))


def test_outside_a_region_float32_is_refused():
    mlp = gdn2.GatedFeedForward(8, 16).cuda()
    for x in (torch.zeros(3, 8, device="cuda"), torch.zeros(3, 8, device="cuda", dtype=torch.float64)):
        with pytest.raises(TypeError, match="float16 or bfloat16"):
            mlp(x)
    with torch.autocast("cuda", dtype=BF), pytest.raises(TypeError):
        mlp(torch.zeros(3, 8, device="cuda", dtype=torch.float64))
