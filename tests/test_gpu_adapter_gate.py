"""The gate of adapter_swiglu (csrc/adapters.hip) by itself: rows whose adapter adds nothing."""
import pytest
import torch

from oracle import requests_ref as ref
from serving import fused_ops
from serving.adapters import AdapterWeights, adapter_swiglu, build_adapter_plan

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_the_gate_is_as_exact_as_the_frameworks():
    """fp32: the sums are base's, so all that is off is the gate's own. In units of 2^-24 of
    the result: the exponential 4 (two steps of fp32), the sum, the quotient and the two
    products half a step (1) each, and one unit each for the quotient's and the exponential's
    effect on the rest: 10. An error in the exponential's argument would be 2^-24 of the
    argument, up to 80 units."""
    w = AdapterWeights(32, (512, 512), 2, 8, dtype=torch.float32, device=DEV)
    g = torch.Generator().manual_seed(8)
    T = 96
    gate = torch.cat([-80 + 60 * torch.rand(T // 3, 512, generator=g),
                      -20 + 18 * torch.rand(T // 3, 512, generator=g),
                      -2 + 82 * torch.rand(T // 3, 512, generator=g)])
    base = torch.cat([gate, torch.randn(T, 512, generator=g)], 1)
    x = torch.randn(T, 32, generator=g).to(DEV)
    want = ref.swiglu(base.double())
    bd, ids = base.to(DEV), torch.arange(T, device=DEV, dtype=torch.int32) % 2
    out = adapter_swiglu(bd, x, w, build_adapter_plan(ids, 2))
    err = (out.cpu().double() - want).abs()
    assert float((err / want.abs()).max()) <= 10 * 2.0 ** -24
    assert torch.equal(out, fused_ops.silu_mul(bd[:, :512], bd[:, 512:]))
