"""The operators' `out` where a gradient graph saved it."""
import pytest
import torch

from serving.adapters import AdapterWeights, adapter_add, build_adapter_plan
from serving.controls import LogitControls, control_logits

pytestmark = pytest.mark.gpu
DEV = "cuda"


def test_a_graph_that_saved_out_finds_it_changed():
    w = AdapterWeights(32, (32,), 2, 8, dtype=torch.float32, device=DEV)
    x, base = torch.randn(4, 32, device=DEV), torch.randn(4, 32, device=DEV)
    out = torch.ones(4, 32, device=DEV)
    plan = build_adapter_plan(torch.tensor([0, 1, -1, 0], dtype=torch.int32, device=DEV), 2)
    for call in (lambda: adapter_add(base, x, w, plan, out=out),
                 lambda: control_logits(base, LogitControls(), out=out)):
        leaf = torch.ones(4, 32, device=DEV, requires_grad=True)
        y = (leaf * out).sum()
        call()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.backward()
