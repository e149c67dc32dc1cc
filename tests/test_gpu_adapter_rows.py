"""Rows without an adapter in a step of the model in which others name one."""
import pytest
import torch

from serving.adapters import AdapterSet
from serving.allocator import BlockAllocator
from serving.batch import build_batch_step
from serving.sequence import Sequence
from test_gpu_requests import adapter_state, make_model, pool_of, prompts_of

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d_model,heads", [(128, 4), (256, 4), (512, 8), (1024, 8)])
def test_rows_without_an_adapter_keep_their_bits_in_long_steps(dtype, d_model, heads):
    """More than 256 rows, which other projection kernels take than a decode step's; also of
    sets that adapt some projections only."""
    model, cfg = make_model(dtype, d_model, heads)
    prompts, alloc = prompts_of([100, 90, 130, 2]), BlockAllocator(64)
    seqs = [Sequence(n, p, 16) for n, p in enumerate(prompts)]
    for s in seqs:
        s.ensure_blocks(alloc)
    batch = build_batch_step([(s, s.token_ids) for s in seqs], DEV)
    plain = model.forward_batch(batch, pool_of(cfg))
    for names, skip in ((("qkv", "out", "gate_up", "down"), ()), (("qkv",), ("out", "mlp")),
                        (("gate_up", "down"), ("attn",))):
        weights = AdapterSet(model, 2, 8, projections=names)
        weights.load(1, adapter_state(model, 3, 8, skip=skip), 1.0)
        mixed = model.forward_batch(batch, pool_of(cfg), weights, [-1, 1, -1, 1])
        assert torch.equal(plain[0], mixed[0]) and torch.equal(plain[2], mixed[2]), names
        assert not torch.equal(plain[1], mixed[1]), names
