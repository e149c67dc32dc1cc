"""Adapter products at the sizes of wide models and prompts: k in three to eight pieces, two
pieces under tiles of 64 rows, and every number of blocks of ranks a workgroup takes. Problems
and tolerances are those of tests/test_gpu_adapters.py."""
import pytest
import torch

from serving.adapters import adapter_add, adapter_swiglu, build_adapter_plan
from test_gpu_adapters import check_add, check_gate, expected, i32, problem

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [  # T, adapters, k, outs, rank
    (20, 3, 4096, (64,), 16),              # eight pieces of k
    (20, 3, 4096 - 8, (64, 16), 8),        # the last piece shorter
    (9, 2, 4096 - 31, (64,), 24),          # and its last step inside x's rows
    (17, 3, 1536, (40,), 16),              # three pieces
    (40, 5, 2500, (72, 8, 8), 16),         # five
    (700, 400, 2048, (64,), 16),           # many tiles: fewer pieces than k would give
    (1500, 3, 1100, (64,), 16),            # tiles of 64 rows, two pieces, one block of ranks
    (1100, 3, 1056, (64, 16, 16), 16),     # three blocks
    (1030, 2, 4096, (48, 16), 16),         # two
    (1025, 2, 777, (33, 5), 40),           # six, in two turns
    (1200, 300, 600, (40,), 64),           # four, tiles of a few rows
])
def test_adapter_add_in_pieces(shape, dtype):
    print(f"[add] {shape} {dtype}", flush=True)
    T, n, k, outs, rank = shape
    ids, w, x, base, R = problem(T, n, k, outs, rank, dtype)
    plan = build_adapter_plan(i32(ids), n)
    y, off = expected(ids, w, x, base, R)
    xd, bd = x.to(DEV), base.to(DEV)
    out = adapter_add(bd, xd, w, plan)
    check_add(out, y, off, dtype)
    none = [t for t, i in enumerate(ids) if i < 0]
    assert torch.equal(out.cpu()[none], base[none])
    assert adapter_add(bd, xd, w, plan, out=bd) is bd and torch.equal(bd, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [
    (20, 3, 4096, (64, 64), 16), (33, 4, 1700, (72, 72), 40), (1100, 3, 1056, (64, 64), 16),
    (1030, 2, 700, (40, 40), 8)])
def test_adapter_swiglu_in_pieces(shape, dtype):
    print(f"[swiglu] {shape} {dtype}", flush=True)
    T, n, k, outs, rank = shape
    ids, w, x, base, R = problem(T, n, k, outs, rank, dtype)
    plan = build_adapter_plan(i32(ids), n)
    y, off = expected(ids, w, x, base, R)
    check_gate(adapter_swiglu(base.to(DEV), x.to(DEV), w, plan), y, off, dtype)
