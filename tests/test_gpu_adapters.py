"""Low-rank adapters of many requests (serving/adapters.py) against the 64-bit restatement
oracle/requests_ref.py.

Tolerance of a result y: half a step of its type on |y|; the fp32 sums of k and of rank
terms, at most (k + rank + 8) 2^-24 of the sum of the terms' magnitudes M; and, for 16-bit
types, A x as the sum of two 16-bit values: bf16 leaves 2^-18 of each value, fp16 2^-24 of
the row's largest (the second value's smallest step). Through the gate an error d of its
inputs grows at most to 1.1 |up| d and |silu(gate)| d, and its own fp32 operations (the
exponential's error is relative to its argument) add 16 (1 + |gate|) 2^-24 of the result."""
import pytest
import torch

from oracle import requests_ref as ref
from serving import _native, fused_ops
from serving.adapters import AdapterWeights, adapter_add, adapter_swiglu, build_adapter_plan

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def gen(*seed):
    return torch.Generator().manual_seed(hash(seed) % (1 << 31))


def random_ids(T, n, none, g):
    ids = torch.randint(0, n, (T,), generator=g)
    return torch.where(torch.rand(T, generator=g) < none, -1, ids).tolist()


def check_plan(ids, n):
    plan = build_adapter_plan(i32(ids), n)
    order, starts, tiles = ref.plan(ids, n, plan.tile_rows)
    assert plan.order.tolist() == order and plan.starts.tolist() == starts
    got = plan.tiles.tolist()
    assert got[:len(tiles)] == tiles
    assert all(t[2] == 0 for t in got[len(tiles):])
    rows = plan.rows.tolist()
    for (_, first, n_rows, _), places in zip(tiles, rows):
        want = order[first:first + n_rows]
        assert places == want + want[-1:] * (plan.tile_rows - n_rows)
    return plan


@pytest.mark.parametrize("T", [0, 1, 2, 15, 16, 17, 63, 64, 65, 255, 1023, 1024, 1025, 5000])
@pytest.mark.parametrize("n", [0, 1, 2, 7, 255, 1000])
def test_plan(T, n):
    print(f"[plan] T={T} n={n}", flush=True)
    for none in (0.0, 0.3, 1.0):
        g = gen(T, n, none)
        check_plan(random_ids(T, n, none, g) if n else [-1] * T, n)


def test_plan_of_one_adapter_and_of_many_rows():
    check_plan([4] * 70000, 5)
    g = gen(3)
    check_plan(random_ids(100003, 999, 0.2, g), 999)


@pytest.mark.parametrize("lens", [[256] * 16, [4096, 1, 255, 257, 4096], [512, 300, 1200, 64] * 4,
                                  [16384], [16383, 1], [1000] * 17])
def test_plan_of_prompts(lens):
    """Runs of rows of one adapter, some of them of the same."""
    ids = [a for i, n in enumerate(lens) for a in [(5 * i) % 7 - 1] * n]
    check_plan(ids, 6)
    bad = list(ids)
    bad[len(ids) // 2] = 6
    st = status()
    plan = build_adapter_plan(i32(bad), 6, status=st)
    assert int(st) == _native.PKV_STATUS_BAD_CONTROL
    bad[len(ids) // 2] = -1
    assert plan.order.tolist() == ref.plan(bad, 6, plan.tile_rows)[0]


def test_plan_reports_ids_of_no_adapter():
    ids = [0, 5, -1, 2, -7, 1, 2 ** 31 - 1, -2 ** 31]
    st = status()
    plan = build_adapter_plan(i32(ids), 5, status=st)
    order, starts, _ = ref.plan(ids, 5, 16)
    assert plan.order.tolist() == order and plan.starts.tolist() == starts
    assert int(st) == _native.PKV_STATUS_BAD_CONTROL
    st = status()
    build_adapter_plan(i32([0, -1, 4]), 5, status=st)
    assert int(st) == 0
    strided = i32([1, 9, 0, 9, 3, 9])[::2]
    assert build_adapter_plan(strided, 4).order.tolist() == [1, 0, 2]


def problem(T, n, k, outs, rank, dtype, none=0.3, r=None):
    g = gen(T, n, k, *outs, rank)
    ids = random_ids(T, n, none, g)
    R = -(-rank // 8) * 8
    w = AdapterWeights(k, outs, n, rank, dtype=dtype, device=DEV)
    for i in range(n):
        parts = [((torch.randn(rank, k, generator=g) * k ** -0.5).to(dtype),
                  (torch.randn(m, rank, generator=g) * rank ** -0.5).to(dtype)) for m in outs]
        w.load(i, parts, float(torch.rand(1, generator=g)) + 0.5)
    x = torch.randn(T, k, generator=g).to(dtype)
    base = torch.randn(T, sum(outs), generator=g).to(dtype)
    return ids, w, x, base, R


def expected(ids, w, x, base, R):
    """(64-bit result, what an fp32 computation of it may be off before its rounding)."""
    a, b = (torch.stack(t).cpu() for t in zip(*(w.unpack(i) for i in range(w.num_adapters))))
    sc = w.scales.cpu()
    outs, k = w.out_features, w.in_features
    y = ref.adapted(base, x, a, b, sc, ids, outs, R)
    terms = ref.adapted_bound(torch.zeros_like(base), x, a, b, sc, ids, outs, R)
    off = (k + R + 8) * 2.0 ** -24 * (terms + base.double().abs())
    if w.dtype == torch.bfloat16:
        off += 2.0 ** -18 * terms
    elif w.dtype == torch.float16:
        for t, i in enumerate(ids):
            if i < 0:
                continue
            low = float(sc[i]) * (a[i].double().abs() @ x[t].double().abs())
            at = 0
            for s, n in enumerate(outs):
                most = low[s * R:(s + 1) * R].max()
                off[t, at:at + n] += 2.0 ** -24 * most * b[i, at:at + n].double().abs().sum(1)
                at += n
    return y, off


def check_add(got, y, off, dtype):
    err = (got.cpu().double() - y).abs()
    tol = torch.finfo(dtype).eps / 2 * (y.abs() + off) + off
    assert bool((err <= tol).all()), f"worst {float((err - tol).max())}"


def check_gate(got, y, off, dtype):
    gate, up = y.chunk(2, 1)
    dg, du = off.chunk(2, 1)
    out = ref.swiglu(y)
    silu = gate * torch.sigmoid(gate)
    d = 1.1 * (up.abs() + du) * dg + silu.abs() * du + 16 * 2.0 ** -24 * (1 + gate.abs()) * out.abs()
    err = (got.cpu().double() - out).abs()
    tol = torch.finfo(dtype).eps / 2 * (out.abs() + d) + d + torch.finfo(dtype).tiny
    assert bool((err <= tol).all()), f"worst {float((err - tol).max())}"


SHAPES = [  # T, adapters, k, outs, rank
    (1, 1, 64, (64,), 8),
    (5, 3, 512, (512,), 8),
    (33, 4, 200, (72,), 4),            # rank below 8
    (64, 24, 1024, (1024, 64, 64), 16),
    (100, 5, 320, (96, 32), 24),
    (37, 6, 333, (77, 5, 3), 12),      # nothing a multiple of 8
    (17, 2, 40, (1,), 1),
    (256, 2, 512, (264,), 64),
    (130, 3, 136, (520, 8, 8, 16), 128),
    (1500, 4, 256, (256,), 32),        # tiles of 64 rows
    (1100, 7, 77, (130, 34), 20),
    (1024, 1, 96, (64, 64), 128),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_adapter_add(shape, dtype):
    print(f"[add] {shape} {dtype}", flush=True)
    T, n, k, outs, rank = shape
    ids, w, x, base, R = problem(T, n, k, outs, rank, dtype)
    plan = build_adapter_plan(i32(ids), n)
    y, off = expected(ids, w, x, base, R)
    xd, bd = x.to(DEV), base.to(DEV)
    out = adapter_add(bd, xd, w, plan)
    check_add(out, y, off, dtype)
    assert torch.equal(bd.cpu(), base)
    none = [t for t, i in enumerate(ids) if i < 0]
    assert torch.equal(out.cpu()[none], base[none])  # rows without an adapter: bit for bit
    # in place, and into a part of a wider buffer
    wide = torch.full((T, sum(outs) + 24), 7.0, dtype=dtype, device=DEV)
    assert adapter_add(bd, xd, w, plan, out=wide[:, 8:8 + sum(outs)]) is not None
    assert torch.equal(wide[:, 8:8 + sum(outs)], out)
    assert bool((wide[:, :8] == 7).all()) and bool((wide[:, 8 + sum(outs):] == 7).all())
    assert adapter_add(bd, xd, w, plan, out=bd) is bd
    assert torch.equal(bd, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [s for s in (
    (1, 1, 64, (64, 64), 8), (50, 4, 200, (136, 136), 16), (37, 3, 75, (33, 33), 12),
    (128, 16, 1024, (512, 512), 16), (300, 2, 264, (520, 520), 128),
    (1300, 5, 512, (256, 256), 32), (1025, 3, 99, (51, 51), 128))])
def test_adapter_swiglu(shape, dtype):
    print(f"[swiglu] {shape} {dtype}", flush=True)
    T, n, k, outs, rank = shape
    ids, w, x, base, R = problem(T, n, k, outs, rank, dtype)
    plan = build_adapter_plan(i32(ids), n)
    y, off = expected(ids, w, x, base, R)
    xd, bd = x.to(DEV), base.to(DEV)
    out = adapter_swiglu(bd, xd, w, plan)
    check_gate(out, y, off, dtype)
    none = [t for t, i in enumerate(ids) if i < 0]
    plain = fused_ops.silu_mul(bd[:, :outs[0]], bd[:, outs[0]:])
    assert torch.equal(out[none], plain[none])
    wide = torch.full((T, outs[0] + 16), 7.0, dtype=dtype, device=DEV)
    adapter_swiglu(bd, xd, w, plan, out=wide[:, :outs[0]])
    assert torch.equal(wide[:, :outs[0]], out) and bool((wide[:, outs[0]:] == 7).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("offset", [0, 1, 8])
def test_rows_of_wider_buffers_at_any_alignment(offset, dtype):
    T, n, k, outs, rank = 40, 3, 64, (48, 16), 16
    ids, w, x, base, R = problem(T, n, k, outs, rank, dtype)
    plan = build_adapter_plan(i32(ids), n)
    xw = torch.randn(T, k + 19, device=DEV).to(dtype)
    bw = torch.randn(T, sum(outs) + 19, device=DEV).to(dtype)
    xw[:, offset:offset + k] = x.to(DEV)
    bw[:, offset:offset + sum(outs)] = base.to(DEV)
    keep = bw.clone()
    out = adapter_add(bw[:, offset:offset + sum(outs)], xw[:, offset:offset + k], w, plan)
    assert torch.equal(out, adapter_add(base.to(DEV), x.to(DEV), w, plan))
    view = bw[:, offset:offset + sum(outs)]
    adapter_add(view, xw[:, offset:offset + k], w, plan, out=view)
    keep[:, offset:offset + sum(outs)] = out
    assert torch.equal(bw, keep)
    # transposed operands are copied
    assert torch.equal(adapter_add(base.to(DEV).t().contiguous().t(),
                                   x.to(DEV).t().contiguous().t(), w, plan), out)


def test_nobody_and_nothing():
    w = AdapterWeights(32, (16,), 3, 8, dtype=torch.bfloat16, device=DEV)
    x, base = torch.randn(5, 32, device=DEV).bfloat16(), torch.randn(5, 16, device=DEV).bfloat16()
    for ids in ([-1] * 5, [0, 1, 2, 0, 1]):  # no adapter, and adapters that were not loaded
        plan = build_adapter_plan(i32(ids), 3)
        assert torch.equal(adapter_add(base, x, w, plan), base)
    empty = build_adapter_plan(i32([]), 3)
    assert adapter_add(base[:0], x[:0], w, empty).shape == (0, 16)
    # cleared again
    w.load(1, [(torch.randn(8, 32), torch.randn(16, 8))], 2.0)
    plan = build_adapter_plan(i32([1] * 5), 3)
    assert not torch.equal(adapter_add(base, x, w, plan), base)
    w.clear(1)
    assert torch.equal(adapter_add(base, x, w, plan), base)


def test_load_replaces_all_of_an_adapter():
    """A smaller adapter after a larger one, and parts without one."""
    g = gen(9)
    w = AdapterWeights(24, (16, 8), 2, 16, dtype=torch.float32, device=DEV)
    big = [(torch.randn(16, 24, generator=g), torch.randn(16, 16, generator=g)),
           (torch.randn(16, 24, generator=g), torch.randn(8, 16, generator=g))]
    w.load(0, big, 1.5)
    small = (torch.randn(3, 24, generator=g), torch.randn(16, 3, generator=g))
    w.load(0, [small, None], 0.5)
    fresh = AdapterWeights(24, (16, 8), 2, 16, dtype=torch.float32, device=DEV)
    fresh.load(0, [small, None], 0.5)
    assert torch.equal(w.a, fresh.a) and torch.equal(w.b, fresh.b)
    assert torch.equal(w.scales, fresh.scales)


@pytest.mark.parametrize("dtype", TYPES)
def test_values_that_are_not_finite_stay_in_their_rows(dtype):
    T, n, k, outs, rank = 70, 3, 64, (64,), 16
    ids, w, x, base, R = problem(T, n, k, outs, rank, dtype)
    ids[0], ids[1], ids[2], ids[3] = 0, 1, 1, 0
    plan = build_adapter_plan(i32(ids), n)
    clean = adapter_add(base.to(DEV), x.to(DEV), w, plan)
    x2, b2 = x.clone(), base.clone()
    x2[0, 5], x2[1, 7], b2[2, 3] = float("nan"), float("inf"), float("-inf")
    out = adapter_add(b2.to(DEV), x2.to(DEV), w, plan)
    assert torch.equal(out[3:], clean[3:])
    assert bool(out[0].isnan().all()) and not bool(out[1].isfinite().any())
    assert float(out[2, 3]) == float("-inf") and torch.equal(out[2, 4:], clean[2, 4:])
    # an adapter of NaN reaches its own rows only
    w.a[2].fill_(float("nan"))
    w.b[2].fill_(float("inf"))
    out = adapter_add(base.to(DEV), x.to(DEV), w, plan)
    other = [t for t, i in enumerate(ids) if i != 2]
    assert torch.equal(out[other], clean[other])


def test_fp16_rows_far_from_one():
    """A x beyond fp16's largest value, and far below its smallest steps."""
    T, n, k, outs, rank = 48, 2, 64, (64,), 16
    ids, w, x, base, R = problem(T, n, k, outs, rank, torch.float16, none=0.0)
    w.a.mul_(torch.tensor([600.0, 2.0 ** -9], device=DEV)[:, None, None])
    w.b.mul_(torch.tensor([2.0 ** -8, 64.0], device=DEV)[:, None, None])
    w.scales.mul_(torch.tensor([400.0, 2.0 ** -14], device=DEV))
    base.zero_()
    y, off = expected(ids, w, x, base, R)
    assert float(y.abs().max()) < 60000
    out = adapter_add(base.to(DEV), x.to(DEV), w, build_adapter_plan(i32(ids), n))
    err = (out.cpu().double() - y).abs()
    # below the smallest normal half a step is 2^-25
    assert bool((err <= 2.0 ** -11 * y.abs() + off + 2.0 ** -25).all())


def test_refusals():
    w = AdapterWeights(32, (16,), 3, 8, dtype=torch.float32, device=DEV)
    x, base = torch.randn(5, 32, device=DEV), torch.randn(5, 16, device=DEV)
    plan = build_adapter_plan(i32([0, 1, 2, -1, 0]), 3)
    with pytest.raises(ValueError, match="base must be"):
        adapter_add(base[:4], x[:4], w, plan)
    with pytest.raises(ValueError, match="base must be"):
        adapter_add(base, x[:, :31], w, plan)
    with pytest.raises(TypeError):
        adapter_add(base.bfloat16(), x, w, plan)
    with pytest.raises(ValueError, match="adapters"):
        adapter_add(base, x, w, build_adapter_plan(i32([0, 1, 2, -1, 0]), 4))
    with pytest.raises(ValueError, match="two parts"):
        adapter_swiglu(base, x, w, plan)
    with pytest.raises(ValueError, match="shares memory"):
        adapter_add(base, x, w, plan, out=x[:, :16])
    buf = torch.randn(7, 16, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):
        adapter_add(buf[:5], x, w, plan, out=buf[1:6])
    with pytest.raises(ValueError, match="out must be"):
        adapter_add(base, x, w, plan, out=torch.empty(5, 15, device=DEV))
    with pytest.raises(ValueError, match="unit column stride"):
        adapter_add(base, x, w, plan, out=torch.empty(16, 5, device=DEV).t())
    with pytest.raises(NotImplementedError):
        adapter_add(base.requires_grad_(), x, w, plan)
    with pytest.raises(RuntimeError):
        adapter_add(base.detach().cpu(), x, w, plan)
    with pytest.raises(ValueError, match="int32"):
        build_adapter_plan(torch.zeros(3, dtype=torch.int64, device=DEV), 2)
    with pytest.raises(ValueError, match="at most"):
        build_adapter_plan(i32([0]), 1001)
    with pytest.raises(IndexError):
        w.load(3, [(torch.randn(8, 32), torch.randn(16, 8))])
    with pytest.raises(ValueError, match="r up to"):
        w.load(0, [(torch.randn(9, 32), torch.randn(16, 9))])
    with pytest.raises(ValueError, match="parts"):
        w.load(0, [])


def test_the_same_bits_every_time_and_on_another_stream():
    T, n, k, outs, rank = 200, 6, 1024, (512, 64, 64), 16
    ids, w, x, base, R = problem(T, n, k, outs, rank, torch.bfloat16)
    xd, bd, di = x.to(DEV), base.to(DEV), i32(ids)
    first = adapter_add(bd, xd, w, build_adapter_plan(di, n))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [adapter_add(bd, xd, w, build_adapter_plan(di, n)) for _ in range(5)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(first, o) for o in got)


def test_two_streams_and_two_graphs_at_once():
    """Plans and scratch of calls in flight together are their own."""
    work, want, graphs, outs = [], [], [], []
    for T, n, k, parts, rank in ((200, 6, 1024, (512, 512), 16), (1500, 3, 512, (256, 256), 40)):
        ids, w, x, base, R = problem(T, n, k, parts, rank, torch.bfloat16)
        work.append((i32(ids), x.to(DEV), base.to(DEV), w, n))

    def step(ids, x, base, w, n):
        plan = build_adapter_plan(ids, n)
        return adapter_add(base, x, w, plan), adapter_swiglu(base, x, w, plan)

    want = [step(*a) for a in work]
    torch.cuda.synchronize()
    for a in work:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        eager = [None, None]
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                eager[1 - i] = step(*work[1 - i])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(want[i], outs[i]))
            assert all(torch.equal(a, b) for a, b in zip(want[i], eager[i]))


def test_rows_that_are_gigabytes_apart():
    T, n, k, parts, rank = 5, 2, 96, (64, 32), 8
    ids, w, x, base, R = problem(T, n, k, parts, rank, torch.bfloat16)
    far = (1 << 30) - 8  # the last rows begin past 2^31 elements
    buf = torch.empty(4 * far + 512, dtype=torch.bfloat16, device=DEV)
    xd, bd = buf.as_strided((T, k), (far, 1)), buf[256:].as_strided((T, sum(parts)), (far, 1))
    xd.copy_(x)
    bd.copy_(base)
    plan = build_adapter_plan(i32(ids), n)
    want = adapter_add(base.to(DEV), x.to(DEV), w, plan)
    assert torch.equal(adapter_add(bd, xd, w, plan), want)
    assert torch.equal(adapter_add(bd, xd, w, plan, out=bd), want)


def test_in_a_graph_with_the_plan():
    """Ids, x and base change between replays; eager calls run in between."""
    T, n, k, outs, rank = 64, 5, 256, (128, 128), 16
    ids, w, x, base, R = problem(T, n, k, outs, rank, torch.bfloat16)
    di, xd, bd = i32(ids), x.to(DEV), base.to(DEV)

    def step():
        plan = build_adapter_plan(di, n)
        return adapter_add(bd, xd, w, plan), adapter_swiglu(bd, xd, w, plan)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for r in range(4):
        g = gen(r, 77)
        di.copy_(i32(random_ids(T, n, 0.3, g)))
        xd.copy_(torch.randn(T, k, generator=g).bfloat16())
        bd.copy_(torch.randn(T, sum(outs), generator=g).bfloat16())
        graph.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, eager))
