"""What the entry points for batches whose requests differ refuse on the host, and the
64-bit restatement that the GPU tests trust, on small cases worked by hand. No kernel is
launched."""
import numpy as np
import pytest
import torch

from oracle import requests_ref as ref
from serving import _native
from serving.adapters import AdapterWeights, _overlap, build_adapter_plan
from serving.controls import LogitControls, RequestParams, control_logits, sample_each
from serving.scheduler import Scheduler


def test_plan_refusals():
    L = _native.lib()

    def plan(order=16, starts=16, tiles=16, places=16, max_tiles=8, ids=16, T=4, n=3, rows=16):
        return L.pkv_adapter_plan(order, starts, tiles, places, max_tiles, ids, T, n, rows, None,
                                  None)

    assert plan(T=-1) == -1 and plan(n=-1) == -1 and plan(rows=32) == -1
    assert plan(max_tiles=3) == -1 and b"max_tiles" in L.pkv_last_error()
    assert plan(ids=None) == -1 and plan(order=None) == -1 and plan(starts=None) == -1
    assert plan(places=None) == -1
    assert plan(tiles=8) == -1 and b"aligned" in L.pkv_last_error()
    assert plan(n=1001, max_tiles=2000) == -2


def test_apply_refusals():
    L = _native.lib()
    good = dict(out=16, os=16, base=32, bs=16, x=48, xs=32, a=64, astr=32, b=80, sc=16, tiles=16,
                places=16, mt=4, rows=16, T=4, N=2, k=32, r=8, parts=1, n0=16, n1=0, n2=0, n3=0,
                epi=0, dt=0, ws=16, wsb=1 << 20)

    def apply(**kw):
        return L.pkv_adapter_apply(*{**good, **kw}.values(), None)

    for kw in (dict(dt=7), dict(epi=2), dict(T=-1), dict(parts=0), dict(parts=5), dict(n0=0),
               dict(k=0), dict(r=0), dict(rows=8), dict(astr=31), dict(astr=40), dict(os=15),
               dict(bs=15), dict(xs=31), dict(out=None), dict(x=None), dict(a=None),
               dict(places=None), dict(sc=None), dict(a=65), dict(tiles=24), dict(epi=1),
               dict(epi=1, parts=2, n1=17, bs=40), dict(ws=24),
               dict(epi=1, parts=2, n1=16, bs=32, out=32)):
        assert apply(**kw) == -1, kw
    assert apply(r=12) == -2 and apply(r=136) == -2 and apply(mt=65536) == -2
    assert apply(ws=None) == -3 and apply(wsb=64) == -3
    assert apply(T=0) == 0 and apply(mt=0) == 0  # nothing to do
    assert L.pkv_adapter_workspace_bytes(0, 4, 16, 32, 8, 1) == 0
    assert L.pkv_adapter_workspace_bytes(4, 4, 16, 32, 8, 1) >= 4 * 8 * 4


def test_control_and_draw_refusals():
    L = _native.lib()
    good = dict(out=16, os=40, x=32, xs=40, rows=2, V=40, tok=16, ts=8, cap=8, lens=16, pl=None,
                rep=None, pres=None, freq=None, bi=None, bv=None, bs=None, nb=0, m=None, nm=0,
                mr=None, dt=0)

    def control(**kw):
        return L.pkv_control_logits(*{**good, **kw}.values(), None, None)

    for kw in (dict(dt=3), dict(rows=-1), dict(V=-1), dict(cap=-1), dict(nb=-1), dict(nm=-1),
               dict(os=39), dict(xs=39), dict(ts=7), dict(out=None), dict(x=None), dict(lens=None),
               dict(bs=16, nb=1), dict(mr=16, nm=1)):
        assert control(**kw) == -1, kw
    assert control(rows=1 << 21) == -2 and control(V=1 << 25, os=1 << 25, xs=1 << 25) == -2
    assert control(rows=0) == 0 and control(V=0) == 0

    def draw(ids=16, x=16, rows=2, V=40, xs=40, temp=16, u=16, dt=0):
        return L.pkv_sample_each(ids, None, x, rows, V, xs, temp, None, None, None, u, dt, None,
                                 None)

    assert draw(dt=3) == -1 and draw(rows=-1) == -1 and draw(V=0) == -1 and draw(xs=39) == -1
    assert draw(ids=None) == -1 and draw(x=None) == -1 and draw(temp=None) == -1
    assert draw(u=None) == -1
    assert draw(V=(1 << 20) + 1, xs=1 << 21) == -2 and draw(rows=1 << 21) == -2
    assert draw(rows=0) == 0


def test_cpu_tensors_are_refused():
    w = AdapterWeights(32, (16,), 2, 4, device="cpu")
    assert w.rank == 8 and w.a.shape == (2, 8, 32) and w.b.shape == (2, 64, 8)
    with pytest.raises(RuntimeError, match="ROCm"):
        build_adapter_plan(torch.zeros(3, dtype=torch.int32), 2)
    with pytest.raises(RuntimeError, match="ROCm"):
        control_logits(torch.zeros(2, 8), LogitControls())
    with pytest.raises(RuntimeError, match="ROCm"):
        sample_each(torch.zeros(2, 8), torch.zeros(2))
    with pytest.raises(ValueError):
        AdapterWeights(32, (16,), 2, 129, device="cpu")
    with pytest.raises(ValueError):
        AdapterWeights(32, (1, 2, 3, 4, 5), 2, 8, device="cpu")
    with pytest.raises(ValueError):
        AdapterWeights(32, (16,), 1001, 8, device="cpu")
    with pytest.raises(TypeError):
        AdapterWeights(32, (16,), 2, 8, dtype=torch.float64, device="cpu")


@pytest.mark.parametrize("k,outs,rank", [(32, (64,), 8), (33, (1, 70, 16), 16), (96, (130,), 24),
                                         (64, (64, 64), 128), (5, (200, 8), 40)])
def test_weights_are_laid_out_as_the_lanes_read_them(k, outs, rank):
    g = torch.Generator().manual_seed(k)
    w = AdapterWeights(k, outs, 2, rank, dtype=torch.float16, device="cpu")
    pairs = [(torch.randn(rank, k, generator=g), torch.randn(n, rank, generator=g)) for n in outs]
    w.load(1, pairs, 2.0)
    a, b = w.unpack(1)
    assert torch.equal(a, torch.cat([p[0] for p in pairs]).half())
    assert torch.equal(b, torch.cat([p[1] for p in pairs]).half())
    ka, flat_a, flat_b = -(-k // 32) * 32, w.a[1].view(-1), w.b[1].view(-1)
    at = 0
    for s, (pa, pb) in enumerate(pairs):
        for r in range(rank):
            r0 = r // 16 * 16
            nr = min(16, rank - r0)
            for c in range(0, k, 7):
                place = (s * rank + r0) * ka + ((c // 8) * nr + r - r0) * 8 + c % 8
                assert flat_a[place] == pa[r, c].half()
        for f in range(pb.shape[0]):
            h, q, l, e = f % 64 // 32, f % 32 // 8, f % 8 // 4, f % 4
            for r in range(0, rank, 3):
                place = ((at + f // 64 * 64) * rank + (r // 8) * 512
                         + ((2 * h + l) * 16 + 4 * q + e) * 8 + r % 8)
                assert flat_b[place] == pb[f, r].half()
        at += -(-pb.shape[0] // 64) * 64
    w.load(1, [None] * len(outs))
    assert not w.a.any() and not w.b.any()


def test_parameters_are_checked_as_the_kernels_get_them():
    for kw in (dict(temperature=-1), dict(temperature=float("nan")), dict(temperature=1e39),
               dict(top_k=-1), dict(top_p=0.0), dict(top_p=1e-60), dict(top_p=1.5),
               dict(min_p=-0.1), dict(min_p=1.5), dict(repetition_penalty=0.0),
               dict(repetition_penalty=1e-60), dict(repetition_penalty=1e39),
               dict(presence_penalty=float("inf")), dict(frequency_penalty=1e39),
               dict(logit_bias={-1: 1.0}), dict(logit_bias={1 << 31: 1.0}),
               dict(logit_bias={3: float("nan")}), dict(logit_bias={3: 1e39})):
        with pytest.raises(ValueError):
            RequestParams(**kw)
    bias = {3: -1e39, 4: 2}
    p = RequestParams(temperature=0, top_p=1, repetition_penalty=1e-30, logit_bias=bias)
    bias[4] = float("nan")  # the request keeps its own
    assert p.logit_bias[4] == 2
    assert RequestParams(logit_bias={"7": np.float32(1.5)}).logit_bias == {7: 1.5}
    with pytest.raises(AttributeError):
        p.top_p = 2.0


def test_a_model_on_the_cpu_takes_no_params():
    model = torch.nn.Module()
    model.lm_head = torch.nn.Linear(4, 8)
    sched = Scheduler(model, None, None, None)
    with pytest.raises(RuntimeError, match="ROCm"):
        sched.add_request([1], 2, params=RequestParams())
    sched.add_request([1], 2)


def test_overlap():
    b = torch.zeros(8, 32)
    assert _overlap(b[:4], b[3:]) and not _overlap(b[:4], b[4:])
    assert not _overlap(b[:, :16], b[:, 16:]) and _overlap(b[:, :17], b[:, 16:])
    assert not _overlap(b[1:, :16], b[:, 16:])  # the same columns a row on
    assert _overlap(b[:, 8:24], b.view(4, 64)) and not _overlap(b[:0], b)


def test_restated_plan_and_adapters():
    order, starts, tiles = ref.plan([1, -1, 0, 1, 9], 2, 2)
    assert order == [2, 0, 3, 1, 4] and starts == [0, 1, 3, 5]
    assert tiles == [[0, 0, 1, 0], [1, 1, 2, 0], [-1, 3, 2, 0]]
    x, base = torch.tensor([[1.0, 2.0], [3.0, 4.0]]), torch.tensor([[10.0, 20.0], [30.0, 40.0]])
    a = torch.tensor([[[1.0, 0.0], [0.0, 1.0]]])      # two parts of rank 1: x0, x1
    b = torch.tensor([[[2.0], [3.0]]])
    y = ref.adapted(base, x, a, b, torch.tensor([0.5]), [0, -1], (1, 1), 1)
    assert y.tolist() == [[11.0, 23.0], [30.0, 40.0]]


def test_restated_controls():
    got = ref.control([2.0, -2.0, 1.0, 0.0], [0, 1, 1, 9], 1, 2.0, 0.5, 0.25, [(2, 1.0), (2, 2.0)],
                      np.array([True, True, True, False]))
    assert got.tolist() == [1.0, -4.0 - 0.5 - 0.5, 4.0, -np.inf]


def test_restated_draws():
    row = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert ref.draw(row, 0, 0, 1, 0, 0.5)[0] == 1
    assert [ref.draw(row, 1.0, 0, 1, 0, u)[0] for u in (0.05, 0.3, 0.65, 0.9)] == [0, 1, 2, 3]
    assert np.allclose(ref.kept(row, 1.0, 2, 1, 0), [0, 1, 0, 0.75])
    assert np.allclose(ref.kept(row, 1.0, 0, 0.5, 0), [0, 1, 0, 0.75])  # 0.4 before the second
    assert np.allclose(ref.kept(row, 1.0, 0, 0.39, 0), [0, 1, 0, 0])
    assert np.allclose(ref.kept(row, 1.0, 0, 1, 0.6), [0, 1, 0, 0.75])
    assert np.allclose(ref.kept(np.zeros(4), 1.0, 2, 1, 0), [1, 1, 1, 1])  # ties of the second
    assert np.allclose(ref.kept(np.zeros(4), 1.0, 0, 0.3, 0), [1, 1, 0, 0])  # by index
