"""paged_tree_attention against the 64-bit definition (oracle/tree_ref.py).

Tolerances, per output element, with u = half a step of the output type, A the
softmax-weighted mean of |v|, S the largest scale * sum |q_i k_i| of the row, L its
number of keys, e = 2^-24:
  - a score is a sum of d products in fp32 (16-bit products are exact in it), times
    the scale and minus the maximum: off by at most (d + 8) e S, which moves the
    softmax's weights by at most twice that, relative: 2 (d + 8) e S A;
  - the sums over L keys (weights, and weighted values) and the join of
    partitions: 2 (L + 16) e A, exponentials included (2 ulp);
  - 16-bit operands: the weights are rounded to the type, u A, in fp16 with steps
    no finer than 2^-24: half of that for every key, against a sum of at
    least 1 (the largest weight counts 1 or more): 2^-25 V1, V1 = sum |v|;
  - the result is rounded once: u |out|.
lse: the score's error, (L + 16) e for the sum and its logarithm, and one rounding.
"""
import numpy as np
import pytest
import torch

from oracle import tree_ref
from serving import _native
from serving.paged_meta import DeviceTables
from serving.tree_decode import TreeMeta, build_tree_meta, paged_tree_attention

pytestmark = pytest.mark.gpu
DEV = "cuda"
E = 2.0 ** -24


def np64(t):
    return t.detach().cpu().double().numpy() if t.dtype != torch.float8_e4m3fn \
        else t.detach().cpu().float().double().numpy()


def random_parents(rng, n):
    return np.array([-1] + [int(rng.integers(max(0, i - 4), i)) for i in range(1, n)],
                    dtype=np.int32)[:n]


class Problem:
    """Random pools, tables over shuffled blocks, trees; `fill` in every slot that no
    context owns."""

    def __init__(self, ctx, nodes, hq, hkv, d, bs, dtype, kv=None, seed=0, fill=None,
                 parents=None, amp=1.0):
        rng = np.random.default_rng(seed)
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.nodes, self.bs = list(ctx), list(nodes), bs
        held = [-(-c // bs) for c in ctx]
        self.nb = sum(held) + 3
        perm = rng.permutation(np.arange(1, self.nb))
        at = np.concatenate([[0], np.cumsum(held)])
        self.tables = [perm[at[i]:at[i + 1]].tolist() for i in range(len(ctx))]
        self.qsl = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int64)
        T = int(self.qsl[-1])
        kv = kv or dtype
        mk = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.kp, self.vp = mk(self.nb, bs, hkv, d).to(kv), mk(self.nb, bs, hkv, d).to(kv)
        if fill is not None:
            free = np.ones(self.nb * bs, dtype=bool)
            for row, c in zip(self.tables, ctx):
                p = np.arange(c)
                free[np.asarray(row, dtype=np.int64)[p // bs] * bs + p % bs] = False
            idx = torch.from_numpy(np.nonzero(free)[0])
            for pool in (self.kp, self.vp):
                flat = pool.float().view(-1, hkv, d)
                flat[idx] = fill
                pool.copy_(flat.view(pool.shape).to(kv))
        self.q, self.k, self.v = (amp * mk(T, hq, d)).to(dtype), mk(T, hkv, d).to(dtype), \
            mk(T, hkv, d).to(dtype)
        self.parents = [random_parents(rng, n) for n in nodes] if parents is None else parents
        self.vis = [tree_ref.visible_from_parents(p)[0] for p in self.parents]
        self.dtype, self.kv = dtype, kv

    def device_tables(self, width=None):
        width = max([len(t) for t in self.tables] + [1]) if width is None else width
        return DeviceTables.from_host(self.tables, self.ctx, [], width, self.bs, self.nb, DEV)

    def meta(self, max_nodes=0, max_ctx=0):
        flat = np.concatenate([np.asarray(p, dtype=np.int32) for p in self.parents])
        return build_tree_meta(self.device_tables(), torch.from_numpy(flat).to(DEV),
                               torch.from_numpy(self.qsl.astype(np.int32)).to(DEV),
                               max_nodes or max(self.nodes), max_ctx or max(self.ctx))

    def expect(self, scale=None):
        k, v = self.k, self.v
        if self.kv == torch.float8_e4m3fn:
            k, v = k.to(self.kv), v.to(self.kv)
        return tree_ref.tree_attention(np64(self.q), np64(k), np64(v), np64(self.kp),
                                       np64(self.vp), self.tables, self.ctx, self.qsl, self.vis,
                                       scale)

    def run(self, meta=None, **kw):
        lse = torch.full(self.q.shape[:2], 7.0, device=DEV)
        out = paged_tree_attention(self.q.to(DEV), self.k.to(DEV), self.v.to(DEV),
                                   self.kp.to(DEV), self.vp.to(DEV), meta or self.meta(),
                                   lse=lse, **kw)
        return out, lse


def check(p, out, lse, scale=None):
    eo, el, A, S, V1 = p.expect(scale)
    d = eo.shape[-1]
    L = np.zeros(eo.shape[:1])
    for s, vis in enumerate(p.vis):
        L[p.qsl[s]:p.qsl[s + 1]] = p.ctx[s] + vis.sum(1)
    L = L[:, None]
    score = (d + 8) * E * S
    tol = (2 * score + 2 * (L + 16) * E)[..., None] * A
    u = torch.finfo(p.dtype).eps / 2
    if p.dtype != torch.float32:
        tol = tol + u * A
        if p.dtype == torch.float16:
            tol = tol + 2.0 ** -25 * V1
    tol = tol + u * np.abs(eo) * (1 + 2.0 ** -6) + 1e-30
    got = np64(out)
    worst = float((np.abs(got - eo) / tol).max()) if np.isfinite(got).all() else np.nan
    assert worst <= 1
    gl = np64(lse)
    fin = np.isfinite(el)
    assert np.array_equal(np.isposinf(gl), ~fin)
    ltol = score + (L + 16) * E + np.abs(np.where(fin, el, 0)) * 2 * E + 1e-6
    assert float((np.abs(gl[fin] - el[fin]) / ltol[fin]).max(initial=0)) <= 1


BF, HF, F32, F8 = torch.bfloat16, torch.float16, torch.float32, torch.float8_e4m3fn

CASES = [  # ctx, nodes, hq, hkv, d, bs, dtype, pool dtype
    ([70, 0, 1, 33], [5, 3, 1, 8], 8, 1, 64, 16, F32, None),
    ([70, 0, 1, 33], [5, 3, 1, 8], 8, 1, 64, 16, BF, None),
    ([200, 16, 15, 17], [4, 1, 2, 4], 8, 1, 128, 16, BF, None),
    ([131, 0, 64], [7, 33, 1], 16, 1, 64, 16, HF, None),
    ([300, 5], [20, 31], 32, 1, 128, 32, BF, None),
    ([300, 5], [20, 31], 32, 1, 128, 8, BF, F8),
    ([90, 257, 1], [3, 2, 1], 4, 1, 32, 16, HF, F8),
    ([90, 257, 1], [3, 2, 1], 4, 1, 32, 1, F32, None),
    ([47, 129], [5, 9], 12, 4, 80, 16, BF, None),
    ([47, 129], [5, 9], 12, 4, 80, 16, F32, None),
    ([47, 129], [5, 9], 6, 6, 96, 4, HF, F8),
    ([65, 31], [6, 3], 8, 1, 256, 16, BF, None),
    ([65, 31], [6, 3], 8, 2, 256, 16, F32, None),
    ([40, 100], [2, 5], 3, 3, 8, 16, BF, F8),
    ([40, 100], [2, 5], 3, 3, 8, 2, F32, None),
    ([40, 100], [2, 60], 6, 2, 128, 16, F32, None),
    ([10, 1000], [130, 67], 4, 2, 64, 16, BF, None),
    ([10, 200], [130, 300], 2, 1, 32, 64, F32, None),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("part", [0, 64])
def test_matches_definition(case, part):
    ctx, nodes, hq, hkv, d, bs, dt, kv = CASES[case]
    print(f"[tree] {CASES[case]} part={part}", flush=True)
    p = Problem(ctx, nodes, hq, hkv, d, bs, dt, kv, seed=case)
    check(p, *p.run(part_tokens=part))


@pytest.mark.parametrize("n", [64, 65, 257, 321])
@pytest.mark.parametrize("dt,hq,part", [(BF, 4, 64), (BF, 40, 0), (F32, 4, 0)])
def test_many_sequences(n, dt, hq, part):
    """Plans of several rounds of 64 sequences, some of them without nodes."""
    print(f"[tree] n={n} {dt} hq={hq} part={part}", flush=True)
    rng = np.random.default_rng(n)
    ctx = rng.integers(0, 40, size=n)
    ctx[::50] = 300
    nodes = rng.integers(0, 4, size=n)
    nodes[-1] = 2
    p = Problem(ctx.tolist(), nodes.tolist(), hq, 1, 64, 16, dt, seed=n)
    check(p, *p.run(part_tokens=part))


@pytest.mark.parametrize("dt,kv,d,bs,nodes", [(BF, None, 128, 16, [3, 2]), (BF, F8, 64, 16, [9, 40]),
                                              (F32, None, 64, 32, [5, 1]), (HF, None, 64, 8, [3, 20])])
@pytest.mark.parametrize("part", [8192, 2048])
def test_long_partitions(dt, kv, d, bs, nodes, part):
    """Partitions of more blocks than the table entries held in a register (64)."""
    print(f"[tree] {dt} {kv} d={d} bs={bs} {nodes} part={part}", flush=True)
    p = Problem([5003, 2100], nodes, 8, 1, d, bs, dt, kv, seed=21)
    check(p, *p.run(part_tokens=part))


@pytest.mark.parametrize("dt,kv,d", [(BF, None, 128), (F32, None, 64), (HF, F8, 64),
                                     (F32, None, 128)])
@pytest.mark.parametrize("fill", [float("nan"), 3e38])
def test_unowned_slots_do_not_reach(dt, kv, d, fill):
    """Slots behind a context in its last block and blocks of nobody hold NaN or
    values past the type's range."""
    p = Problem([33, 1, 0, 95], [5, 9, 2, 40], 8, 1, d, 16, dt, kv, seed=3, fill=fill)
    for part in (0, 64):
        check(p, *p.run(part_tokens=part))


@pytest.mark.parametrize("dt", [BF, HF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_hidden_nodes_do_not_reach(dt, bad):
    """A node whose K and V rows are not finite changes only the nodes that see it."""
    p = Problem([40, 7], [9, 50], 8, 2, 64, 16, dt, seed=4,
                parents=[np.array([-1, 0, 0, 1, 2, 2, 3, 4, 1], dtype=np.int32),
                         np.array([-1] + [0] * 49, dtype=np.int32)])
    clean = p.expect()
    hit = np.zeros(59, dtype=bool)
    for s, i in ((0, 2), (1, 33)):
        t = int(p.qsl[s]) + i
        p.k[t, :, 3] = bad
        p.v[t, 0, 5] = bad
        p.v[t, 1, 63] = -bad
        hit[p.qsl[s]:p.qsl[s + 1]] |= p.vis[s][:, i]
    out, lse = p.run()
    got = np64(out)
    assert np.isfinite(got[~hit]).all()
    # the others as if the rows were finite
    u = torch.finfo(dt).eps
    tol = 2 * u * (clean[2] + np.abs(clean[0])) + 2000 * E
    assert (np.abs(got - clean[0])[~hit] <= tol[~hit]).all()
    assert np.isnan(got[hit]).any()


@pytest.mark.parametrize("dt", [BF, F32])
def test_value_infinity_is_seen(dt):
    """With finite keys, an infinite value gives infinity to the nodes that see it."""
    p = Problem([40], [4], 8, 1, 64, 16, dt, seed=5,
                parents=[np.array([-1, 0, 0, 1], dtype=np.int32)])
    p.v[1, 0, 9] = float("inf")
    got = np64(p.run()[0])
    assert np.isposinf(got[[1, 3], :, 9]).all()
    assert np.isfinite(got[[0, 2]]).all()
    assert np.isfinite(np.delete(got, 9, axis=2)).all()


@pytest.mark.parametrize("dt,d", [(BF, 64), (F32, 64), (BF, 128)])
def test_arbitrary_masks_and_empty_rows(dt, d):
    """Any bits, also above a row's own node; a row that sees nothing; bits behind
    the run's end are no keys."""
    rng = np.random.default_rng(6)
    p = Problem([0, 50, 0], [5, 70, 3], 8, 1, d, 16, dt, seed=6)
    p.vis = [rng.random((n, n)) < 0.3 for n in p.nodes]
    p.vis[0][2] = False
    p.vis[2][:] = False
    meta = p.meta()
    m = tree_ref.pack_masks(p.vis, int(p.qsl[-1]), 2).view(np.uint64)
    for s, n in enumerate(p.nodes):  # garbage behind the run
        for w in range(2):
            keep = max(0, min(64, n - 64 * w))
            m[p.qsl[s]:p.qsl[s + 1], w] |= np.uint64(((1 << 64) - 1) & ~((1 << keep) - 1))
    meta.masks = torch.from_numpy(m.view(np.int64)).to(DEV)
    for part in (0, 64):
        out, lse = p.run(meta, part_tokens=part)
        check(p, out, lse)
        assert (out[2] == 0).all() and torch.isposinf(lse[2]).all()
        assert (out[-3:] == 0).all() and torch.isposinf(lse[-3:]).all()


@pytest.mark.parametrize("dt,d", [(BF, 64), (F32, 64), (BF, 128), (BF, 256)])
def test_nan_that_is_seen_stays(dt, d):
    """A query of NaN, and a context key of NaN: every row that they meet is NaN, whole or
    split (in whichever piece the key lies), the other rows as they were."""
    for at in (3, 120, 190):
        p = Problem([200, 60], [6, 4], 8, 1, d, 16, dt, seed=16)
        slot = p.tables[0][at // 16] * 16 + at % 16
        p.q[7, 2, 5] = float("nan")
        clean = [np64(x) for x in p.run()]
        p.kp.view(-1, 1, d)[slot, 0, 1] = float("nan")
        for part in (0, 64):
            out, lse = (np64(x) for x in p.run(part_tokens=part))
            assert np.isnan(out[:6]).all() and np.isnan(lse[:6]).all()
            assert np.isnan(out[7, 2]).all() and np.isnan(lse[7, 2])
            rest = np.ones((10, 8), dtype=bool)
            rest[:6] = False
            rest[7, 2] = False
            u = torch.finfo(dt).eps
            assert np.isfinite(out[rest]).all()
            assert (np.abs(out - clean[0])[rest] <= 2 * u * 4 + 1e-4).all()


def test_large_scores_and_scale():
    p = Problem([300], [12], 8, 1, 64, 16, BF, seed=7, amp=40.0)
    check(p, *p.run())
    p = Problem([300], [12], 8, 1, 64, 16, F32, seed=7, amp=3.0)
    check(p, *p.run(scale=0.7), scale=0.7)


def test_rows_of_no_sequence_and_bad_runs():
    """Rows behind the last sequence stay as they were; a run outside [0, T) or longer
    than the bound is skipped and flagged."""
    p = Problem([20, 30], [4, 6], 8, 1, 64, 16, BF, seed=8)
    meta = p.meta()
    pad = 5
    q, k, v = (torch.cat([x, torch.ones(pad, *x.shape[1:], dtype=x.dtype)]).to(DEV)
               for x in (p.q, p.k, p.v))
    full = TreeMeta(**{**meta.__dict__, "num_tokens": 10 + pad,
                       "masks": torch.cat([meta.masks, meta.masks[:pad]]).contiguous()})
    out = torch.full_like(q, 9.0)
    lse = torch.full(q.shape[:2], 9.0, device=DEV)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    paged_tree_attention(q, k, v, p.kp.to(DEV), p.vp.to(DEV), full, out=out, lse=lse, status=st)
    assert (out[10:] == 9).all() and (lse[10:] == 9).all() and int(st) == 0
    check(p, out[:10], lse[:10])
    for qsl, bound in (([0, 4, 99], 6), ([0, 4, 10], 5), ([-3, 4, 10], 7)):
        m = TreeMeta(**{**meta.__dict__, "max_nodes": bound,
                        "query_start_loc": torch.tensor(qsl, dtype=torch.int32, device=DEV)})
        out = torch.full((10, 8, 64), 9.0, dtype=BF, device=DEV)
        st.zero_()
        paged_tree_attention(p.q.to(DEV), p.k.to(DEV), p.v.to(DEV), p.kp.to(DEV), p.vp.to(DEV), m,
                             out=out, status=st)
        assert int(st) == _native.PKV_STATUS_BAD_QLOC, qsl
        skipped = slice(4, 10) if qsl[0] == 0 else slice(0, 4)
        assert (out[skipped] == 9).all()


def test_bad_blocks_read_as_zeros():
    p = Problem([40, 40], [3, 3], 8, 1, 64, 16, BF, seed=9)
    meta = p.meta()
    meta.block_tables[1, 1] = p.nb + 5
    meta.block_tables[1, 2] = -4
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    out, lse = p.run(meta, status=st)
    assert int(st) == _native.PKV_STATUS_BAD_BLOCK
    p.tables[1][1:] = [0, 0]  # blocks 1 and 2 of sequence 1 as zeros
    p.kp[0] = 0
    p.vp[0] = 0
    check(p, out, lse)


def test_context_bounds_are_only_hints():
    """A context past max_ctx_len, one past the table, and a negative one."""
    p = Problem([500, 64], [5, 5], 8, 1, 64, 16, BF, seed=10)
    for part in (0, 64):
        check(p, *p.run(p.meta(max_ctx=1), part_tokens=part))
    meta = p.meta()
    meta.ctx_lens = torch.tensor([9000, -3], dtype=torch.int32, device=DEV)
    q = Problem([512, 0], [5, 5], 8, 1, 64, 16, BF, seed=10)
    q.tables = [p.tables[0], []]
    q.q, q.k, q.v, q.kp, q.vp, q.vis = p.q, p.k, p.v, p.kp, p.vp, p.vis
    out, lse = p.run(meta)
    check(q, out, lse)


def test_layouts_alignment_and_out():
    """Strided and unaligned q / k / v, a strided out."""
    p = Problem([77, 12], [6, 3], 8, 2, 64, 16, BF, seed=11)
    base = p.run()[0]
    T = 9
    big = torch.zeros(T, 8 * 64 + 2 * 64 * 2 + 3, dtype=BF, device=DEV)
    q = big[:, 1:1 + 512].unflatten(1, (8, 64))
    k = big[:, 514:514 + 128].unflatten(1, (2, 64))
    v = big[:, 643:643 + 128].unflatten(1, (2, 64))
    q.copy_(p.q)
    k.copy_(p.k)
    v.copy_(p.v)
    out = torch.full((T, 8, 65), 5.0, dtype=BF, device=DEV)[:, :, 1:]
    got = paged_tree_attention(q, k, v, p.kp.to(DEV), p.vp.to(DEV), p.meta(), out=out)
    assert got is out and torch.equal(out, base)


def test_far_slots():
    """Slots whose byte offsets pass 2^32, at the end of a 4.3 GiB pool."""
    hkv, d, bs, nb = 8, 256, 16, (1 << 20) // 16 + 64
    p = Problem([100], [4], 8, hkv, d, bs, BF, seed=12)
    kp = torch.empty(nb, bs, hkv, d, dtype=BF, device=DEV)
    vp = torch.empty(nb, bs, hkv, d, dtype=BF, device=DEV)
    last = [nb - 1 - i for i in range(len(p.tables[0]))]
    kp[last] = p.kp[p.tables[0]].to(DEV)
    vp[last] = p.vp[p.tables[0]].to(DEV)
    meta = p.meta()
    meta.block_tables[0, :len(last)] = torch.tensor(last, dtype=torch.int32, device=DEV)
    lse = torch.empty(4, 8, device=DEV)
    out = paged_tree_attention(p.q.to(DEV), p.k.to(DEV), p.v.to(DEV), kp, vp, meta, lse=lse)
    check(p, out, lse)


def test_streams_and_graphs():
    """Two captured graphs and eager calls between their replays: every replay equals
    the eager result on the same inputs."""
    a = Problem([900, 30], [7, 4], 8, 1, 64, 16, BF, seed=13)
    b = Problem([400], [40], 8, 1, 128, 16, F32, seed=14)
    runs = []
    for p in (a, b):
        meta = p.meta()
        ts = [x.to(DEV) for x in (p.q, p.k, p.v, p.kp, p.vp)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            eager = paged_tree_attention(*ts, meta, part_tokens=64)
        torch.cuda.current_stream().wait_stream(side)
        out = torch.empty_like(eager)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            paged_tree_attention(*ts, meta, out=out, part_tokens=64)
        runs.append((p, meta, ts, out, graph))
    for it in range(3):
        for p, meta, ts, out, graph in runs:
            ts[0].copy_(ts[0].flip(0) * (0.5 + it))
            out.zero_()
        for p, meta, ts, out, graph in runs:
            graph.replay()
        eager = [paged_tree_attention(*ts, meta, part_tokens=64) for _, meta, ts, _, _ in runs]
        torch.cuda.synchronize()
        for (p, meta, ts, out, graph), e in zip(runs, eager):
            assert torch.equal(out, e)


def test_two_calls_at_once():
    p = Problem([2000, 100], [5, 9], 8, 1, 64, 16, BF, seed=15)
    meta = p.meta()
    ts = [x.to(DEV) for x in (p.q, p.k, p.v, p.kp, p.vp)]
    want = paged_tree_attention(*ts, meta, part_tokens=64)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(paged_tree_attention(*ts, meta, part_tokens=64))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
