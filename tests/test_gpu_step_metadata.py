"""Metadata that build_batch_meta makes on the device, handed on to what takes a
step's metadata: appends, attention, the model's step, the accepted rows' way into
the pool. num_tokens and max_q_len are bounds there, sequences may have no token, and
a step may fail or be dropped and taken again; and what the tree attention does with
metadata and tree rows that are not as they should be. Copied rows are compared byte by byte;
a token of one batch runs through the same kernels with the same partitions as the
host-packed batch it is compared with, except where a tolerance says otherwise."""
import numpy as np
import pytest
import torch

from oracle import paged_ref, tree_ref
from serving.kv_pool import KVPool
from serving.paged_meta import DeviceTables, build_batch_meta, pack_batch_meta

pytestmark = pytest.mark.gpu
DEV = "cuda"
F8, BF, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float32


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def bits(t):
    return t.view(torch.uint8) if t.dtype == F8 else t


class Batch:
    """Sequences of ctx tokens over shuffled blocks of bs, blocks behind them for q more."""

    def __init__(self, ctx, q, bs=16, seed=0):
        rng = np.random.default_rng(seed)
        self.ctx, self.q, self.bs = list(ctx), list(q), bs
        held = [-(-c // bs) for c in ctx]
        need = [max(0, -(-(c + n) // bs) - h) if n else 0 for c, n, h in zip(ctx, q, held)]
        self.nb = sum(held) + sum(need) + 3
        ids = rng.permutation(np.arange(1, self.nb)).tolist()
        self.rows, self.free = [], ids[sum(held):]
        self.after = []  # the rows with the blocks the step adds
        for h in held:
            self.rows.append(ids[:h])
            ids = ids[h:]
        spare = list(self.free)
        for row, n in zip(self.rows, need):
            self.after.append(row + spare[:n])
            spare = spare[n:]
        self.width = max([len(r) for r in self.after] + [1]) + 1

    def tables(self):
        return DeviceTables.from_host(self.rows, self.ctx, self.free, self.width, self.bs,
                                      self.nb, DEV)

    def meta(self, pad=0, bound=0, max_kv=0):
        return build_batch_meta(self.tables(), i32(self.q), sum(self.q) + pad,
                                bound or max(self.q), max_kv)[0]

    def host_meta(self):
        """pack_batch_meta of the sequences that have tokens."""
        some = [s for s, n in enumerate(self.q) if n]
        pos = [self.ctx[s] + i for s in some for i in range(self.q[s])]
        return pack_batch_meta([self.after[s] for s in some],
                               np.cumsum([0] + [self.q[s] for s in some]).tolist(), pos,
                               len(pos), torch.device(DEV), self.bs)

    def slots(self):
        return np.concatenate([np.asarray(paged_ref.make_slot_mapping(c, n, t, self.bs),
                                          dtype=np.int64)
                               for c, n, t in zip(self.ctx, self.q, self.after)])

    def pool(self, hkv, d, dtype, layers=1, seed=1):
        pool = KVPool(layers, self.bs, self.nb, hkv, d, dtype, DEV)
        g = torch.Generator().manual_seed(seed)
        pool.kv.copy_(torch.randn(pool.kv.shape, generator=g).to(dtype))
        return pool


# ---- rows behind the last token

PADDED = [([20, 3, 37], [4, 1, 0]), ([20, 3, 37], [0, 5, 2]), ([5], [3]), ([33, 16], [0, 0]),
          ([16, 31, 0, 8], [1, 0, 1, 0])]


@pytest.mark.parametrize("ctx,q", PADDED)
@pytest.mark.parametrize("dtype,kv,d", [(F32, F32, 8), (BF, BF, 64), (BF, BF, 5), (BF, F8, 64),
                                        (F32, F8, 8)])
def test_padding_is_not_appended(ctx, q, dtype, kv, d):
    """KVPool.write_from_table with more rows than tokens: the others' slots keep what
    they held, the last sequence's context among them."""
    print(f"[append] {ctx} {q} {dtype} {kv} d={d}", flush=True)
    b = Batch(ctx, q)
    for pad in (1, 40):
        T = sum(q) + pad
        pool, want = b.pool(2, d, kv, 2), b.pool(2, d, kv, 2)
        g = torch.Generator().manual_seed(2)
        k, v = (torch.randn(T, 2, d, generator=g).to(dtype).to(DEV) for _ in range(2))
        pool.write_from_table(1, k, v, b.meta(pad, 8))
        real = torch.from_numpy(b.slots()).to(DEV)
        for flat, rows in ((want.flat_k[1], k), (want.flat_v[1], v)):
            bits(flat)[real] = bits(rows[:sum(q)].to(kv))
        assert torch.equal(bits(pool.kv), bits(want.kv))


def test_padding_is_not_appended_many_sequences():
    """More sequences than query_start_loc entries fit the append's LDS."""
    n = 4200
    rng = np.random.default_rng(3)
    b = Batch(rng.integers(0, 5, size=n).tolist(), (rng.integers(0, 3, size=n - 1)).tolist() + [0],
              bs=4)
    pool, want = b.pool(1, 8, F32), b.pool(1, 8, F32)
    k = torch.randn(sum(b.q) + 50, 1, 8, device=DEV)
    pool.write_from_table(0, k, -k, b.meta(50))
    real = torch.from_numpy(b.slots()).to(DEV)
    want.flat_k[0][real], want.flat_v[0][real] = k[:sum(b.q)], -k[:sum(b.q)]
    assert torch.equal(pool.kv, want.kv)


@pytest.mark.parametrize("dtype,kv,hq,hkv,d", [(F32, F32, 8, 1, 64), (F32, F32, 4, 4, 80),
                                               (BF, BF, 8, 1, 64), (BF, BF, 16, 1, 64),
                                               (BF, BF, 32, 1, 128), (BF, F8, 16, 1, 64)])
@pytest.mark.parametrize("ctx,q", [([20, 300, 37], [1, 0, 1]), ([20, 300, 37], [1, 1, 0]),
                                   ([20, 70, 37], [0, 1, 7]), ([20, 5, 37], [40, 1, 0]),
                                   ([5000, 17, 90], [1, 1, 0]), ([5000, 17, 90], [1, 9, 0])])
def test_padded_steps_append_and_attend(ctx, q, dtype, kv, hq, hkv, d):
    """paged_attention_append_meta (fused or not) of a padded step: pool and rows as the
    host-packed batch of the sequences with tokens gives them, rows behind untouched."""
    from serving.fake_paged_attn import paged_attention_append_meta
    print(f"[fused] {ctx} {q} {dtype} {kv} {hq}x{hkv}x{d}", flush=True)
    b = Batch(ctx, q)
    T, pad = sum(q), 4
    g = torch.Generator().manual_seed(4)
    rows = [torch.randn(T + pad, h, d, generator=g).to(dtype).to(DEV) for h in (hq, hkv, hkv)]
    want = b.pool(hkv, d, kv)
    ref = paged_attention_append_meta(*[x[:T].contiguous() for x in rows], want, 0, b.host_meta())
    # other partitions of the contexts: sums of at most 5001 weights in another order, and
    # 16-bit probabilities against another maximum; values of at most 6
    u = torch.finfo(dtype).eps / 2
    tol = 6 * (2 * 5001 * 2.0 ** -24 + (2 * u if dtype != F32 else 0)) + 2 * u
    for bound in (max(q), 9 + max(q)):  # looser, the prompt kernels' too
        got = b.pool(hkv, d, kv)
        out = torch.full_like(rows[0], 9.0)
        paged_attention_append_meta(*rows, got, 0, b.meta(pad, bound), out=out)
        assert torch.equal(bits(got.kv), bits(want.kv))
        assert float((out[:T].float() - ref.float()).abs().max()) <= tol
        assert (out[T:] == 9).all()


# ---- sequences without a token in the model's step

def small_model(dtype=F32):
    from serving.layers import ModelConfig
    from serving.paged_model import PagedTransformer
    cfg = ModelConfig(vocab_size=97, d_model=128, num_layers=2, num_heads=4, num_kv_heads=1,
                      max_seq_len=160)
    torch.manual_seed(0)
    return cfg, PagedTransformer(cfg).to(DEV, dtype).eval()


def test_bounds_are_no_decode_batch():
    b = Batch([20, 5], [1, 1])
    assert b.host_meta().is_decode
    assert not b.meta().is_decode  # one token a sequence at most, as far as the host knows


@pytest.mark.parametrize("ctx,q,pad", [([20, 3, 37], [1, 0, 1], 1), ([20, 3, 37], [1, 1, 0], 1),
                                       ([20, 3, 37], [0, 1, 1], 1), ([20, 3, 37], [0, 3, 0], 0),
                                       ([20, 3, 37], [5, 0, 2], 9), ([20, 3], [0, 0], 2),
                                       ([20, 3], [0, 0], 0), ([20, 3, 37], [1, 1, 1], 0)])
def test_forward_step_with_empty_sequences(ctx, q, pad):
    """Logits row s is sequence s's: its last token's, zeros where it has none. The pass
    is the host-packed batch's of the other sequences, its projections over another
    number of rows: sums of at most 128 terms in another order, 9 of them (see
    test_gpu_speculative.py)."""
    print(f"[step] {ctx} {q} pad={pad}", flush=True)
    cfg, model = small_model()
    b = Batch(ctx, q)
    T = sum(q)
    got, want = (b.pool(1, cfg.head_dim, F32, cfg.num_layers) for _ in range(2))
    ids = torch.arange(T + pad, device=DEV) % 97
    logits = model.forward_step(ids, got, b.meta(pad, max(max(q), 1)))
    assert logits.shape == (len(q), 97)
    some = [s for s, n in enumerate(q) if n]
    if some:
        ref = model.forward_step(ids[:T], want, b.host_meta())
        scale = float(ref.abs().max())
        assert float((logits[some] - ref).abs().max()) <= 1e-4 * scale
        assert float((got.kv - want.kv).abs().max()) <= 1e-4 * float(want.kv.abs().max())
    else:
        assert torch.equal(got.kv, want.kv)
    none = [s for s, n in enumerate(q) if not n]
    assert (logits[none] == 0).all()


def test_decode_graph_refuses_bounds():
    from serving.graph_step import DecodeStepGraph
    cfg, model = small_model()
    b = Batch([20, 3], [1, 0])
    pool = b.pool(1, cfg.head_dim, F32, cfg.num_layers)
    ids = torch.zeros(2, dtype=torch.long, device=DEV)
    with pytest.raises(ValueError, match="decode batch"):
        DecodeStepGraph(model, pool, b.meta(1), ids)


# ---- advance_

@pytest.mark.parametrize("ctx,q,pad", [([20, 3, 31], [1, 0, 1], 2), ([16, 15], [1, 1], 0),
                                       ([4, 9], [0, 3], 1)])
def test_advance_leaves_padding_and_slots_of_nobody(ctx, q, pad):
    b = Batch(ctx, q)
    meta, T = b.meta(pad), sum(q)
    was = {n: getattr(meta, n).tolist() for n in ("seq_lens", "start_pos", "positions")}
    for step in (1, 2):
        meta.advance_()
        assert meta.seq_lens.tolist() == [x + step if n else 0 for x, n in zip(was["seq_lens"], q)]
        assert meta.start_pos.tolist() == [x + step if n else 0
                                           for x, n in zip(was["start_pos"], q)]
        assert meta.positions.tolist() == [x + step for x in was["positions"][:T]] + [0] * pad
    # the next tokens' slots are another step's to give: an append skips these
    assert meta.slot_mapping.tolist() == [tree_ref.NO_SLOT] * (T + pad)
    pool, want = b.pool(1, 8, F32), b.pool(1, 8, F32)
    k = torch.ones(T + pad, 1, 8, device=DEV)
    pool.write(0, meta.slot_mapping, k, k)
    assert torch.equal(pool.kv, want.kv)


def test_advance_in_a_graph():
    b = Batch([20, 3, 31], [1, 0, 1])
    meta, twin = b.meta(2), b.meta(2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        meta.advance_()
        twin.advance_()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        meta.advance_()
    for it in range(4):
        graph.replay()
        twin.advance_()
        torch.cuda.synchronize()
        for name in ("seq_lens", "start_pos", "positions", "slot_mapping"):
            assert torch.equal(getattr(meta, name), getattr(twin, name)), (it, name)


# ---- a step that fails is no step for anybody

FAILS = {  # sequence 0 lacks a block, sequence 1 has one to spare
    "blocks": dict(free=[]),
    "cursor": dict(cursor=7),
    "short": dict(q=[40, 3]),
    "far": dict(ctx=[16, 2147483000]),
    "long": dict(q=[3, 9]),          # past max_q_len
    "negative": dict(q=[3, -1]),
    "tokens": dict(T=5),             # more tokens than rows
    "held": dict(held=[1, -1]),
}


@pytest.mark.parametrize("what", FAILS)
@pytest.mark.parametrize("stale", [0, 5])
def test_failed_steps_write_nothing(what, stale):
    """Every way of a step's rows into the pool: accepted rows, the append through the
    table, the append through slots, attention's own append. Row 0 of the table may
    name a block behind those it holds that is another sequence's by now."""
    from serving.fake_paged_attn import paged_attention_append_meta
    from serving.tree_decode import TreeAccept, build_tree_meta
    print(f"[failed] {what} stale={stale}", flush=True)
    a = dict(ctx=[16, 10], q=[3, 3], held=[1, 1], free=[6, 7], cursor=0, T=12)
    a.update(FAILS[what])
    dt = DeviceTables(block_tables=i32([1, stale, stale, 2, 0, 0]).view(2, 3),
                      blocks_held=i32(a["held"]), ctx_lens=i32(a["ctx"]),
                      free_blocks=i32(a["free"]), free_cursor=i32([a["cursor"]]), block_size=16,
                      num_blocks=9)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    tree = build_tree_meta(dt, i32([-1, 0, 1] * 2), i32([0, 3, 6]), 3)
    meta, after = build_batch_meta(dt, i32(a["q"]), a["T"], 8 if what != "short" else 50,
                                   status=st)
    assert int(st) != 0
    assert after.blocks_held.tolist() == a["held"] and after.ctx_lens.tolist() == a["ctx"]
    for dtype, kv, hq in ((F32, F32, 8), (BF, BF, 16), (BF, F8, 16)):
        b = Batch([16, 10], [3, 3])
        b.nb = 9
        pool, want = b.pool(1, 64, kv, 2), b.pool(1, 64, kv, 2)
        rows = torch.ones(2, 6, 1, 64, dtype=dtype, device=DEV)
        acc = TreeAccept(lens=i32([3, 3]), path=i32([0, 1, 2] * 2).view(2, 3), tokens=None)
        pool.write_accepted(rows, rows, tree, acc, meta)
        assert torch.equal(bits(pool.kv), bits(want.kv)), "write_accepted"
        k = torch.ones(a["T"], 1, 64, dtype=dtype, device=DEV)
        pool.write_from_table(1, k, k, meta)
        assert torch.equal(bits(pool.kv), bits(want.kv)), "write_from_table"
        pool.write(0, meta.slot_mapping, k, k)
        assert torch.equal(bits(pool.kv), bits(want.kv)), "write"
        q = torch.ones(a["T"], hq, 64, dtype=dtype, device=DEV)
        paged_attention_append_meta(q, k, k, pool, 0, meta)
        assert torch.equal(bits(pool.kv), bits(want.kv)), "paged_attention_append_meta"


def test_a_failed_step_after_a_dropped_one():
    """A dropped step's block goes to another sequence, and a step that then fails
    leaves that sequence's rows alone."""
    from serving.tree_decode import TreeAccept, build_tree_meta
    dt = DeviceTables.from_host([[1], [2]], [16, 16], [5, 6], 3, 16, 9, DEV)
    build_batch_meta(dt, i32([1, 0]), 2, 1)                      # block 5 to row 0: dropped
    _, dt = build_batch_meta(dt, i32([0, 1]), 2, 1)              # sequence 1's by now
    pool = KVPool(1, 16, 9, 1, 8, F32, DEV)
    pool.kv.normal_()
    before = pool.kv.clone()
    tree = build_tree_meta(dt, i32([-1, -1]), i32([0, 1, 2]), 1)
    meta, _ = build_batch_meta(dt, i32([1, 17]), 18, 17)         # two blocks of the one left
    rows = torch.ones(1, 2, 1, 8, device=DEV)
    pool.write_accepted(rows, rows, tree, TreeAccept(i32([1, 1]), i32([0, 0]).view(2, 1), None),
                        meta)
    assert torch.equal(pool.kv, before)


def test_rows_hold_their_blocks_and_zeros_behind_them():
    """After a step the table names no block that a dropped step had put there, whether
    the step succeeds or fails; the same sequence may take the same block again."""
    dt = DeviceTables.from_host([[1], [2], [3]], [16, 16, 9], [5, 6, 7, 8], 4, 16, 9, DEV)
    build_batch_meta(dt, i32([33, 0, 7]), 64, 40)
    assert dt.block_tables.tolist() == [[1, 5, 6, 7], [2, 0, 0, 0], [3, 0, 0, 0]]
    build_batch_meta(dt, i32([0, 0, 60]), 64, 60)               # fails: row 2 is too short
    assert dt.block_tables.tolist() == [[1, 0, 0, 0], [2, 0, 0, 0], [3, 0, 0, 0]]
    build_batch_meta(dt, i32([33, 0, 7]), 64, 40)
    _, after = build_batch_meta(dt, i32([1, 20, 0]), 64, 40)
    assert after.block_tables.tolist() == [[1, 5, 0, 0], [2, 6, 7, 0], [3, 0, 0, 0]]
    _, last = build_batch_meta(after, i32([0, 0, 0]), 64, 40)   # nothing to add
    assert last.block_tables.tolist() == [[1, 5, 0, 0], [2, 6, 7, 0], [3, 0, 0, 0]]


def test_stale_entries_of_many_sequences():
    n = 700
    dt = DeviceTables.from_host([[1 + s] for s in range(n)], [16] * n, range(n + 1, 4 * n + 1), 5,
                                16, 4 * n + 1, DEV)
    build_batch_meta(dt, i32([33] * n), 33 * n, 33)
    rng = np.random.default_rng(5)
    q = rng.integers(0, 34, size=n).tolist()
    _, after = build_batch_meta(dt, i32(q), 33 * n, 33)
    host = [[1 + s, 0, 0, 0, 0] for s in range(n)]
    tree_ref.build_step(host, [1] * n, [16] * n, q, list(range(n + 1, 4 * n + 1)), 0, 16, 4 * n + 1,
                        33 * n, 33)
    assert after.block_tables.tolist() == host


@pytest.mark.parametrize("kv", [F32, F8])
@pytest.mark.parametrize("packed", [False, True])
def test_write_accepted_writes_the_steps_tokens_only(kv, packed):
    """Paths longer than the tokens the step has for a sequence (a finished one's 0, a
    goal's rest): the rows behind them are not written, neither into the context's
    first positions nor past the sequence's blocks."""
    from serving.tree_decode import TreeAccept, build_tree_meta
    b = Batch([20, 14, 3, 40], [0, 2, 4, 0])
    dt = b.tables()
    tree = build_tree_meta(dt, i32([-1, 0, 1, 2] * 4), i32([0, 4, 8, 12, 16]), 4)
    if packed:
        meta = pack_batch_meta(b.after, [0, 0, 2, 6, 6], [14, 15, 3, 4, 5, 6], 6,
                               torch.device(DEV), 16)
    else:
        meta, _ = build_batch_meta(dt, i32(b.q), 16, 4)
    acc = TreeAccept(i32([4, 4, 4, 3]), i32([0, 1, 2, 3] * 3 + [0, 1, 2, -1]).view(4, 4), None)
    pool, want = b.pool(2, 8, kv, 3), b.pool(2, 8, kv, 3)
    k, v = torch.randn(2, 3, 16, 2, 8, device=DEV).unbind(0)
    pool.write_accepted(k, v, tree, acc, meta)
    slots = torch.from_numpy(b.slots()).to(DEV)
    for layer in range(3):
        for flat, rows in ((want.flat_k[layer], k), (want.flat_v[layer], v)):
            bits(flat)[slots] = bits(rows[layer, [4, 5, 8, 9, 10, 11]].to(kv))
    assert torch.equal(bits(pool.kv), bits(want.kv))


# ---- metadata that is not what the kernels read

def tree_call(kv=F32, layers=1):
    from serving.tree_decode import build_tree_meta
    b = Batch([20, 5], [0, 0])
    tree = build_tree_meta(b.tables(), i32([-1, 0, -1]), i32([0, 2, 3]), 2)
    return b, tree, torch.ones(3, 8, 64, device=DEV), torch.ones(3, 1, 64, device=DEV), \
        b.pool(1, 64, kv, layers)


@pytest.mark.parametrize("name", ["block_tables", "ctx_lens", "query_start_loc"])
def test_tree_attention_refuses_other_tensors(name):
    """Tables and lengths of another type or device, or with gaps, before anything is
    launched."""
    from dataclasses import replace
    from serving.tree_decode import paged_tree_attention
    b, tree, q, k, pool = tree_call()
    good = getattr(tree, name)
    gaps = torch.stack([good, good], -1)[..., 0]
    assert not gaps.is_contiguous()
    for bad in (good.long(), good.float(), good.cpu(), gaps):
        with pytest.raises((ValueError, RuntimeError), match=f"{name}|device"):
            paged_tree_attention(q, k, k, *pool.kv[0], replace(tree, **{name: bad}))
    paged_tree_attention(q, k, k, *pool.kv[0], tree)


def test_tree_attention_refuses_a_smaller_pool():
    """Tables that may name blocks which the pool does not have."""
    from serving.tree_decode import paged_tree_attention
    b, tree, q, k, pool = tree_call()
    with pytest.raises(ValueError, match="blocks"):
        paged_tree_attention(q, k, k, *pool.kv[0, :, :b.nb - 1], tree)
    big = torch.cat([pool.kv[0], pool.kv[0]], 1)
    assert torch.equal(paged_tree_attention(q, k, k, *big, tree),
                       paged_tree_attention(q, k, k, *pool.kv[0], tree))


def test_tree_context_bounds_of_any_size():
    """A bound past what an int holds bounds nothing."""
    from serving.tree_decode import build_tree_meta, paged_tree_attention
    b, tree, q, k, pool = tree_call()
    want = paged_tree_attention(q, k, k, *pool.kv[0], tree)
    for bound in (1 << 31, 1 << 40, 1 << 70):
        big = build_tree_meta(b.tables(), i32([-1, 0, -1]), i32([0, 2, 3]), 2, bound)
        assert torch.equal(paged_tree_attention(q, k, k, *pool.kv[0], big), want)


# ---- what a step's status tells

def test_forward_tree_reports_bad_blocks_and_runs():
    from serving import _native
    from serving.tree_decode import build_tree_meta
    cfg, model = small_model()
    b = Batch([20, 5], [0, 0])
    pool = b.pool(1, cfg.head_dim, F32, cfg.num_layers)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    ids = torch.arange(3, device=DEV)
    parents = i32([-1, 0, -1])

    def run(dt, qsl, bound=2):
        st.zero_()
        tree = build_tree_meta(dt, parents, qsl, bound)  # reports to nobody
        model.forward_tree(ids, pool, tree, status=st)
        return int(st)

    dt = b.tables()
    assert run(dt, i32([0, 2, 3])) == 0
    assert run(dt, i32([0, 2, 3]), 1) == _native.PKV_STATUS_BAD_QLOC
    dt.block_tables[0, 1] = b.nb
    assert run(dt, i32([0, 2, 3])) == _native.PKV_STATUS_BAD_BLOCK


def test_generate_speculative_reports_bad_blocks():
    """A block id past the pool that only the model's pass meets: the prompt's."""
    from serving.allocator import BlockAllocator
    from serving.generation import generate_speculative
    cfg, model = small_model()
    alloc = BlockAllocator(40)
    pool = KVPool(cfg.num_layers, 16, 8, 1, cfg.head_dim, F32, DEV)
    low = alloc.allocate_n(7)
    high = alloc.allocate_n(1)  # block 8: the pool has 0 ... 7
    assert high == [8] and low == list(range(1, 8))

    class Ids:  # hands out the bad block first
        ids = high + low

        def allocate(self):
            return self.ids.pop(0)

        def allocate_n(self, n):
            return [self.allocate() for _ in range(n)]

        def free(self, blocks):
            pass

    with pytest.raises(AssertionError, match="block id"):
        generate_speculative(model, [[1, 2, 3]], 5, pool, Ids(), lambda h: ([], []))


# ---- a pool of more layers than the model

def test_generate_speculative_in_a_larger_pool():
    from serving.allocator import BlockAllocator
    from serving.generation import generate_batched, generate_speculative
    cfg, model = small_model()
    prompts = [[5, 6, 7], [9] * 20]
    pool, alloc = KVPool(cfg.num_layers + 2, 16, 20, 1, cfg.head_dim, F32, DEV), BlockAllocator(20)
    pool.kv[cfg.num_layers:].fill_(3.0)
    truth = generate_batched(model, prompts, 20, pool, alloc)
    draft = lambda h: ([(h[-1] + 1) % 97, h[0]], [-1, 0])  # noqa: E731
    assert generate_speculative(model, prompts, 20, pool, alloc, draft) == truth
    assert (pool.kv[cfg.num_layers:] == 3.0).all()


def test_write_accepted_refuses_more_layers_than_the_pool_has():
    from serving.tree_decode import tree_accept
    b, tree, _, _, pool = tree_call(layers=2)
    ids = torch.zeros(3, dtype=torch.long, device=DEV)
    acc = tree_accept(ids, ids, tree, 2)
    meta, _ = build_batch_meta(b.tables(), torch.zeros_like(acc.lens), 4, 2)
    for layers in (1, 2):
        rows = torch.ones(layers, 3, 1, 64, device=DEV)
        pool.write_accepted(rows, rows, tree, acc, meta)
    rows = torch.ones(3, 3, 1, 64, device=DEV)
    with pytest.raises(AssertionError):
        pool.write_accepted(rows, rows, tree, acc, meta)


# ---- values that are not finite, in the trees' rows

@pytest.mark.parametrize("dtype,kv,d,hkv", [(F32, F32, 64, 1), (BF, BF, 64, 2), (BF, BF, 128, 1),
                                            (BF, F8, 64, 1), (torch.float16, torch.float16, 64, 2),
                                            (BF, BF, 256, 1), (F32, F32, 8, 1)])
@pytest.mark.parametrize("part", [0, 64])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), 470.0])
def test_values_that_are_not_finite_reach_all_that_see_them(dtype, kv, d, hkv, part, bad):
    """A tree value of NaN or infinity (with an fp8 pool also one past 464, which rounds to
    NaN) makes that column of every row and head that sees its node not finite, and
    changes nothing else; a key of NaN makes whole rows NaN. Contexts of several
    partitions, and none."""
    from serving.tree_decode import build_tree_meta, paged_tree_attention
    print(f"[odd] {dtype} {kv} d={d} hkv={hkv} part={part} {bad}", flush=True)
    if bad == 470.0 and kv != F8:  # finite in the operand's type
        bad = -float("inf")
    hq = 8
    b = Batch([300, 0, 7], [0, 0, 0])
    parents = [[-1, 0, 0, 1, 2, 2, 3, 4, 1], [-1, 0, 1, 1], [-1] + [0] * 69]
    nodes = [len(p) for p in parents]
    qsl = np.concatenate([[0], np.cumsum(nodes)])
    T = int(qsl[-1])
    g = torch.Generator().manual_seed(7)
    q, k, v = (torch.randn(T, h, d, generator=g).to(dtype).to(DEV) for h in (hq, hkv, hkv))
    pool = b.pool(hkv, d, kv)
    tree = build_tree_meta(b.tables(), i32(np.concatenate(parents)), i32(qsl), max(nodes), 300)
    vis = [tree_ref.visible_from_parents(p)[0] for p in parents]
    run = lambda: paged_tree_attention(q, k, v, *pool.kv[0], tree, part_tokens=part)  # noqa: E731
    clean = run().float().cpu()
    assert torch.isfinite(clean).all()
    sees = np.zeros((T, 3), dtype=bool)  # the node with the bad value, of each sequence
    for s, node in enumerate((2, 1, 33)):
        sees[qsl[s]:qsl[s + 1], s] = vis[s][:, node]
        v[int(qsl[s]) + node, 0, 5] = bad
    got = run().float().cpu()
    hit = torch.from_numpy(sees.any(1))
    heads = torch.arange(hq) < hq // hkv  # those of kv head 0
    want = torch.zeros(T, hq, d, dtype=torch.bool)
    want[:, :, 5] = hit[:, None] & heads
    assert torch.equal(~torch.isfinite(got), want)
    assert torch.equal(got[~want], clean[~want])
    if kv != F8 and abs(bad) == float("inf"):
        assert (got[want] == bad).all()
    for s, node in enumerate((2, 1, 33)):  # and a key
        k[int(qsl[s]) + node, 0, 3] = float("nan")
    got = run().float().cpu()
    rows = hit[:, None] & heads
    assert torch.isnan(got[rows]).all() and torch.isfinite(got[~rows]).all()
    # A row's weights are 2^(s - m), and m moves for the 32 rows of a wavefront together,
    # at the largest of their new scores that passes it by the lazy step: a row of NaN never
    # does, so the others may keep an earlier m, and each of their roundings falls
    # elsewhere. Two results whose every weight (16-bit operands: u, fp16 steps of 2^-24)
    # and sum are rounded anew differ by twice what one may be off by (the bounds are those
    # of test_gpu_tree_attention.py): 2 (u A + 2 (d + 8) e S A + 2 (L + 16) e A +
    # 2^-25 V1 + u |out|), A the weighted mean of |v|, S at most the scale times the
    # largest norms of q and k, L at most 370 keys.
    e, u = 2.0 ** -24, torch.finfo(dtype).eps / 2
    k, v = torch.nan_to_num(k, nan=0.0), v.nan_to_num(0.0, 0.0, 0.0).abs()
    v[v > 464] = 0
    pool.flat_v[0].copy_(pool.flat_v[0].float().abs().to(kv))
    A = run().float().cpu()[~rows] * (1 + 2 * u + 1e-3)
    S = d ** -0.5 * float(q.float().norm(dim=-1).max()) * max(
        float(x.float().norm(dim=-1).max()) for x in (k, pool.flat_k[0]))
    V1 = 370 * max(float(x.float().max()) for x in (v, pool.flat_v[0]))
    tol = (2 * (d + 8) * e * S + 2 * (370 + 16) * e) * A + u * clean[~rows].abs() * (1 + 2.0 ** -6)
    if dtype != F32:
        tol += u * A + (2.0 ** -25 * V1 if dtype == torch.float16 else 0)
    assert ((got - clean)[~rows].abs() <= 2 * tol).all()


# ---- the ends of a step's sizes

def test_a_step_without_nodes():
    """Every sequence finished: nothing to verify, nothing changes."""
    from serving.tree_decode import build_tree_meta, tree_accept
    cfg, model = small_model()
    b = Batch([20, 5], [0, 0])
    pool = b.pool(1, cfg.head_dim, F32, cfg.num_layers)
    before, dt = pool.kv.clone(), b.tables()
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    ids = torch.zeros(0, dtype=torch.long, device=DEV)
    tree = build_tree_meta(dt, i32([]), i32([0, 0, 0]), 4, status=st)
    logits, k, v = model.forward_tree(ids, pool, tree, st)
    assert logits.shape == (0, 97) and k.shape == v.shape == (cfg.num_layers, 0, 1, cfg.head_dim)
    acc = tree_accept(ids, ids, tree, 3, status=st)
    assert acc.lens.tolist() == [0, 0] and (acc.path == -1).all()
    meta, after = build_batch_meta(dt, acc.lens, 0, 3, status=st)
    pool.write_accepted(k, v, tree, acc, meta)
    assert int(st) == 0 and torch.equal(pool.kv, before)
    assert after.ctx_lens.tolist() == [20, 5] and after.free_cursor.tolist() == [0]


def test_generate_speculative_without_a_limit_on_depth():
    """max_depth past what a step could keep costs nothing."""
    from serving.allocator import BlockAllocator
    from serving.generation import generate_batched, generate_speculative
    cfg, model = small_model()
    pool, alloc = KVPool(cfg.num_layers, 16, 20, 1, cfg.head_dim, F32, DEV), BlockAllocator(20)
    prompts = [[5, 6, 7], [9] * 20]
    truth = generate_batched(model, prompts, 12, pool, alloc)
    right = lambda h: (next(p + t for p, t in zip(prompts, truth)  # noqa: E731
                            if (p + t)[:len(h)] == h)[len(h):], list(range(-1, 11)))
    draft = lambda h: (right(h)[0], right(h)[1][:len(right(h)[0])])  # noqa: E731
    for depth in (8, 1 << 31, 1 << 62):
        assert generate_speculative(model, prompts, 12, pool, alloc, draft, max_depth=depth) == truth
    assert alloc.num_free == 19


# ---- captured

def test_padded_step_in_a_graph():
    """build_batch_meta and forward_step captured once and replayed over other lengths, a
    sequence without a token, a step that fails and one that is taken after it: the
    eager step's results, and nothing of the failed step in the pool."""
    from serving import _native
    cfg, model = small_model()
    b = Batch([20, 3, 31], [9, 9, 9])
    dt = b.tables()
    pool, q = b.pool(1, cfg.head_dim, F32, cfg.num_layers), i32([2, 0, 1])
    kv0, table0 = pool.kv.clone(), dt.block_tables.clone()
    ids = torch.arange(12, device=DEV) * 7 % 97
    st = torch.zeros(1, dtype=torch.int32, device=DEV)

    def step():
        pool.kv.copy_(kv0)
        dt.block_tables.copy_(table0)
        st.zero_()
        meta, after = build_batch_meta(dt, q, 12, 9, status=st)
        logits = model.forward_step(ids, pool, meta)
        return [logits, pool.kv, after.block_tables, after.blocks_held, after.ctx_lens,
                after.free_cursor, meta.slot_mapping, st]

    ws = _native.Workspace()
    with _native.workspace_scope(ws):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = step()
    for lens, fails in (([2, 0, 1], 0), ([0, 9, 3], 0), ([9, 9, 0], 1), ([1, 1, 1], 0),
                        ([0, 0, 0], 0), ([3, 10, 0], 1), ([4, 4, 4], 0)):
        q.copy_(i32(lens))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for a, c in zip(got[1:], want[1:]):
            assert torch.equal(a, c), lens
        assert bool(int(got[-1])) == bool(fails), lens
        if fails:
            assert torch.equal(got[1], kv0) and torch.equal(got[2], table0)
        else:
            assert torch.equal(got[0], want[0]), lens
            assert (got[0][[i for i, n in enumerate(lens) if n == 0]] == 0).all()


def test_failed_tree_step_in_a_graph():
    """The verification step captured, with too few blocks at some replays."""
    from serving.tree_decode import TreeAccept, build_tree_meta
    b = Batch([16, 10], [3, 3])
    pool, dt = b.pool(2, 64, BF, 2), b.tables()
    kv0, table0, cursor = pool.kv.clone(), dt.block_tables.clone(), dt.free_cursor
    lens, rows = i32([2, 3]), torch.randn(2, 6, 2, 64, device=DEV).to(BF)
    st = torch.zeros(1, dtype=torch.int32, device=DEV)
    parents, qsl, path = i32([-1, 0, 1] * 2), i32([0, 3, 6]), i32([0, 1, 2] * 2).view(2, 3)

    def step():
        pool.kv.copy_(kv0)
        dt.block_tables.copy_(table0)
        st.zero_()
        tree = build_tree_meta(dt, parents, qsl, 3, status=st)
        meta, after = build_batch_meta(dt, lens, 6, 3, status=st)
        pool.write_accepted(rows, -rows, tree, TreeAccept(lens, path, None), meta)
        return [pool.kv, after.block_tables, after.blocks_held, after.ctx_lens, st]

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for it, at in enumerate((0, len(b.free), 0, len(b.free) + 1, 0)):
        cursor.fill_(at)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = [t.clone() for t in step()]
        assert all(torch.equal(a, c) for a, c in zip(got, want)), it
        assert bool(int(got[-1])) == (at > 0)
        assert torch.equal(got[0], kv0) == (at > 0)


@pytest.mark.parametrize("dtype,kv,hq,hkv,d", [(F32, F32, 8, 1, 64), (BF, BF, 8, 1, 64),
                                               (BF, BF, 16, 1, 64), (BF, BF, 32, 1, 128),
                                               (BF, F8, 16, 1, 64), (F32, F32, 4, 4, 80)])
@pytest.mark.parametrize("q", [[1, 1], [1, 9]])
@pytest.mark.parametrize("width", [3, 300])
def test_failed_decode_and_mixed_steps_write_nothing(dtype, kv, hq, hkv, d, q, width):
    """Each form of the attention's own append (fused with decode partitions, the prompt
    kernel or both in one launch, or a launch before the persistent kernel)."""
    from serving.fake_paged_attn import paged_attention_append_meta
    print(f"[failed] {dtype} {kv} {hq}x{hkv}x{d} q={q} width={width}", flush=True)
    b = Batch([16, 10], q)
    b.width = width
    pool, want = b.pool(hkv, d, kv), b.pool(hkv, d, kv)
    dt = b.tables()
    dt.free_cursor.fill_(len(b.free))
    meta, _ = build_batch_meta(dt, i32(q), sum(q), max(q))
    g = torch.Generator().manual_seed(8)
    rows = [torch.randn(sum(q), h, d, generator=g).to(dtype).to(DEV) for h in (hq, hkv, hkv)]
    out = paged_attention_append_meta(*rows, pool, 0, meta)
    assert torch.equal(bits(pool.kv), bits(want.kv))
    assert (out == 0).all()  # it attends to nothing either


def test_lengths_that_the_caller_knows():
    """One token for every sequence, said to be so: a decode batch, captured and advanced
    (within the blocks that the rows hold) as the host-packed one."""
    from dataclasses import replace
    from serving.graph_step import DecodeStepGraph
    cfg, model = small_model()
    b = Batch([20, 3, 34], [1, 1, 1])
    ids = torch.tensor([3, 14, 15], device=DEV)
    meta, host = replace(b.meta(), exact=True), b.host_meta()
    assert meta.is_decode
    pools = [b.pool(1, cfg.head_dim, F32, cfg.num_layers) for _ in range(2)]
    graphs = [DecodeStepGraph(model, p, m, ids) for p, m in zip(pools, (meta, host))]
    assert meta.slot_mapping.tolist() == [tree_ref.NO_SLOT] * 3
    for it in range(4):
        got, want = (g.replay().tolist() for g in graphs)
        assert got == want, it
    assert meta.seq_lens.tolist() == host.seq_lens.tolist()
    assert float((pools[0].kv - pools[1].kv).abs().max()) <= 1e-4 * float(pools[1].kv.abs().max())
