"""The step around the tree attention on the device: build_batch_meta,
build_tree_meta, tree_accept and KVPool.write_accepted, each against its plain
definition on Python lists (oracle/tree_ref.py). Whole numbers and copied bytes:
compared exactly."""
import numpy as np
import pytest
import torch

from oracle import paged_ref, tree_ref
from serving import _native
from serving.allocator import BlockAllocator
from serving.kv_pool import KVPool
from serving.paged_meta import (DeviceTables, build_batch_meta, pack_batch_meta,
                                raise_step_status)
from serving.tree_decode import TreeAccept, build_tree_meta, tree_accept

pytestmark = pytest.mark.gpu
DEV = "cuda"
BITS = {"qloc": _native.PKV_STATUS_BAD_QLOC, "short": _native.PKV_STATUS_SHORT_TABLE,
        "blocks": _native.PKV_STATUS_OUT_OF_BLOCKS, "block": _native.PKV_STATUS_BAD_BLOCK}


def i32(x):
    return torch.tensor(list(x), dtype=torch.int32, device=DEV)


def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def raw_tables(tables, held, ctx, free, cursor, bs, nb):
    n = len(tables)
    return DeviceTables(block_tables=torch.tensor(tables, dtype=torch.int32, device=DEV)
                        .reshape(n, -1), blocks_held=i32(held), ctx_lens=i32(ctx),
                        free_blocks=i32(free), free_cursor=i32([cursor]), block_size=bs,
                        num_blocks=nb)


def compare_step(tables, held, ctx, q, free, cursor, bs, nb, T, max_q):
    dt = raw_tables(tables, held, ctx, free, cursor, bs, nb)
    st = status()
    meta, after = build_batch_meta(dt, i32(q), T, max_q, status=st)
    host = [list(r) for r in tables]
    e = tree_ref.build_step(host, held, ctx, q, free, cursor, bs, nb, T, max_q)
    assert int(st) == sum(BITS[b] for b in e["status"])
    assert after.block_tables.tolist() == host
    assert after.blocks_held.tolist() == e["held"] and after.ctx_lens.tolist() == e["ctx"]
    assert after.free_cursor.tolist() == [e["cursor"]]
    for name in ("seq_lens", "start_pos", "positions"):
        assert getattr(meta, name).tolist() == e[name], name
    assert meta.query_start_loc.tolist() == e["qsl"]
    assert meta.slot_mapping.tolist() == e["slots"]
    # the state before is as it was
    assert dt.blocks_held.tolist() == list(held) and dt.ctx_lens.tolist() == list(ctx)
    assert dt.free_cursor.tolist() == [cursor]
    return meta, after


def random_step(rng, n, width, bs, qhi):
    held = rng.integers(0, width + 1, size=n)
    ctx = [int(rng.integers(0, h * bs + 1)) for h in held]
    q = [min(int(rng.integers(0, qhi + 1)), width * bs - c) for c in ctx]
    ids = rng.permutation(np.arange(1, n * width * 2 + 40)).tolist()
    tables, at = [], 0
    for h in held:
        tables.append(ids[at:at + h] + [0] * (width - h))
        at += int(h)
    return tables, held.tolist(), ctx, q, ids[at:], len(ids) + 1


@pytest.mark.parametrize("n", [1, 3, 63, 256, 257, 700])
@pytest.mark.parametrize("bs,width,qhi", [(16, 5, 40), (1, 7, 3), (32, 3, 96), (8, 40, 6)])
def test_build_batch_meta(n, bs, width, qhi):
    print(f"[step] n={n} bs={bs} width={width} qhi={qhi}", flush=True)
    rng = np.random.default_rng([n, bs])
    tables, held, ctx, q, free, nb = random_step(rng, n, width, bs, qhi)
    for T in (sum(q), sum(q) + 37):
        compare_step(tables, held, ctx, q, [9] * 4 + free, 4, bs, nb, T, qhi)


def test_build_batch_meta_many_sequences():
    """The scan's LDS past 64 KiB."""
    rng = np.random.default_rng(1)
    tables, held, ctx, q, free, nb = random_step(rng, 16384, 3, 4, 5)
    compare_step(tables, held, ctx, q, free, 0, 4, nb, sum(q), 5)


def test_build_batch_meta_small_ends():
    compare_step([[3, 0]], [1], [4], [0], [5, 6], 0, 16, 9, 0, 0)   # nothing to do
    compare_step([[0, 0]], [0], [0], [1], [5, 6], 1, 16, 9, 1, 1)   # a first token
    compare_step([[3, 4]], [2], [5], [2], [], 0, 16, 9, 2, 2)       # held blocks suffice
    compare_step([[3, 4]], [2], [0], [32], [], 0, 16, 9, 40, 32)    # exactly full
    none = DeviceTables(block_tables=torch.zeros(0, 2, dtype=torch.int32, device=DEV),
                        blocks_held=i32([]), ctx_lens=i32([]), free_blocks=i32([1]),
                        free_cursor=i32([0]), block_size=16, num_blocks=4)
    meta, after = build_batch_meta(none, i32([]), 3, 4)             # no sequence
    assert meta.query_start_loc.tolist() == [0] and after.free_cursor.tolist() == [0]
    assert meta.positions.tolist() == [0] * 3
    assert meta.slot_mapping.tolist() == [tree_ref.NO_SLOT] * 3


@pytest.mark.parametrize("what,kw", [
    ("blocks", dict(free=[5, 6], q=[30, 30])),
    ("blocks", dict(cursor=9)),
    ("blocks", dict(cursor=-1)),
    ("short", dict(q=[1, 49])),
    ("short", dict(ctx=[3, 2147483000])),
    ("qloc", dict(q=[1, -2])),
    ("qloc", dict(q=[1, 60])),
    ("qloc", dict(T=5)),
    ("qloc", dict(ctx=[-1, 0])),
    ("qloc", dict(held=[1, -7])),
])
def test_build_batch_meta_all_or_nothing(what, kw):
    print(f"[step] {what} {kw}", flush=True)
    a = dict(tables=[[1, 0, 0], [2, 0, 0]], held=[1, 1], ctx=[3, 16], q=[2, 20],
             free=[5, 6, 7, 8], cursor=0, T=100)
    a.update(kw)
    dt = raw_tables(a["tables"], a["held"], a["ctx"], a["free"], a["cursor"], 16, 9)
    st = status()
    meta, after = build_batch_meta(dt, i32(a["q"]), a["T"], 50, status=st)
    assert int(st) & BITS[what]
    assert after.block_tables.tolist() == a["tables"]
    assert after.blocks_held.tolist() == a["held"] and after.ctx_lens.tolist() == a["ctx"]
    assert after.free_cursor.tolist() == [a["cursor"]]
    with pytest.raises((RuntimeError, ValueError)):
        raise_step_status(st, "step")
    # slots only in held blocks
    slots = meta.slot_mapping.cpu().numpy()
    real = slots[slots != tree_ref.NO_SLOT]
    assert np.isin(real // 16, [1, 2]).all()


@pytest.mark.parametrize("what,held,ctx,q", [("qloc", 1, 16, -1), ("qloc", -1, 16, 3),
                                             ("short", 1, 16, 40), ("short", 5, 16, 1)])
@pytest.mark.parametrize("n,at", [(1, 0), (64, 63), (256, 64), (256, 255), (301, 256), (301, 300),
                                  (2000, 1999)])
def test_build_batch_meta_one_bad_length_stops_every_sequence(n, at, what, held, ctx, q):
    """Whichever wavefront and turn of the scan meets it, and beside a fault of the
    whole step (a free list too short), which must not hide it."""
    print(f"[step] {what} sequence {at} of {n}", flush=True)
    for free in (n + 8, 0):
        helds, ctxs, qs = [1] * n, [16] * n, [2] * n
        helds[at], ctxs[at], qs[at] = held, ctx, q
        tables = [[1, 0, 0] for _ in range(n)]
        dt = raw_tables(tables, helds, ctxs, [2] * free, 0, 16, 9)
        st = status()
        meta, after = build_batch_meta(dt, i32(qs), 2 * n + 50, 50, status=st)
        short = free == 0 and n > 1  # the others lack a block each
        assert int(st) == BITS[what] | (BITS["blocks"] if short else 0)
        assert after.block_tables.tolist() == tables and after.free_cursor.tolist() == [0]
        assert after.blocks_held.tolist() == helds and after.ctx_lens.tolist() == ctxs
        slots = meta.slot_mapping  # only a table row said to be longer than it is has slots
        assert bool(((slots == tree_ref.NO_SLOT) | (slots // 16 == 1)).all())


def test_build_batch_meta_failed_steps_stay_within_the_rows():
    """More tokens than T: a sequence's rows end at T for whatever runs on."""
    st = status()
    meta, _ = build_batch_meta(raw_tables([[1, 0]] * 3, [1] * 3, [3] * 3, [5], 0, 16, 9),
                               i32([4, 4, 4]), 6, 4, status=st)
    assert int(st) & BITS["qloc"]
    assert meta.query_start_loc.tolist() == [0, 4, 6, 6]


def test_build_batch_meta_bad_block_ids():
    compare_step([[1, 0], [9, 0]], [1, 1], [10, 10], [10, 3], [77, 4], 0, 16, 9, 20, 10)
    with pytest.raises(AssertionError):
        st = status()
        build_batch_meta(raw_tables([[0, 0]], [1], [1], [], 0, 16, 9), i32([1]), 1, 1, status=st)
        raise_step_status(st, "step")


def test_build_batch_meta_equals_the_host_path():
    """The blocks BlockAllocator hands out, and pack_batch_meta's tensors."""
    bs, lens, q = 16, [5, 16, 40, 1], [3, 17, 1, 31]
    alloc = BlockAllocator(64)
    tables = [alloc.allocate_n(-(-x // bs)) for x in lens]
    alloc.free(tables.pop())  # reused first
    tables.append(alloc.allocate_n(1))
    spare = alloc.allocate_n(8)
    dt = DeviceTables.from_host(tables, lens, spare, 4, bs, 64, DEV)
    meta, after = build_batch_meta(dt, i32(q), sum(q), max(q), max_kv_len=64)
    alloc.free(spare)
    for t, c, x in zip(tables, lens, q):
        need = -(-(c + x) // bs) - len(t)
        t.extend(spare[:need])
        spare = spare[need:]
    qsl = np.concatenate([[0], np.cumsum(q)]).tolist()
    pos = [p for c, x in zip(lens, q) for p in range(c, c + x)]
    host = pack_batch_meta(tables, qsl, pos, sum(q), torch.device(DEV), bs)
    w = host.block_tables.shape[1]
    assert torch.equal(meta.block_tables[:, :w], host.block_tables)
    for name in ("seq_lens", "start_pos", "positions", "query_start_loc"):
        assert torch.equal(getattr(meta, name), getattr(host, name)), name
    pool = KVPool(1, bs, 64, 1, 8, torch.float32, DEV)
    slots = torch.cat([pool.make_slot_mapping(c, x, t) for t, c, x in zip(tables, lens, q)])
    assert torch.equal(meta.slot_mapping, slots)
    before = meta.seq_lens.clone()
    meta.advance_()
    assert torch.equal(meta.seq_lens, before + 1)


def test_padded_slots_are_skipped_by_write():
    pool = KVPool(1, 16, 8, 1, 8, torch.float32, DEV)
    dt = raw_tables([[0, 0]], [0], [0], [3, 5], 0, 16, 8)
    meta, _ = build_batch_meta(dt, i32([20]), 24, 20)
    k = torch.randn(24, 1, 8, device=DEV)
    pool.write(0, meta.slot_mapping, k, -k)
    flat = pool.flat_k[0]
    assert torch.equal(flat[48:64], k[:16]) and torch.equal(flat[80:84], k[16:20])
    assert int((flat != 0).any(-1).sum()) == 20


def random_trees(rng, nodes):
    return [np.array([-1] + [int(rng.integers(max(0, i - 5), i)) for i in range(1, n)],
                     dtype=np.int32)[:n] for n in nodes]


@pytest.mark.parametrize("nodes", [[1], [0, 3, 0], [5, 64, 1, 63], [65, 2], [200, 128, 129],
                                   list(range(1, 40)), [700]])
@pytest.mark.parametrize("pad", [0, 3])
def test_build_tree_meta(nodes, pad):
    print(f"[masks] {nodes} pad={pad}", flush=True)
    rng = np.random.default_rng(len(nodes))
    trees = random_trees(rng, nodes)
    if nodes[-1] == 700:  # one chain
        trees = [np.arange(-1, 699, dtype=np.int32)]
    n, T = len(nodes), sum(nodes)
    ctx = rng.integers(0, 1000, size=n)
    qsl = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    flat = np.concatenate(trees + [np.full(pad, 77, dtype=np.int32)]).astype(np.int32)
    dt = raw_tables([[0]] * n, [0] * n, ctx.tolist(), [], 0, 16, 4)
    st = status()
    meta = build_tree_meta(dt, torch.from_numpy(flat).to(DEV), torch.from_numpy(qsl).to(DEV),
                           max(nodes), status=st)
    both = [tree_ref.visible_from_parents(t) for t in trees]
    words = meta.masks.shape[1]
    want = tree_ref.pack_masks([b[0] for b in both], T, words)
    assert int(st) == 0 and words == -(-max(nodes) // 64)
    assert np.array_equal(meta.masks[:T].cpu().numpy(), want)
    pos = np.concatenate([c + b[1] for c, b in zip(ctx, both)])
    assert meta.positions[:T].tolist() == pos.tolist()
    assert (meta.masks[T:] == 0).all() and (meta.positions[T:] == 0).all()


def test_build_tree_meta_bad_parents_and_runs():
    dt = raw_tables([[0]] * 2, [0] * 2, [7, 9], [], 0, 16, 4)
    st = status()
    parents = [-1, 0, 5, -2, 3, -1, 5, 0]
    meta = build_tree_meta(dt, i32(parents), i32([0, 5, 8]), 5, status=st)
    assert int(st) == _native.PKV_STATUS_BAD_PARENT
    vis = [tree_ref.visible_from_parents(parents[:5]), tree_ref.visible_from_parents(parents[5:])]
    assert np.array_equal(meta.masks.cpu().numpy(),
                          tree_ref.pack_masks([v[0] for v in vis], 8, 1))
    with pytest.raises(ValueError):
        raise_step_status(st, "trees")
    for qsl in ([0, 5, 12], [0, 6, 8], [-1, 3, 8]):  # out of range, past the bound
        st.zero_()
        build_tree_meta(dt, i32(parents), i32(qsl), 5, status=st)
        assert int(st) & _native.PKV_STATUS_BAD_QLOC, qsl


@pytest.mark.parametrize("nodes", [[1], [0, 4], [8, 1, 64, 30], [150, 65, 2], [20] * 70])
@pytest.mark.parametrize("depth", [1, 2, 7, 200])
def test_tree_accept(nodes, depth):
    print(f"[accept] {nodes[:6]} depth={depth}", flush=True)
    rng = np.random.default_rng([len(nodes), depth])
    trees = random_trees(rng, nodes)
    if nodes == [1]:
        trees = [np.array([-1], dtype=np.int32)]
    T = sum(nodes)
    parents = np.concatenate(trees).astype(np.int32)
    tokens = rng.integers(0, 4, size=T)   # few values: siblings share tokens
    picks = rng.integers(0, 4, size=T)
    qsl = np.concatenate([[0], np.cumsum(nodes)]).astype(np.int32)
    dt = raw_tables([[0]] * len(nodes), [0] * len(nodes), [0] * len(nodes), [], 0, 16, 4)
    meta = build_tree_meta(dt, i32(parents), i32(qsl), max(nodes))
    st = status()
    a = tree_accept(torch.from_numpy(picks).to(DEV), torch.from_numpy(tokens).to(DEV), meta,
                    depth, status=st)
    lens, path, out = tree_ref.accept(picks, tokens, parents, qsl, depth)
    assert int(st) == 0
    assert a.lens.tolist() == lens and a.path.tolist() == path and a.tokens.tolist() == out


def test_tree_accept_long_chain_and_large_ids():
    n = 300
    parents = np.arange(-1, n - 1).astype(np.int32)
    tokens = (np.arange(n) + (1 << 40)).astype(np.int64)
    picks = np.roll(tokens, -1)
    dt = raw_tables([[0]], [0], [0], [], 0, 16, 4)
    meta = build_tree_meta(dt, i32(parents), i32([0, n]), n)
    a = tree_accept(torch.from_numpy(picks).to(DEV), torch.from_numpy(tokens).to(DEV), meta, 400)
    assert a.lens.tolist() == [n] and a.path[0, :n].tolist() == list(range(n))
    assert a.tokens[0, :n].tolist() == picks.tolist() and (a.tokens[0, n:] == -1).all()


F8 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype,kv", [(torch.float32, None), (torch.bfloat16, None),
                                      (torch.float16, None), (torch.bfloat16, F8),
                                      (torch.float32, F8)])
@pytest.mark.parametrize("hkv,d,layers,bs", [(1, 64, 3, 16), (2, 8, 1, 1), (3, 5, 2, 8),
                                             (1, 1, 1, 16)])
def test_write_accepted(dtype, kv, hkv, d, layers, bs):
    print(f"[commit] {dtype} {kv} hkv={hkv} d={d} layers={layers} bs={bs}", flush=True)
    rng = np.random.default_rng(d)
    g = torch.Generator().manual_seed(d)
    nodes, ctx, depth = [6, 0, 30, 1], [15, 3, 0, 31], 5
    lens = [3, 0, 5, 1]
    T, n = sum(nodes), len(nodes)
    path = np.full((n, depth), -1, dtype=np.int32)
    for s in range(n):
        path[s, :lens[s]] = np.sort(rng.choice(nodes[s], size=lens[s], replace=False)) \
            if lens[s] else []
    width = -(-64 // bs)
    nb = n * width + 2
    tables = rng.permutation(np.arange(1, n * width + 1)).reshape(n, width).tolist()
    pool = KVPool(layers, bs, nb, hkv, d, kv or dtype, DEV)
    init = torch.randn(pool.kv.shape, generator=g).to(kv or dtype)
    pool.kv.copy_(init)
    k = (30 * torch.randn(layers, T, hkv, d, generator=g)).to(dtype)
    v = (200 * torch.randn(layers, T, hkv, d, generator=g)).to(dtype)
    qsl = np.concatenate([[0], np.cumsum(nodes)])
    dt = DeviceTables.from_host(tables, ctx, [], width, bs, nb, DEV)
    tree = build_tree_meta(dt, i32([-1] * T), i32(qsl), max(nodes))
    meta, _ = build_batch_meta(dt, i32(lens), n * depth, depth)
    acc = TreeAccept(lens=i32(lens), path=torch.from_numpy(path).to(DEV), tokens=None)
    pool.debug = True
    pool.write_accepted(k.to(DEV), v.to(DEV), tree, acc, meta)
    want = init.clone()
    for s in range(n):
        if not lens[s]:
            continue
        slots = torch.from_numpy(paged_ref.make_slot_mapping(ctx[s], lens[s], tables[s], bs))
        src = torch.from_numpy(qsl[s] + path[s, :lens[s]]).long()
        for layer in range(layers):
            for j, rows in enumerate((k, v)):
                flat = want[layer, j].view(torch.uint8 if kv else dtype).view(-1, hkv, d)
                new = rows[layer, src].to(kv or dtype)
                flat[slots] = new.view(torch.uint8) if kv else new
    got = pool.kv.cpu()
    if kv:
        got, want = got.view(torch.uint8), want.view(torch.uint8)
    assert torch.equal(got, want)


def test_write_accepted_unaligned_rows():
    pool = KVPool(2, 16, 4, 1, 8, torch.bfloat16, DEV)
    base = torch.randn(1 + 2 * 3 * 8, device=DEV).bfloat16()
    k = base[1:].view(2, 3, 1, 8)
    dt = raw_tables([[2]], [1], [3], [], 0, 16, 4)
    tree = build_tree_meta(dt, i32([-1, 0, 0]), i32([0, 3]), 3)
    meta, _ = build_batch_meta(dt, i32([2]), 2, 2)
    acc = TreeAccept(lens=i32([2]), path=i32([0, 2]).view(1, 2), tokens=None)
    pool.write_accepted(k, k, tree, acc, meta)
    for layer in range(2):
        assert torch.equal(pool.flat_k[layer][35:37], k[layer, [0, 2]])
        assert torch.equal(pool.flat_v[layer][35:37], k[layer, [0, 2]])
        assert int((pool.flat_k[layer] != 0).any(-1).sum()) == 2


def test_write_accepted_bad_entries_write_nothing():
    """Paths outside the run, positions past the table, block 0 and ids past the pool."""
    pool = KVPool(1, 16, 4, 1, 8, torch.float32, DEV)
    k = torch.ones(1, 8, 1, 8, device=DEV)
    tables = raw_tables([[1], [0], [9], [2]], [1] * 4, [0, 0, 0, 15], [], 0, 16, 4)
    tree = build_tree_meta(tables, i32([-1] * 8), i32([0, 2, 4, 6, 8]), 2)
    meta, _ = build_batch_meta(tables, i32([1] * 4), 4, 1)
    acc = TreeAccept(lens=i32([2, 1, 1, 2]), path=i32([2, -1, 0, 0, 0, 0, 1, 1]).view(4, 2),
                     tokens=None)
    pool.write_accepted(k, k, tree, acc, meta)
    used = (pool.flat_k[0] != 0).any(-1).nonzero()[:, 0].tolist()
    assert used == [2 * 16 + 15]
    pool.debug = True
    with pytest.raises((AssertionError, ValueError)):
        pool.write_accepted(k, k, tree, acc, meta)


def test_step_in_a_graph():
    """accept -> build_batch_meta -> write_accepted captured once: every replay, on new
    picks, gives the eager result."""
    rng = np.random.default_rng(3)
    nodes = [7, 3, 20]
    trees = random_trees(rng, nodes)
    T, bs, layers = sum(nodes), 16, 2
    tokens = torch.from_numpy(rng.integers(0, 3, size=T)).to(DEV)
    picks = torch.from_numpy(rng.integers(0, 3, size=T)).to(DEV)
    ctx = [14, 16, 31]
    tables = [[1], [2], [3, 4]]
    qsl = i32(np.concatenate([[0], np.cumsum(nodes)]))
    parents = i32(np.concatenate(trees))
    k = torch.randn(layers, T, 1, 16, device=DEV)
    pool = KVPool(layers, bs, 16, 1, 16, torch.float32, DEV)

    def step():
        dt = DeviceTables(block_tables=state.block_tables.clone(), blocks_held=state.blocks_held,
                          ctx_lens=state.ctx_lens, free_blocks=state.free_blocks,
                          free_cursor=state.free_cursor, block_size=bs, num_blocks=16)
        tree = build_tree_meta(dt, parents, qsl, 20)
        acc = tree_accept(picks, tokens, tree, 6)
        meta, after = build_batch_meta(dt, acc.lens, 18, 6)
        pool.write_accepted(k, -k, tree, acc, meta)
        return [tree.masks, tree.positions, acc.lens, acc.path, acc.tokens, meta.positions,
                meta.slot_mapping, after.block_tables, after.blocks_held, after.free_cursor]

    state = DeviceTables.from_host(tables, ctx, [5, 6, 7, 8], 4, bs, 16, DEV)
    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for it in range(4):
        picks.copy_(torch.from_numpy(rng.integers(0, 3, size=T)))
        k.add_(1.0)
        pool.kv.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got, kv = [t.clone() for t in captured], pool.kv.clone()
        pool.kv.zero_()
        want = step()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), it
        assert torch.equal(kv, pool.kv)
