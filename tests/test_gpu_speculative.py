"""The verification step put together: PagedTransformer.forward_tree against
token-by-token decoding, and generate_speculative against generate_batched.

forward_tree's logits of a node are those of decoding its path token by token: both
are fp32 sums of the same terms in another order. The pass is 2 layers of
projections of at most 128 terms and attention over at most 60 keys; a sum of n
terms is off by at most n 2^-24 of the terms' absolute sum, and the bound used,
1e-4 of the logits' scale, leaves a factor of 1700 over 2^-24 for the absolute sums
and their passage through 9 projections of up to 128 terms (9 * 128 = 1152)."""
from dataclasses import replace

import numpy as np
import pytest
import torch

from serving.allocator import BlockAllocator
from serving.batch import build_batch_step
from serving.generation import generate_batched, generate_speculative
from serving.kv_pool import KVPool
from serving.layers import ModelConfig
from serving.paged_meta import DeviceTables, build_batch_meta, raise_step_status
from serving.paged_model import PagedTransformer
from serving.sequence import Sequence
from serving.tree_decode import build_tree_meta, paged_tree_attention, tree_accept

pytestmark = pytest.mark.gpu
DEV = "cuda"


def small_model(dtype=torch.float32, heads=4, kv_heads=1):
    cfg = ModelConfig(vocab_size=97, d_model=128, num_layers=2, num_heads=heads,
                      num_kv_heads=kv_heads, max_seq_len=160)
    torch.manual_seed(0)
    return cfg, PagedTransformer(cfg).to(DEV, dtype).eval()


def make_pool(cfg, dtype, blocks=128, bs=16):
    return KVPool(cfg.num_layers, bs, blocks, cfg.num_kv_heads, cfg.head_dim, dtype, DEV)


def prefill(model, pool, alloc, prompts, bs=16):
    seqs = [Sequence(i, list(p), bs) for i, p in enumerate(prompts)]
    for s in seqs:
        s.ensure_blocks(alloc)
    logits = model.forward_batch(build_batch_step([(s, s.token_ids) for s in seqs], DEV), pool)
    return seqs, logits.argmax(-1).tolist()


@pytest.mark.parametrize("heads,kv_heads", [(4, 1), (4, 2), (2, 2)])
def test_forward_tree_equals_decoding_each_path(heads, kv_heads):
    cfg, model = small_model(heads=heads, kv_heads=kv_heads)
    rng = np.random.default_rng(1)
    prompts = [rng.integers(0, 97, size=n).tolist() for n in (5, 33, 16)]
    pool, alloc = make_pool(cfg, torch.float32), BlockAllocator(128)
    seqs, _ = prefill(model, pool, alloc, prompts)
    trees = [[-1, 0, 0, 1, 2, 2, 5], [-1], [-1, 0, 1, 2, 3]]
    tokens = [rng.integers(0, 97, size=len(t)).tolist() for t in trees]
    flat = torch.tensor([t for ts in tokens for t in ts], device=DEV)
    parents = torch.tensor([p for t in trees for p in t], dtype=torch.int32, device=DEV)
    qsl = torch.tensor(np.concatenate([[0], np.cumsum([len(t) for t in trees])]),
                       dtype=torch.int32, device=DEV)
    tables = DeviceTables.from_host([s.block_table for s in seqs], [len(p) for p in prompts], [],
                                    8, 16, 128, DEV)
    before = pool.kv.clone()
    logits, k_rows, v_rows = model.forward_tree(flat, pool, build_tree_meta(tables, parents, qsl, 7))
    assert torch.equal(pool.kv, before)  # read only
    at = 0
    for s, tree in enumerate(trees):
        for i in range(len(tree)):
            path, up = [], i
            while up >= 0:
                path.insert(0, tokens[s][up])
                up = tree[up]
            scratch, a2 = make_pool(cfg, torch.float32), BlockAllocator(128)
            seq = Sequence(0, prompts[s] + path, 16)
            seq.ensure_blocks(a2)
            want = model.forward_batch(build_batch_step([(seq, seq.token_ids)], DEV), scratch)[0]
            scale = float(want.abs().max())
            assert float((logits[at + i] - want).abs().max()) <= 1e-4 * scale, (s, i)
            # the row that would be committed is the one decoding writes
            slot = seq.block_table[(seq.num_tokens - 1) // 16] * 16 + (seq.num_tokens - 1) % 16
            for layer in range(cfg.num_layers):
                for rows, flat_pool in ((k_rows, scratch.flat_k), (v_rows, scratch.flat_v)):
                    w = flat_pool[layer][slot]
                    assert float((rows[layer, at + i] - w).abs().max()) <= \
                        1e-4 * float(w.abs().max())
        at += len(tree)


def drafts(kind, truth, prompts):
    """Drafting functions: the greedy continuation itself, on one branch among wrong
    ones or cut short, wrong tokens only, or nothing."""
    rng = np.random.default_rng(5)

    def find(history):
        for p, t in zip(prompts, truth):
            full = p + t
            if full[:len(history)] == history:
                return full[len(history):]
        raise AssertionError("the history left the greedy continuation")

    def draft(history):
        rest = find(history)
        if kind == "none":
            return [], []
        if kind == "wrong":
            bad = [(rest[0] + 1) % 97 if rest else 0] * 3
            return bad, [-1, 0, -1]
        if kind == "chain":
            chain = rest[:int(rng.integers(0, 6))]
            return chain, list(range(-1, len(chain) - 1))
        # branches: at each depth a wrong token first, then the right one
        toks, pars, last = [], [], -1
        for t in rest[:5]:
            toks += [(t + 1) % 97, t]
            pars += [last, last]
            last = len(toks) - 1
        return toks, pars

    return draft


@pytest.mark.parametrize("kind", ["none", "wrong", "chain", "branches"])
def test_generate_speculative_gives_the_greedy_tokens(kind):
    print(f"[speculative] {kind}", flush=True)
    cfg, model = small_model()
    rng = np.random.default_rng(2)
    prompts = [rng.integers(0, 97, size=n).tolist() for n in (7, 1, 40)]
    pool, alloc = make_pool(cfg, torch.float32), BlockAllocator(128)
    truth = generate_batched(model, prompts, 60, pool, alloc)
    longer = generate_batched(model, prompts, 70, pool, alloc)
    free = alloc.num_free
    calls = []
    fn = drafts(kind, longer, prompts)

    def counted(history):
        calls.append(len(history))
        return fn(history)

    got = generate_speculative(model, prompts, 60, pool, alloc, counted, max_drafts=11,
                               max_depth=6)
    assert got == truth and alloc.num_free == free
    if kind == "branches":  # a bonus token and five drafts a step
        assert len(calls) <= 3 * 11
    if kind in ("none", "wrong"):
        assert len(calls) == 3 * 59


def test_generate_speculative_16_bit_and_fp8_pools():
    """16-bit passes round along the way, so a token may differ from the other kernels'
    where two logits lie within the rounding of each other: the tokens are checked to be
    greedy under the paged decode path, up to 2^-5 of the logits' scale (8 roundings of
    2^-8 relative)."""
    for dtype, kv in ((torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float8_e4m3fn)):
        # fp8 decode attention needs 16 heads of 64
        cfg = ModelConfig(vocab_size=97, d_model=1024, num_layers=1, num_heads=16,
                          num_kv_heads=1, max_seq_len=160)
        torch.manual_seed(0)
        model = PagedTransformer(cfg).to(DEV, dtype).eval()
        rng = np.random.default_rng(3)
        prompts = [rng.integers(0, 97, size=n).tolist() for n in (20, 5)]
        pool, alloc = make_pool(cfg, kv), BlockAllocator(128)
        got = generate_speculative(model, prompts, 24, pool, alloc,
                                   lambda h: ([h[-1], h[0], 3], [-1, -1, 0]))
        for p, toks in zip(prompts, got):
            assert len(toks) == 24
            seq = Sequence(0, list(p), 16)
            seq.ensure_blocks(alloc)
            logits = model.forward_batch(build_batch_step([(seq, seq.token_ids)], DEV), pool)[0]
            for t in toks:
                top = logits.float().max()
                assert float(top - logits[t].float()) <= 2 ** -5 * float(logits.float().abs().max())
                seq.append_token(t)
                seq.ensure_blocks(alloc)
                logits = model.forward_batch(build_batch_step([(seq, [t])], DEV), pool)[0]
            seq.release(alloc)


def test_generate_speculative_edges():
    cfg, model = small_model()
    pool, alloc = make_pool(cfg, torch.float32, blocks=10), BlockAllocator(10)
    none = lambda h: ([], [])  # noqa: E731
    assert generate_speculative(model, [], 5, pool, alloc, none) == []
    assert generate_speculative(model, [[1]], 0, pool, alloc, none) == [[]]
    one = generate_speculative(model, [[1, 2]], 1, pool, alloc, none)
    assert one == generate_batched(model, [[1, 2]], 1, pool, alloc)
    assert generate_speculative(model, [[1, 2]], 9, pool, alloc, none, max_drafts=0,
                                max_depth=1) == generate_batched(model, [[1, 2]], 9, pool, alloc)
    for bad in ([], [0]), ([1], [0]), ([1, 2], [-1, 1]), ([1], [-2]), ([97], [-1]), ([-1], [-1]):
        with pytest.raises(ValueError):
            generate_speculative(model, [[1, 2]], 5, pool, alloc, lambda h, b=bad: b)
    with pytest.raises(ValueError):
        generate_speculative(model, [[1], []], 5, pool, alloc, none)
    with pytest.raises(ValueError):
        generate_speculative(model, [[1]], -1, pool, alloc, none)
    with pytest.raises(ValueError):
        generate_speculative(model, [[1]], 5, pool, alloc, none, max_depth=0)
    with pytest.raises(RuntimeError):  # more than the pool holds
        generate_speculative(model, [[1]], 500, pool, alloc, none)
    assert alloc.num_free == 9


@pytest.mark.parametrize("new", [1, 2, 17, 33])
def test_generate_speculative_needs_what_generate_batched_needs(new):
    """A pool that holds exactly the tokens, prompts that end with the model's last
    position, and drafts that are right and go on past the goal."""
    cfg, model = small_model()
    n = cfg.max_seq_len + 1 - new  # the last token takes no position
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 97, size=n).tolist(), rng.integers(0, 97, size=3).tolist()]
    blocks = 1 + cfg.max_seq_len // 16 + -(-(3 + new - 1) // 16)
    pool, alloc = make_pool(cfg, torch.float32, blocks=blocks), BlockAllocator(blocks)
    truth = generate_batched(model, prompts, new, pool, alloc)
    fn = drafts("chain", [t + [1] * 20 for t in truth], prompts)
    assert generate_speculative(model, prompts, new, pool, alloc, fn) == truth
    assert alloc.num_free == blocks - 1


def test_step_captured_with_the_model():
    """A whole verification step (masks, model, picks, acceptance, blocks, commit) as one
    graph, replayed on other trees' tokens: the eager step's results."""
    cfg, model = small_model()
    rng = np.random.default_rng(4)
    prompts = [rng.integers(0, 97, size=n).tolist() for n in (15, 30)]
    pool, alloc = make_pool(cfg, torch.float32), BlockAllocator(128)
    seqs, first = prefill(model, pool, alloc, prompts)
    stock = alloc.allocate_n(6)
    tables = DeviceTables.from_host([s.block_table for s in seqs], [15, 30], stock, 5, 16, 128, DEV)
    parents = torch.tensor([-1, 0, 0, 1, 3, -1, 0, 1, 2, 2], dtype=torch.int32, device=DEV)
    qsl = torch.tensor([0, 5, 10], dtype=torch.int32, device=DEV)
    ids = torch.tensor(rng.integers(0, 97, size=10), device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    kv0 = pool.kv.clone()

    def step():
        pool.kv.copy_(kv0)
        dt = DeviceTables(tables.block_tables.clone(), tables.blocks_held, tables.ctx_lens,
                          tables.free_blocks, tables.free_cursor, 16, 128)
        tree = build_tree_meta(dt, parents, qsl, 5, status=status)
        logits, k, v = model.forward_tree(ids, pool, tree)
        acc = tree_accept(logits.argmax(-1), ids, tree, 4, status=status)
        meta, after = build_batch_meta(dt, acc.lens, 8, 4, status=status)
        pool.write_accepted(k, v, tree, acc, meta)
        return [logits, acc.lens, acc.path, acc.tokens, after.block_tables, after.blocks_held,
                after.ctx_lens, after.free_cursor, pool.kv]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for it in range(3):
        # drafts that the model confirms now and then: its own greedy tokens
        out = step()
        ids.copy_(torch.from_numpy(rng.integers(0, 97, size=10)))
        if it:
            ids[1], ids[6] = out[0][0].argmax(), out[0][5].argmax()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        want = [t.clone() for t in step()]
        assert all(torch.equal(a, b) for a, b in zip(got, want)), it
    raise_step_status(status, "step")


def test_metadata_of_another_batch_is_refused():
    cfg, model = small_model()
    pool = make_pool(cfg, torch.float32, blocks=4)
    tables = DeviceTables.from_host([[1], [2]], [5, 9], [3], 2, 16, 4, DEV)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    tree = build_tree_meta(tables, i32([-1, 0, -1]), i32([0, 2, 3]), 2)
    x = torch.zeros(3, cfg.num_heads, cfg.head_dim, device=DEV)
    kv = torch.zeros(3, 1, cfg.head_dim, device=DEV)
    ids = torch.zeros(3, dtype=torch.long, device=DEV)
    for name in ("ctx_lens", "query_start_loc"):
        bad = replace(tree, **{name: getattr(tree, name)[:-1]})
        with pytest.raises(ValueError):
            paged_tree_attention(x, kv, kv, pool.flat_k[0].view(4, 16, 1, -1),
                                 pool.flat_v[0].view(4, 16, 1, -1), bad)
    for name in ("parents", "query_start_loc"):
        with pytest.raises(ValueError):
            tree_accept(ids, ids, replace(tree, **{name: getattr(tree, name)[:-1]}), 2)
    accepted = tree_accept(ids, ids, tree, 2)
    meta, _ = build_batch_meta(tables, accepted.lens, 4, 2)
    rows = torch.zeros(cfg.num_layers, 3, 1, cfg.head_dim, device=DEV)
    for name in ("block_tables", "start_pos"):
        with pytest.raises(ValueError):
            pool.write_accepted(rows, rows, tree, accepted,
                                replace(meta, **{name: getattr(meta, name)[:-1]}))
    with pytest.raises(ValueError):
        pool.write_accepted(rows, rows, replace(tree, query_start_loc=tree.query_start_loc[:-1]),
                            accepted, meta)
    pool.write_accepted(rows, rows, tree, accepted, meta)
