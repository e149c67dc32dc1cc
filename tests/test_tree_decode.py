"""Refusals of the tree-verification calls, on the host: argument checks of the C
entry points and of the Python wrappers. Nothing is launched."""
import numpy as np
import pytest
import torch

from oracle import tree_ref
from serving import _native
from serving.generation import _draft_tree
from serving.kv_pool import KVPool
from serving.paged_meta import DeviceTables, build_batch_meta, raise_step_status
from serving.tree_decode import (TreeAccept, TreeMeta, build_tree_meta, paged_tree_attention,
                                 tree_accept)

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


def attention(**kw):
    a = dict(out=16, lse=None, q=16, k=16, v=16, kp=16, vp=16, nb=8, bs=16, table=16, max_blk=4,
             ctx=16, qsl=16, masks=16, words=1, n=2, T=8, nodes=4, max_ctx=64, hq=8, hkv=1, d=64,
             scale=0.0, part=0, dtype=2, ws=None, wsb=0)
    a.update(kw)
    return _native.lib().pkv_paged_tree_attention(*a.values(), None, None)


@pytest.mark.parametrize("rc,word,kw", [
    (INVALID, b"dtype", dict(dtype=9)),
    (UNSUPPORTED, b"fp8", dict(dtype=0x100)),
    (INVALID, b"multiple of Hkv", dict(hq=8, hkv=3)),
    (INVALID, b"multiple of Hkv", dict(hkv=0)),
    (INVALID, b"multiple of 8", dict(d=60)),
    (INVALID, b"multiple of 8", dict(d=0)),
    (UNSUPPORTED, b"256", dict(d=264)),
    (INVALID, b"power of two", dict(bs=12)),
    (INVALID, b"power of two", dict(bs=0)),
    (INVALID, b"sizes", dict(n=-1)),
    (INVALID, b"sizes", dict(part=-1)),
    (INVALID, b"sizes", dict(nodes=-1)),
    (UNSUPPORTED, b"4096", dict(nodes=4097, words=65)),
    (UNSUPPORTED, b"2^30", dict(max_blk=(1 << 26) + 1)),
    (UNSUPPORTED, b"65536", dict(n=65537)),
    (UNSUPPORTED, b"2 GiB", dict(bs=1 << 24, max_blk=1)),
    (INVALID, b"max_nodes", dict(nodes=65)),
    (INVALID, b"max_nodes", dict(words=0)),
    (INVALID, b"null", dict(masks=None)),
    (INVALID, b"null", dict(k=None)),
    (INVALID, b"null", dict(table=None)),
    (UNSUPPORTED, b"aligned", dict(q=18)),
    (UNSUPPORTED, b"aligned", dict(vp=24)),
    (UNSUPPORTED, b"aligned", dict(vp=20, dtype=0x102)),
    (WORKSPACE, b"workspace", dict(part=64, max_blk=64, max_ctx=1024)),
    (WORKSPACE, b"workspace", dict(part=64, max_blk=64, max_ctx=1024, ws=16, wsb=100)),
])
def test_attention_refusals(rc, word, kw):
    assert attention(**kw) == rc
    assert word in _native.lib().pkv_last_error()


def test_attention_with_nothing_to_do():
    for kw in (dict(n=0), dict(T=0), dict(nodes=0)):
        assert attention(**kw, q=None, table=None) == 0


def test_workspace_sizing():
    f = _native.lib().pkv_tree_attention_workspace_bytes
    args = dict(n=2, nodes=4, hq=8, hkv=1, d=64, max_blk=64, bs=16, max_ctx=1024, part=64, dtype=2)
    size = lambda **kw: f(*{**args, **kw}.values())  # noqa: E731
    assert size() >= 2 * 16 * 32 * 66 * 4       # 16 pieces of 32 rows each
    assert size(part=1024) == 0                 # one piece
    assert size(max_ctx=64, part=0) == 0        # never split
    assert size(max_ctx=0) == size() and size(max_ctx=0, part=0) == size(part=0) > 0
    assert size(nodes=0) == size(hkv=0) == size(part=-1) == size(d=0) == 0


def step(**kw):
    a = dict(table=16, max_blk=4, held=16, ctx=16, q=16, n=2, free=16, nfree=4, cursor=16, bs=16,
             nb=8, T=8, max_q=4, held_out=32, ctx_out=48, cursor_out=64, qsl=16, seq=16, start=16,
             pos=16, slots=16)
    a.update(kw)
    return _native.lib().pkv_build_step(*a.values(), None, None)


@pytest.mark.parametrize("rc,word,kw", [
    (INVALID, b"power of two", dict(bs=24)),
    (INVALID, b"sizes", dict(n=-1)),
    (INVALID, b"sizes", dict(T=-1)),
    (INVALID, b"sizes", dict(max_q=-1)),
    (UNSUPPORTED, b"16384", dict(n=16385)),
    (UNSUPPORTED, b"too large", dict(n=16384, max_q=1 << 20)),
    (UNSUPPORTED, b"too large", dict(max_blk=1 << 30)),
    (UNSUPPORTED, b"too large", dict(T=(1 << 30) + 1)),
    (INVALID, b"null", dict(held=None)),
    (INVALID, b"null", dict(table=None)),
    (INVALID, b"null", dict(free=None)),
    (INVALID, b"null", dict(slots=None)),
    (INVALID, b"null", dict(cursor_out=None)),
    (INVALID, b"blocks_held_out", dict(held_out=16)),
    (INVALID, b"ctx_lens_out", dict(ctx_out=16)),
    (INVALID, b"free_cursor_out", dict(cursor_out=16)),
])
def test_build_step_refusals(rc, word, kw):
    assert step(**kw) == rc and word in _native.lib().pkv_last_error()


def test_mask_accept_and_commit_refusals():
    L = _native.lib()
    assert L.pkv_tree_masks(16, 1, 16, 16, 16, 16, 2, 8, 65, None, None) == INVALID
    assert L.pkv_tree_masks(16, 0, 16, 16, 16, 16, 2, 8, 0, None, None) == INVALID
    assert L.pkv_tree_masks(16, 1, None, 16, 16, 16, 2, 8, 4, None, None) == INVALID
    assert L.pkv_tree_masks(16, 1, 16, 16, 16, 16, -1, 8, 4, None, None) == INVALID
    assert L.pkv_tree_masks(None, 1, None, None, None, None, 2, 0, 4, None, None) == 0
    accept = lambda n, t, depth, picks=16: L.pkv_tree_accept(  # noqa: E731
        16, 16, 16, picks, 16, 16, 16, n, t, depth, None, None)
    assert accept(2, 8, 0) == INVALID and b"max_depth" in L.pkv_last_error()
    assert accept(-1, 8, 1) == INVALID and accept(2, 8, 1, None) == INVALID
    assert accept(0, 0, 1) == 0
    commit = lambda **kw: L.pkv_write_accepted(*{**dict(  # noqa: E731
        kp=16, vp=16, pl=64, layers=1, nb=4, bs=16, k=16, v=16, rl=64, table=16, max_blk=2,
        start=16, qsl=16, path=16, lens=16, n=2, T=8, depth=2, row=64, dtype=2), **kw}.values(),
        None, None)
    assert commit(dtype=7) == INVALID and commit(bs=10) == INVALID
    assert commit(row=0) == INVALID and commit(layers=-1) == INVALID
    assert commit(path=None) == INVALID and commit(table=None) == INVALID
    assert commit(layers=0, k=None) == 0 and commit(n=0) == 0 and commit(depth=0) == 0


def host_tables():
    return DeviceTables.from_host([[1, 2], [3]], [20, 16], [4, 5], 3, 16, 8, "cpu")


def test_from_host():
    t = host_tables()
    assert t.block_tables.tolist() == [[1, 2, 0], [3, 0, 0]] and t.blocks_held.tolist() == [2, 1]
    assert t.ctx_lens.tolist() == [20, 16] and t.free_blocks.tolist() == [4, 5]
    with pytest.raises(ValueError, match="rows hold"):
        DeviceTables.from_host([[1, 2]], [1], [], 1, 16, 8, "cpu")
    with pytest.raises(ValueError, match="tokens in"):
        DeviceTables.from_host([[1]], [17], [], 1, 16, 8, "cpu")
    with pytest.raises(ValueError, match="lengths"):
        DeviceTables.from_host([[1]], [], [], 1, 16, 8, "cpu")


def tree_meta():
    t = host_tables()
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)  # noqa: E731
    return TreeMeta(block_tables=t.block_tables, ctx_lens=t.ctx_lens, query_start_loc=i32(0, 2, 3),
                    parents=i32(-1, 0, -1), masks=torch.zeros(3, 1, dtype=torch.int64),
                    positions=i32(20, 21, 16), num_seqs=2, num_tokens=3, max_nodes=2,
                    max_ctx_len=20, block_size=16, num_blocks=8)


def test_wrappers_need_a_device():
    i32 = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm"):
        build_batch_meta(host_tables(), i32, 2, 1)
    with pytest.raises(RuntimeError, match="ROCm"):
        build_tree_meta(host_tables(), i32, torch.zeros(3, dtype=torch.int32), 1)
    q, k, p = torch.zeros(3, 8, 64), torch.zeros(3, 1, 64), torch.zeros(8, 16, 1, 64)
    with pytest.raises(RuntimeError, match="ROCm"):
        paged_tree_attention(q, k, k, p, p, tree_meta())
    with pytest.raises(RuntimeError, match="ROCm"):
        tree_accept(torch.zeros(3, dtype=torch.int64), torch.zeros(3, dtype=torch.int64),
                    tree_meta(), 2)
    pool = KVPool(1, 16, 8, 1, 64, torch.float32, "cpu")
    with pytest.raises(RuntimeError, match="ROCm"):
        pool.write_accepted(k[None], k[None], tree_meta(),
                            TreeAccept(i32, i32.view(2, 1), None), None)


def test_status_word():
    for bits, err in ((_native.PKV_STATUS_OUT_OF_BLOCKS, RuntimeError),
                      (_native.PKV_STATUS_SHORT_TABLE, ValueError),
                      (_native.PKV_STATUS_BAD_QLOC, ValueError),
                      (_native.PKV_STATUS_BAD_PARENT, ValueError),
                      (_native.PKV_STATUS_BAD_BLOCK, AssertionError)):
        with pytest.raises(err):
            raise_step_status(torch.tensor([bits], dtype=torch.int32), "step")
    raise_step_status(torch.zeros(1, dtype=torch.int32), "step")


def test_oracle_against_hand_counts():
    vis, depth = tree_ref.visible_from_parents([-1, 0, 0, 2, 7])
    assert vis.sum(1).tolist() == [1, 2, 2, 3, 1] and depth.tolist() == [0, 1, 1, 2, 0]
    assert tree_ref.pack_masks([vis], 5, 1)[:, 0].tolist() == [1, 3, 5, 13, 16]
    assert tree_ref.accept([5, 6, 7, 8], [1, 5, 5, 6], [-1, 0, 0, 1], [0, 4], 3) == (
        [3], [[0, 1, 3]], [[5, 6, 8]])
    q = np.array([[[1.0]], [[0.0]]])
    k, v = np.array([[[2.0]], [[5.0]]]), np.array([[[1.0]], [[3.0]]])
    pool = np.zeros((2, 1, 1, 1))
    out, lse, _, _, _ = tree_ref.tree_attention(q, k, v, pool, pool + 7, [[1]], [1], [0, 2],
                                                [np.array([[True, False], [False, True]])])
    w = np.exp(2.0) / (np.exp(2.0) + 1)
    assert abs(out[0, 0, 0] - (w * 1 + (1 - w) * 7)) < 1e-12 and abs(out[1, 0, 0] - 5) < 1e-12
    assert abs(lse[1, 0] - np.log(2)) < 1e-12
    t = [[3, 0], [0, 0]]
    r = tree_ref.build_step(t, [1, 0], [15, 0], [2, 1], [6, 7, 8], 1, 16, 9, 4, 2)
    assert t == [[3, 7], [8, 0]] and r["slots"][:3] == [63, 112, 128] and r["cursor"] == 3


@pytest.mark.parametrize("limit,depth,want", [
    (9, 9, ([5, 6, 7, 8, 9, 10], [0, 1, 0, 2, 3, 4])),
    (4, 9, ([5, 6, 7, 8], [0, 1, 0, 2])),
    (9, 3, ([5, 6, 7, 9], [0, 1, 0, 3])),
    (3, 3, ([5, 6, 7], [0, 1, 0])),
    (9, 2, ([5, 7], [0, 0])),
    (9, 1, ([], [])),
    (0, 9, ([], [])),
])
def test_draft_trees_are_cut_to_what_a_step_can_keep(limit, depth, want):
    """Nodes too deep, and those below them, leave their places to others."""
    draft = lambda h: ([5, 6, 7, 8, 9, 10], [-1, 0, -1, 1, 2, 3])  # noqa: E731
    assert _draft_tree(draft, [1], limit, depth, 97) == want
