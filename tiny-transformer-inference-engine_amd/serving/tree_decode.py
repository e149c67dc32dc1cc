"""Verification of drafted token trees over the paged cache (the target model's
step of speculative decoding).

A step takes, per sequence, a tree of drafted tokens: node 0 is the last token
the sequence is sure of (its K/V are not in the pool yet), every other node
continues an earlier one. The model runs all nodes at once; each attends to its
sequence's paged context and to itself and its ancestors. The nodes' K/V rows stay
in dense tensors until it is known which are kept, so rejected drafts cost
no pool slots.

  build_tree_meta        ancestor masks and RoPE positions from parent indices
  paged_tree_attention   the attention of one layer
  tree_accept            each tree's longest path the model's picks confirm
  paged_meta.build_batch_meta   blocks and slots for the accepted tokens, from
                         lengths that only the device knows
  KVPool.write_accepted  the accepted rows of all layers into the pool

None of these synchronises the host. serving.generation.generate_speculative
runs them with a drafting function. The reference has no counterpart; its greedy loop
(serving/generation.py:112-148) gives the tokens that a verified run has to give.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _native
from .paged_meta import DeviceTables, _status_ptr

__all__ = ["TreeMeta", "TreeAccept", "build_tree_meta", "paged_tree_attention", "tree_accept"]

MAX_TREE_NODES = 4096
_I32 = torch.int32


@dataclass
class TreeMeta:
    block_tables: torch.Tensor     # int32 [N, max_blocks]
    ctx_lens: torch.Tensor         # int32 [N] context in the pool
    query_start_loc: torch.Tensor  # int32 [N + 1] first node of each sequence
    parents: torch.Tensor          # int32 [T] parent's index in its tree, -1: none
    masks: torch.Tensor            # int64 [T, W] bit j: tree key j is visible
    positions: torch.Tensor        # int32 [T] context length + depth
    num_seqs: int
    num_tokens: int
    max_nodes: int
    max_ctx_len: int
    block_size: int
    num_blocks: int                # that the tables may name: the pools have as many, or more


@dataclass
class TreeAccept:
    lens: torch.Tensor    # int32 [N] nodes accepted, the root among them
    path: torch.Tensor    # int32 [N, max_depth] their indices in the tree, then -1
    tokens: torch.Tensor  # int64 [N, max_depth] the pick at each: the next tokens


def _int_tensor(t, dtype, numel, device, name, what):
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{what}: {name} must be {dtype} on {device} (got {t.dtype} on {t.device})")
    if t.numel() != numel:
        raise ValueError(f"{what}: {name} has {t.numel()} elements, expected {numel}")
    return t if t.is_contiguous() else t.contiguous()


def build_tree_meta(tables: DeviceTables, parents: torch.Tensor, query_start_loc: torch.Tensor,
                    max_nodes: int, max_ctx_len: int = 0,
                    status: Optional[torch.Tensor] = None) -> TreeMeta:
    """Masks and positions of a step's trees: parents int32 [T], sequence s's
    nodes in rows query_start_loc[s] ... query_start_loc[s + 1] - 1 (int32 [N + 1]).
    A node's parent is an earlier node of its tree or -1 (a root). max_nodes bounds
    the trees' sizes, max_ctx_len (0: the table's capacity) the contexts. Rows
    behind the last sequence get empty masks and position 0. `status` as in
    build_batch_meta."""
    what = "build_tree_meta"
    bt = tables.block_tables
    _native.require_device(bt, what=what)
    dev = bt.device
    n, max_blocks = bt.shape
    T = parents.numel()
    parents = _int_tensor(parents, torch.int32, T, dev, "parents", what)
    qsl = _int_tensor(query_start_loc, torch.int32, n + 1, dev, "query_start_loc", what)
    max_nodes = int(max_nodes)
    if not 0 <= max_nodes <= MAX_TREE_NODES:
        raise ValueError(f"{what}: max_nodes must be in [0, {MAX_TREE_NODES}]")
    words = max(1, -(-max_nodes // 64))
    previous = _native.make_current(dev)
    try:
        masks = torch.empty((T, words), dtype=torch.int64, device=dev)
        positions = bt.new_empty(T)
        rc = _native.calls().pkv_tree_masks(
            masks.data_ptr(), words, positions.data_ptr(), parents.data_ptr(), qsl.data_ptr(),
            tables.ctx_lens.data_ptr(), n, T, max_nodes,
            None if status is None else _status_ptr(status, dev, what), _native.stream_ptr(dev))
    finally:
        _native.restore(previous)
    if rc:
        _native.check(rc, what)
    bs = tables.block_size
    cap = max_blocks * bs  # contexts past the table do not exist
    return TreeMeta(bt, tables.ctx_lens, qsl, parents, masks, positions, n, T, max_nodes,
                    min(int(max_ctx_len), cap) if max_ctx_len > 0 else cap, bs,
                    tables.num_blocks)


def _dense(t: torch.Tensor) -> torch.Tensor:
    """t contiguous and 16-byte aligned, as the kernel reads it."""
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def paged_tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                         k_pool: torch.Tensor, v_pool: torch.Tensor, meta: TreeMeta,
                         scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                         lse: Optional[torch.Tensor] = None, part_tokens: int = 0,
                         status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """q [T, Hq, D] of the trees' nodes attends to each sequence's context in the
    pools [num_blocks, block_size, Hkv, D] and to the tree keys of k, v [T, Hkv, D]
    that meta.masks shows each node. fp32, float16 or bfloat16; pools of the same
    type or float8_e4m3fn (the tree's rows then count as rounded to it). `out` /
    `lse` (float32 [T, Hq]): where to write, memory of no other operand; rows of no
    sequence are left as they were there. A row that sees no key gives 0 and lse +inf. part_tokens (0:
    automatic) forces the length of the pieces a context is split into. `status` as in
    build_batch_meta."""
    what = "paged_tree_attention"
    masks, table = meta.masks, meta.block_tables
    dev = q.device
    if not (q.is_cuda and k.device == dev and v.device == dev and k_pool.device == dev
            and v_pool.device == dev and masks.device == dev and table.device == dev):
        _native.require_device(q, k, v, k_pool, v_pool, masks, what=what)
        raise RuntimeError(f"{what}: q, k, v, the pools and the metadata must share a device")
    if ((q.requires_grad or k.requires_grad or v.requires_grad or k_pool.requires_grad
         or v_pool.requires_grad) and torch.is_grad_enabled()):
        raise NotImplementedError(
            f"{what} is forward-only (inference); run it under torch.no_grad()")
    shape, pool_shape = q.shape, k_pool.shape
    if len(shape) != 3 or len(pool_shape) != 4 or pool_shape != v_pool.shape:
        raise ValueError(f"{what}: q must be [T, Hq, D], the pools [num_blocks, block_size, Hkv, D]")
    T, hq, d = shape
    nb, bs, hkv, pd = pool_shape
    if pd != d or k.shape != (T, hkv, d) or v.shape != k.shape:
        raise ValueError(f"{what}: k and v must be [{T}, {hkv}, {d}] (got {tuple(k.shape)}, "
                         f"{tuple(v.shape)}), the pools' head dim {d} (got {pd})")
    if T != meta.num_tokens or bs != meta.block_size or nb < meta.num_blocks:
        raise ValueError(f"{what}: {T} rows and {nb} blocks of {bs}, the metadata has "
                         f"{meta.num_tokens} and {meta.num_blocks} of {meta.block_size}")
    dtype = q.dtype
    if k.dtype != dtype or v.dtype != dtype or v_pool.dtype != k_pool.dtype:
        raise TypeError(f"{what}: q, k and v must share a dtype, and so must the pools")
    if not (k_pool.is_contiguous() and v_pool.is_contiguous()):
        raise ValueError(f"{what}: the pools must be contiguous")
    code = _native.kv_code(dtype, k_pool.dtype)
    if masks.dtype != torch.int64 or masks.dim() != 2 or masks.shape[0] != T:
        raise ValueError(f"{what}: masks must be int64 [{T}, words]")
    if lse is not None and (lse.shape != (T, hq) or lse.dtype != torch.float32
                            or lse.device != dev or not lse.is_contiguous()):
        raise ValueError(f"{what}: lse must be contiguous float32 [{T}, {hq}] on {dev}")
    n, max_blk = table.shape
    ctx, qsl = meta.ctx_lens, meta.query_start_loc
    if ctx.numel() != n or qsl.numel() != n + 1:
        raise ValueError(f"{what}: the metadata's tensors are not those of {n} sequences")
    if (table.dtype != _I32 or ctx.dtype != _I32 or qsl.dtype != _I32 or ctx.device != dev
            or qsl.device != dev or not (table.is_contiguous() and ctx.is_contiguous()
                                         and qsl.is_contiguous())):
        raise ValueError(f"{what}: block_tables, ctx_lens and query_start_loc must be contiguous "
                         f"int32 on {dev}")
    max_nodes, max_ctx = meta.max_nodes, meta.max_ctx_len
    calls = _native.calls()
    previous = _native.make_current(dev)
    try:
        q, k, v = _dense(q), _dense(k), _dense(v)
        if not masks.is_contiguous():
            masks = masks.contiguous()
        if out is None:
            out = dst = q.new_empty(shape)
        elif out.shape != shape or out.dtype != dtype or out.device != dev:
            raise ValueError(f"{what}: out must be {tuple(shape)} {dtype} on {dev}")
        else:
            dst = _dense(out)  # a copy holds the rows of no sequence, too
        nbytes = calls.pkv_tree_attention_workspace_bytes(
            n, max_nodes, hq, hkv, d, max_blk, bs, max_ctx, part_tokens, code)
        # this call's own memory, from the allocator's pool of the current stream
        # (or of the graph being captured): nothing is shared between calls
        ws = torch.empty(nbytes, dtype=torch.uint8, device=dev) if nbytes else None
        rc = calls.pkv_paged_tree_attention(
            dst.data_ptr(), None if lse is None else lse.data_ptr(), q.data_ptr(), k.data_ptr(),
            v.data_ptr(), k_pool.data_ptr(), v_pool.data_ptr(), nb, bs,
            table.data_ptr() if max_blk else None, max_blk, ctx.data_ptr(),
            qsl.data_ptr(), masks.data_ptr(), masks.shape[1], n, T, max_nodes,
            max_ctx, hq, hkv, d, float(scale) if scale is not None and scale > 0 else 0.0,
            part_tokens, code, None if ws is None else ws.data_ptr(), nbytes,
            None if status is None else _status_ptr(status, dev, what), _native.stream_ptr(dev))
        if rc:
            _native.check(rc, what)
        if dst is not out:
            out.copy_(dst)
    finally:
        _native.restore(previous)
    return out


def tree_accept(picks: torch.Tensor, tokens: torch.Tensor, meta: TreeMeta, max_depth: int,
                status: Optional[torch.Tensor] = None) -> TreeAccept:
    """The nodes of each tree that the model confirms: from node 0 down to the
    lowest-numbered child whose token is the pick at its parent, at most max_depth
    nodes. picks, tokens int64 [T]: the token chosen after each node (argmax, or a
    draw: accepting exactly the drafts a draw hits leaves the model's
    distribution as it is), and each node's own."""
    what = "tree_accept"
    _native.require_device(picks, tokens, what=what)
    parents, qsl, T, n = meta.parents, meta.query_start_loc, meta.num_tokens, meta.num_seqs
    dev = parents.device
    qsl = _int_tensor(qsl, torch.int32, n + 1, dev, "query_start_loc", what)
    parents = _int_tensor(parents, torch.int32, T, dev, "parents", what)
    picks = _int_tensor(picks, torch.int64, T, dev, "picks", what)
    tokens = _int_tensor(tokens, torch.int64, T, dev, "tokens", what)
    max_depth = int(max_depth)
    if max_depth < 1:
        raise ValueError(f"{what}: max_depth must be at least 1")
    previous = _native.make_current(dev)
    try:
        lens = qsl.new_empty(n)
        path = qsl.new_empty((n, max_depth))
        out = picks.new_empty((n, max_depth))
        rc = _native.calls().pkv_tree_accept(
            lens.data_ptr(), path.data_ptr(), out.data_ptr(), picks.data_ptr(),
            tokens.data_ptr(), parents.data_ptr(), qsl.data_ptr(), n, T, max_depth,
            None if status is None else _status_ptr(status, dev, what), _native.stream_ptr(dev))
    finally:
        _native.restore(previous)
    if rc:
        _native.check(rc, what)
    return TreeAccept(lens, path, out)
