"""Device-resident metadata of one paged step.

The reference rebuilds block tables, slot mappings and kv lengths per layer
and per sequence with host round trips (serving/paged_mqa.py:87-96,
serving/fake_paged_attn.py:52-100). Here the ragged host lists are validated
and packed once per step into a single int32 buffer, copied to the device in
one transfer, and reused by every layer's append and attention launch.

Where a step's lengths are known on the device only (tokens accepted by a
verification, serving.tree_decode), build_batch_meta makes the same metadata
there, from a batch's DeviceTables: blocks taken from a free list, table rows,
positions and slots in one kernel, without a host round trip.
"""
from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from . import _native


@dataclass
class PagedBatchMeta:
    block_tables: torch.Tensor     # int32 [N, max_blocks], zero padded
    seq_lens: torch.Tensor         # int32 [N]  kv length after this step
    query_start_loc: torch.Tensor  # int32 [N+1]
    start_pos: torch.Tensor        # int32 [N]  position of each sequence's first new token
    positions: torch.Tensor        # int32 [T]  absolute position of every new token
    num_seqs: int
    num_tokens: int
    max_blocks: int
    max_q_len: int
    max_kv_len: int
    block_size: int
    # seq_lens, start_pos and positions as one contiguous view (pack_batch_meta
    # lays them out back to back), so a decode step advances them with one add
    step_view: torch.Tensor | None = None
    # int64 [T], build_batch_meta only: each token's pool slot (KVPool.write's
    # slot_mapping), NO_SLOT behind the last token
    slot_mapping: torch.Tensor | None = None
    # False (build_batch_meta): num_tokens and max_q_len are bounds on lengths that
    # only the device knows; there may be rows of no sequence and sequences of no token
    exact: bool = True

    @property
    def is_decode(self) -> bool:
        """One token a sequence: token row s is sequence s's."""
        return self.exact and self.max_q_len == 1 and self.num_tokens == self.num_seqs

    def advance_(self) -> None:
        """Every sequence one token further, on the device: seq_lens,
        start_pos and positions + 1 (one kernel when they share step_view).
        Where the lengths are bounds (exact False) only sequences that have tokens,
        and their rows. slot_mapping becomes NO_SLOT throughout, as the slots of later
        tokens are another build_batch_meta's to give."""
        if self.slot_mapping is not None:
            self.slot_mapping.fill_(NO_SLOT)
        if not self.exact:
            some = (self.query_start_loc[1:] > self.query_start_loc[:-1]).int()
            self.seq_lens.add_(some)
            self.start_pos.add_(some)
            rows = torch.arange(self.num_tokens, dtype=torch.int32,
                                device=self.positions.device)
            self.positions.add_((rows < self.query_start_loc[-1]).int())
            return
        v = self.step_view
        n, t = self.num_seqs, self.num_tokens
        if (v is not None and v.numel() == 2 * n + t and v.dtype == torch.int32
                and self.seq_lens.data_ptr() == v.data_ptr()
                and self.start_pos.data_ptr() == v.data_ptr() + 4 * n
                and self.positions.data_ptr() == v.data_ptr() + 8 * n):
            v.add_(1)
            return
        self.positions.add_(1)
        self.start_pos.add_(1)
        self.seq_lens.add_(1)


def _as_list(x):
    if isinstance(x, torch.Tensor):
        return x.tolist()
    return list(x)


def pack_batch_meta(block_tables, query_start_loc, positions, T: int, device,
                    block_size: int, check_append: bool = True) -> PagedBatchMeta:
    """Validate and pack one step's ragged metadata.

    Checks, with the reference's exception types and messages:
      - query_start_loc / positions lengths (fake_paged_attn.py:60-66, ValueError)
      - kv_len = positions[last] + 1 fits the table (fake_paged_attn.py:86-92, ValueError)
      - with check_append: the new tokens' slots fit the table and avoid
        reserved block 0 (kv_pool.py:41-42, :52-53, AssertionError)
    """
    tables = [_as_list(bt) for bt in block_tables]
    qsl = [int(x) for x in _as_list(query_start_loc)]
    pos = [int(x) for x in _as_list(positions)]
    n = len(tables)
    if len(qsl) != n + 1:
        raise ValueError("query_start_loc must have length num_seqs + 1")
    if qsl[0] != 0 or qsl[-1] != T:
        raise ValueError("query_start_loc must start at 0 and end at T")
    if len(pos) != T:
        raise ValueError(f"positions must have length T ({T})")

    max_blocks = max((len(bt) for bt in tables), default=0)
    seq_lens = np.zeros(n, dtype=np.int32)
    start_pos = np.zeros(n, dtype=np.int32)
    max_q_len = 0
    for i, bt in enumerate(tables):
        s0, s1 = qsl[i], qsl[i + 1]
        q_len = s1 - s0
        max_q_len = max(max_q_len, q_len)
        if q_len <= 0:
            continue
        kv_len = pos[s1 - 1] + 1
        cap = len(bt) * block_size
        if kv_len > cap:
            raise ValueError(f"seq {i}: kv_len {kv_len} exceeds {len(bt)} * blocksize ({cap})")
        seq_lens[i] = kv_len
        start = pos[s0]
        start_pos[i] = start
        if check_append:
            assert start + q_len <= cap, \
                f"block table too short: need {start + q_len} slots, table gives {cap}"
            first_blk, last_blk = start // block_size, (start + q_len - 1) // block_size
            if 0 in bt[first_blk:last_blk + 1]:
                raise AssertionError("slot mapping touches block 0, which is reserved")

    # one int32 host buffer -> one H2D copy; device views carved out of it
    # (seq_lens, start_pos, positions back to back: one add advances them)
    sizes = [n * max_blocks, n + 1, n, n, T]
    buf = np.zeros(sum(sizes), dtype=np.int32)
    off = 0
    if max_blocks:
        tab = buf[:n * max_blocks].reshape(n, max_blocks)
        for i, bt in enumerate(tables):
            tab[i, :len(bt)] = bt
    off += sizes[0]
    buf[off:off + n + 1] = qsl
    off += n + 1
    buf[off:off + n] = seq_lens
    off += n
    buf[off:off + n] = start_pos
    off += n
    buf[off:off + T] = pos
    host = torch.from_numpy(buf)
    if torch.device(device).type == "cuda":
        host = host.pin_memory()
    dev = host.to(device, non_blocking=True)
    views = torch.split(dev, sizes)
    step0 = sizes[0] + sizes[1]
    return PagedBatchMeta(
        block_tables=views[0].view(n, max_blocks),
        seq_lens=views[2],
        query_start_loc=views[1],
        start_pos=views[3],
        positions=views[4],
        step_view=dev[step0:step0 + 2 * n + T],
        num_seqs=n,
        num_tokens=T,
        max_blocks=max_blocks,
        max_q_len=max_q_len,
        max_kv_len=int(seq_lens.max()) if n else 0,
        block_size=block_size,
    )


NO_SLOT = -(1 << 63)  # a slot that an append skips


@dataclass(frozen=True)
class DeviceTables:
    """Block tables of a running batch on the device, and the blocks it may
    still take: contiguous int32 tensors of one device, checked when the object
    is made (its fields are not assigned again)."""
    block_tables: torch.Tensor  # [N, max_blocks]
    blocks_held: torch.Tensor   # [N] blocks each row holds
    ctx_lens: torch.Tensor      # [N] tokens whose K/V are in the pool
    free_blocks: torch.Tensor   # [F] block ids, in the order they are handed out
    free_cursor: torch.Tensor   # [1] the next of them
    block_size: int
    num_blocks: int             # the pool's

    def __post_init__(self):
        bt = self.block_tables
        if bt.dim() != 2:
            raise ValueError("DeviceTables: block_tables must be [N, max_blocks]")
        n = bt.shape[0]
        for name, numel in (("block_tables", bt.numel()), ("blocks_held", n), ("ctx_lens", n),
                            ("free_blocks", self.free_blocks.numel()), ("free_cursor", 1)):
            t = getattr(self, name)
            if t.dtype != torch.int32 or not t.is_contiguous():
                raise ValueError(f"DeviceTables: {name} must be a contiguous int32 tensor")
            if t.device != bt.device:
                raise RuntimeError(f"DeviceTables: {name} on {t.device}, block_tables on {bt.device}")
            if t.numel() != numel:
                raise ValueError(f"DeviceTables: {name} has {t.numel()} elements, expected {numel}")

    @classmethod
    def from_host(cls, tables, ctx_lens, free_blocks, max_blocks: int, block_size: int,
                  num_blocks: int, device) -> "DeviceTables":
        """From the host's block tables (lists of ids), lengths and the ids set
        aside for growth (BlockAllocator.allocate_n), rows of max_blocks."""
        n = len(tables)
        if len(ctx_lens) != n:
            raise ValueError(f"{n} block tables but {len(ctx_lens)} context lengths")
        buf = np.zeros((n, max_blocks), dtype=np.int32)
        for i, (row, length) in enumerate(zip(tables, ctx_lens)):
            if len(row) > max_blocks:
                raise ValueError(f"seq {i}: {len(row)} blocks, rows hold {max_blocks}")
            if not 0 <= length <= len(row) * block_size:
                raise ValueError(f"seq {i}: {length} tokens in {len(row)} blocks of {block_size}")
            buf[i, :len(row)] = row
        i32 = lambda x: torch.tensor(list(x), dtype=torch.int32, device=device)  # noqa: E731
        return cls(block_tables=torch.from_numpy(buf).to(device),
                   blocks_held=i32(len(t) for t in tables), ctx_lens=i32(ctx_lens),
                   free_blocks=i32(free_blocks), free_cursor=i32([0]), block_size=block_size,
                   num_blocks=num_blocks)

    def _after(self, blocks_held, ctx_lens, free_cursor) -> "DeviceTables":
        """The same tables in a later state (tensors of the checked kind)."""
        new = object.__new__(DeviceTables)
        new.__dict__.update(self.__dict__, blocks_held=blocks_held, ctx_lens=ctx_lens,
                            free_cursor=free_cursor)
        return new


def raise_step_status(status: torch.Tensor, what: str) -> None:
    """Reads the status word of the calls that make and use a step's metadata
    (this waits for them) and raises what the host's checks raise."""
    bits = int(status.item())
    if bits & _native.PKV_STATUS_OUT_OF_BLOCKS:
        raise RuntimeError(f"{what}: out of KV blocks")
    if bits & _native.PKV_STATUS_SHORT_TABLE:
        raise ValueError(f"{what}: a sequence exceeds its block table row")
    if bits & _native.PKV_STATUS_BAD_QLOC:
        raise ValueError(f"{what}: a length or query range is outside its bounds")
    if bits & _native.PKV_STATUS_BAD_PARENT:
        raise ValueError(f"{what}: a node's parent is neither -1 nor an earlier node")
    if bits & _native.PKV_STATUS_BAD_BLOCK:
        raise AssertionError(f"{what}: a block id is block 0 or outside the pool")
    if bits & _native.PKV_STATUS_BAD_TOKEN:
        raise ValueError(f"{what}: a token or bias id is outside the vocabulary")
    if bits & _native.PKV_STATUS_BAD_CONTROL:
        raise ValueError(f"{what}: an adapter, length, mask or sampling parameter is outside "
                         "its range")
    if bits & _native.PKV_STATUS_NONFINITE:
        raise ValueError(f"{what}: logits contain NaN or infinity")
    if bits & _native.PKV_STATUS_BAD_DISTRIBUTION:
        raise ValueError(f"{what}: a row has no token left to draw")
    if bits:
        raise RuntimeError(f"{what}: status {bits}")


def _status_ptr(status, device, what):
    if status.dtype != torch.int32 or status.numel() != 1 or status.device != device:
        raise ValueError(f"{what}: status must be one int32 on {device}")
    return status.data_ptr()


def build_batch_meta(tables: DeviceTables, q_lens: torch.Tensor, num_tokens: int, max_q_len: int,
                     max_kv_len: int = 0, status: torch.Tensor | None = None):
    """A step's metadata from lengths on the device: sequence i gets q_lens[i]
    (int32 [N]) more tokens, the blocks it lacks come from the free list in
    sequence order and are written to tables.block_tables. num_tokens bounds the
    sum of q_lens and is T of the result, whose rows behind the last token have
    position 0 and slot NO_SLOT; max_q_len bounds each length, max_kv_len (0: the
    table's capacity) the contexts after the step.

    Returns (PagedBatchMeta with slot_mapping, DeviceTables after the step).
    Values as pack_batch_meta gives them, and like its result the step can go to
    KVPool.write_from_table, paged_attention_append_meta and
    PagedTransformer.forward_step, though not as a decode batch (is_decode): its
    lengths are not the host's to know (a caller who knows that they are the bounds,
    one token for every sequence, says so by dataclasses.replace(meta, exact=True)); the given tables' other tensors are not
    changed, so a step whose result is dropped can be taken again (the table itself
    is one for all states: its rows are those of the last step taken, zeros behind
    the blocks they hold). With too few
    free blocks, a row past max_blocks or a length out of bounds nothing is taken
    (all or nothing) and the metadata names no slot or position that an append
    writes to, so the calls launched with it leave the pool as it is; `status` (int32
    [1], zeroed by the caller, read with raise_step_status) reports it. No host
    synchronisation."""
    bt = tables.block_tables
    _native.require_device(bt, what="build_batch_meta")
    dev = bt.device
    n, max_blocks = bt.shape
    if q_lens.dtype != torch.int32 or q_lens.device != dev or q_lens.numel() != n:
        raise ValueError(f"build_batch_meta: q_lens must be int32 [{n}] on {dev}")
    T, max_q_len = int(num_tokens), int(max_q_len)
    if T < 0 or max_q_len < 0:
        raise ValueError("build_batch_meta: num_tokens and max_q_len must be >= 0")
    q = q_lens if q_lens.is_contiguous() else q_lens.contiguous()
    bs = tables.block_size
    free = tables.free_blocks
    previous = _native.make_current(dev)
    try:
        i32 = bt.new_empty(5 * n + 2 + T)
        slots = torch.empty(T, dtype=torch.int64, device=dev)
        at = i32.data_ptr()
        held, ctx = at + 4 * (3 * n + 1 + T), at + 4 * (4 * n + 1 + T)
        rc = _native.calls().pkv_build_step(
            bt.data_ptr(), max_blocks, tables.blocks_held.data_ptr(), tables.ctx_lens.data_ptr(),
            q.data_ptr(), n, free.data_ptr(), free.numel(), tables.free_cursor.data_ptr(), bs,
            tables.num_blocks, T, max_q_len, held, ctx, ctx + 4 * n, at + 4 * (2 * n + T), at,
            at + 4 * n, at + 8 * n, slots.data_ptr(),
            None if status is None else _status_ptr(status, dev, "build_batch_meta"),
            _native.stream_ptr(dev))
    finally:
        _native.restore(previous)
    if rc:
        _native.check(rc, "build_batch_meta")
    seq_lens, start_pos, positions, qsl, held, ctx, cursor = i32.split_with_sizes(
        (n, n, T, n + 1, n, n, 1))
    if max_kv_len <= 0:
        max_kv_len = max_blocks * bs
    meta = PagedBatchMeta(bt, seq_lens, qsl, start_pos, positions, n, T, max_blocks, max_q_len,
                          int(max_kv_len), bs, None, slots, False)
    return meta, tables._after(held, ctx, cursor)
