"""Low-rank adapters of many requests beside the shared projections.

Row t of a step may name an adapter i; a projection's output of that row is then
y = W x + scale_i B_i (A_i x). AdapterWeights holds the A and B of several adapters
for one (fused) projection, build_adapter_plan groups a step's rows by adapter once
for all layers, and adapter_add / adapter_swiglu take the projection's output and
finish it (csrc/adapters.hip):

  weights = AdapterWeights(d_model, (hq * d, hkv * d, hkv * d), num_adapters=16, max_rank=16)
  weights.load(3, [(A_q, B_q), (A_k, B_k), None], scale=alpha / r)
  plan = build_adapter_plan(ids, 16)                  # int32 [T], -1: no adapter
  qkv = adapter_add(linear(x, w_qkv), x, weights, plan)

AdapterSet holds the weights of every projection of a PagedTransformer; its
forward_batch, forward_step and generate_batched, and the Scheduler's requests, take
adapters by index. No counterpart in the reference. Nothing here synchronises the
host, and every call's scratch is its own.
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import Optional

import torch

from . import _native
from .paged_meta import _status_ptr

__all__ = ["AdapterWeights", "AdapterPlan", "AdapterSet", "StepAdapters", "build_adapter_plan",
           "adapter_add", "adapter_swiglu", "step_adapters"]

MAX_ADAPTERS = 1000
MAX_RANK = 128
_I32 = torch.int32
# Rows a tile: 16 leaves no empty matrix rows where most adapters have a few rows;
# 64 reads an adapter's weights a quarter as often where a step holds prompts. us of both
# products by tiles of 16 / 64 rows (q/k/v of 4096 + 256 features, k 4096, rank 16, bf16):
#   rows                  256        768        1024       1536       2048       4096
#   one adapter         9.2/16.6  14.0/18.9  17.8/20.3  20.6/23.2  24.5/25.2  39.6/32.8
#   24, rows mixed     10.8/13.0  16.7/19.5  19.1/22.1  23.5/25.0  27.3/27.5  41.6/37.0
#   256, rows mixed    30.0/37.0  38.6/40.6  40.4/42.5  47.4/44.5  51.8/47.4  70.7/58.5
# and alike for rank 64 and for the gate (512 rows of one adapter 13.3/19.3, 1024 20.3/23.2, 4096
# 51.6/42.4). The border is early for few adapters: from 1024 to some 2000 rows tiles of 16
# would take up to 3 us less.
TILE_ROWS_FEW, TILE_ROWS_MANY, TILE_MANY_FROM = 16, 64, 1024


class AdapterWeights:
    """A and B of num_adapters adapters beside a projection of in_features features
    to the parts out_features (one, or those of a fused projection, at most 4), of at
    most max_rank ranks a part. a [num_adapters, parts * rank, in_features rounded up
    to 32], b [num_adapters, out_features each rounded up to 64, rank] and scales (float32)
    are what the kernels read, rank being max_rank rounded up to a multiple of 8, a and b in
    the order of their lanes (unpack() gives them in plain order); unused ranks are 0, and
    so is an adapter that was not loaded."""

    def __init__(self, in_features: int, out_features, num_adapters: int, max_rank: int,
                 dtype: torch.dtype = torch.float32, device="cuda"):
        outs = (out_features,) if isinstance(out_features, int) else tuple(out_features)
        _native.dtype_code(dtype)
        if in_features < 1 or not 1 <= len(outs) <= 4 or min(outs) < 1:
            raise ValueError("AdapterWeights: needs features in and 1 to 4 parts of features out")
        if not 1 <= num_adapters <= MAX_ADAPTERS or not 1 <= max_rank <= MAX_RANK:
            raise ValueError(f"AdapterWeights: 1 to {MAX_ADAPTERS} adapters of rank 1 to {MAX_RANK}")
        self.in_features, self.out_features = int(in_features), outs
        self.num_adapters, self.rank, self.dtype = int(num_adapters), -(-max_rank // 8) * 8, dtype
        self.a = torch.zeros((num_adapters, len(outs) * self.rank, -(-in_features // 32) * 32),
                             dtype=dtype, device=device)
        self.b = torch.zeros((num_adapters, sum(-(-n // 64) * 64 for n in outs), self.rank),
                             dtype=dtype, device=device)
        self.scales = torch.zeros(num_adapters, dtype=torch.float32, device=device)
        self.device = self.a.device
        # what every call hands on
        self._place, self._features, self._parts = self.a.get_device(), sum(outs), len(outs)
        self._a_stride, self._ns = self.a.shape[2], outs + (0,) * (4 - len(outs))

    def _index(self, index):
        if not 0 <= index < self.num_adapters:
            raise IndexError(f"adapter {index} of {self.num_adapters}")
        return index

    def _check_parts(self, index, parts):
        self._index(index)
        if len(parts) != len(self.out_features):
            raise ValueError(f"AdapterWeights.load: {len(self.out_features)} parts, "
                             f"got {len(parts)}")
        for n, pair in zip(self.out_features, parts):
            if pair is None:
                continue
            a, b = pair
            r = a.shape[0] if a.dim() == 2 else -1
            if (not 0 <= r <= self.rank or a.shape != (r, self.in_features)
                    or b.shape != (n, r)):
                raise ValueError(
                    f"AdapterWeights.load: A {tuple(a.shape)} and B {tuple(b.shape)} are not "
                    f"[r, {self.in_features}] and [{n}, r] with r up to {self.rank}")

    @torch.no_grad()
    def load(self, index: int, parts, scale: float = 1.0) -> None:
        """Puts an adapter in place `index`: per part (A [r, in_features], B
        [out_features, r]) with r up to the rank, or None for a part without one."""
        self._check_parts(index, parts)
        for (dst_a, dst_b), n, pair in zip(self._parts_of(index), self.out_features, parts):
            r = 0 if pair is None else pair[0].shape[0]
            if r == 0:
                for d in (*dst_a, dst_b):
                    d.zero_()
                continue
            a, b = self._whole(pair[0], self.rank, self.a.shape[2]), self._whole(
                pair[1], -(-n // 64) * 64, self.rank)
            at = 0
            for d in dst_a:
                d.copy_(a[at:at + d.shape[0] * d.shape[1]].view(d.shape))
                at += d.shape[0] * d.shape[1]
            dst_b.copy_(b.view(dst_b.shape))
        self.scales[index] = float(scale)

    def _whole(self, t, rows, cols):
        """t on the device, in the type and with zeros up to [rows, cols]."""
        if t.shape == (rows, cols):
            return t.to(self.device, self.dtype).contiguous()
        out = torch.zeros((rows, cols), dtype=self.dtype, device=self.device)
        out[:t.shape[0], :t.shape[1]] = t
        return out

    def _parts_of(self, index):
        """Views of each part's A, ranks in blocks of 16 and then of 8 ([blocks, ranks, steps,
        4, 8]), and B ([blocks of 64 features, 2, 4, 2, 4, 8s of ranks, 8]), whose elements in
        order are the rows in order."""
        R, steps, at = self.rank, self.a.shape[2] // 32, 0
        for s, n in enumerate(self.out_features):
            a, full = self.a[index, s * R:(s + 1) * R], R // 16 * 16
            views = []
            for rows, of in ((a[:full], 16), (a[full:], 8)):
                if len(rows):
                    views.append(rows.view(-1, steps, 4, of, 8).permute(0, 3, 1, 2, 4))
            wide = -(-n // 64) * 64
            b = self.b[index, at:at + wide].view(-1, R // 8, 2, 2, 4, 4, 8)
            at += wide
            yield views, b.permute(0, 2, 4, 3, 5, 1, 6)

    def unpack(self, index: int):
        """(A [parts * rank, in_features], B [sum(out_features), rank]) of an adapter, copies
        in plain order."""
        a_rows, b_rows = [], []
        for (views, b), n in zip(self._parts_of(self._index(index)), self.out_features):
            a_rows += [v.reshape(-1, self.a.shape[2])[:, :self.in_features] for v in views]
            b_rows.append(b.reshape(-1, self.rank)[:n])
        return torch.cat(a_rows), torch.cat(b_rows)

    @torch.no_grad()
    def clear(self, index: int) -> None:
        """Takes adapter `index` out: rows that name it get the projection alone."""
        index = self._index(index)
        self.a[index].zero_()
        self.b[index].zero_()
        self.scales[index] = 0.0


@dataclass(frozen=True)
class AdapterPlan:
    order: torch.Tensor   # int32 [T] rows sorted by adapter, those without one last
    starts: torch.Tensor  # int32 [num_adapters + 2] first place of each adapter's rows
    tiles: torch.Tensor   # int32 [max_tiles, 4] adapter or -1, first place, rows, 0
    rows: torch.Tensor    # int32 [max_tiles, tile_rows] the tiles' rows
    num_tokens: int
    num_adapters: int
    tile_rows: int


def build_adapter_plan(ids: torch.Tensor, num_adapters: int,
                       status: Optional[torch.Tensor] = None) -> AdapterPlan:
    """Groups the rows of a step by adapter: ids int32 [T], -1 for a row without
    one. Any other id outside [0, num_adapters) counts as none and is reported in
    `status` (int32 [1], zeroed by the caller, read with raise_step_status)."""
    what = "build_adapter_plan"
    _native.require_device(ids, what=what)
    if ids.dtype != _I32 or ids.dim() != 1:
        raise ValueError(f"{what}: ids must be int32 [T]")
    n = int(num_adapters)
    if not 0 <= n <= MAX_ADAPTERS:
        raise ValueError(f"{what}: at most {MAX_ADAPTERS} adapters")
    T, dev = ids.shape[0], ids.device
    rows = TILE_ROWS_MANY if T >= TILE_MANY_FROM else TILE_ROWS_FEW
    max_tiles = T // rows + min(n + 1, T)
    previous = _native.make_current(dev)
    try:
        if not ids.is_contiguous():
            ids = ids.contiguous()
        # one allocation; the tiles lead, their rows are 16 bytes
        sizes = (4 * max_tiles, rows * max_tiles, T, n + 2)
        tiles, places, order, starts = ids.new_empty(sum(sizes)).split_with_sizes(sizes)
        rc = _native.calls().pkv_adapter_plan(
            order.data_ptr(), starts.data_ptr(), tiles.data_ptr(), places.data_ptr(), max_tiles,
            ids.data_ptr(), T, n, rows, None if status is None else _status_ptr(status, dev, what),
            _native.stream_ptr(dev))
    finally:
        _native.restore(previous)
    if rc:
        _native.check(rc, what)
    return AdapterPlan(order, starts, tiles.view(max_tiles, 4), places.view(max_tiles, rows), T, n,
                       rows)


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two 2-D tensors with unit column stride share memory."""
    if a.numel() == 0 or b.numel() == 0:
        return False
    es = a.element_size()
    pa, pb = a.data_ptr(), b.data_ptr()
    wa, wb = a.shape[1] * es, b.shape[1] * es
    if (pa + (a.shape[0] - 1) * a.stride(0) * es + wa <= pb
            or pb + (b.shape[0] - 1) * b.stride(0) * es + wb <= pa):
        return False
    if a.stride(0) == b.stride(0):  # columns of one buffer
        pitch = a.stride(0) * es
        off = (pa - pb) % pitch
        return not (off >= wb and off + wa <= pitch)
    return True


def _rows(t: torch.Tensor):
    """A 2-D tensor with unit column stride and rows that do not overlap, t where it is
    one, and its row stride."""
    n, width = t.shape
    stride, one = t.stride()
    if one != 1 or (n > 1 and stride < width):
        return t.contiguous(), width
    return t, stride if n > 1 else width


def _apply(base, x, weights, plan, out, written, epilogue, what):
    a, dev, dtype, T = weights.a, weights.device, weights.dtype, plan.num_tokens
    place, tiles = weights._place, plan.tiles
    if not (place >= 0 and base.get_device() == place and x.get_device() == place
            and tiles.get_device() == place):
        _native.require_device(base, x, tiles, a, what=what)
        raise RuntimeError(f"{what}: base, x, the weights and the plan must share a device")
    if base.dtype != dtype or x.dtype != dtype:
        raise TypeError(f"{what}: base and x must be {dtype}, as the weights are")
    if (base.requires_grad or x.requires_grad) and torch.is_grad_enabled():
        raise NotImplementedError(
            f"{what} is forward-only (inference); run it under torch.no_grad()")
    n, k = weights._features, weights.in_features
    if base.shape != (T, n) or x.shape != (T, k):
        raise ValueError(f"{what}: base must be [{T}, {n}] and x [{T}, {k}] for this plan and "
                         f"these weights (got {tuple(base.shape)}, {tuple(x.shape)})")
    if plan.num_adapters != weights.num_adapters:
        raise ValueError(f"{what}: a plan of {plan.num_adapters} adapters, weights of "
                         f"{weights.num_adapters}")
    in_place, given = out is base, out is not None
    (base, base_stride), (x, x_stride) = _rows(base), _rows(x)
    calls, max_tiles = _native.calls(), tiles.shape[0]
    previous = _native.make_current(dev)
    try:
        if out is None:
            out, out_stride = base.new_empty((T, written)), written
        elif in_place and out is base and written == n:  # and not a copy of its rows
            out_stride = base_stride
            if _overlap(out, x):
                raise ValueError(f"{what}: out shares memory with base or x")
        else:
            if out.shape != (T, written) or out.dtype != dtype or out.get_device() != place:
                raise ValueError(f"{what}: out must be [{T}, {written}] {dtype} on {dev}")
            dst, out_stride = _rows(out)
            if dst is not out:
                raise ValueError(f"{what}: out needs unit column stride and rows of its own")
            if out.requires_grad and torch.is_grad_enabled():
                raise NotImplementedError(f"{what} is forward-only (inference)")
            same = (out.data_ptr() == base.data_ptr() and written == n
                    and out_stride == base_stride)
            if (not same and _overlap(out, base)) or _overlap(out, x):
                raise ValueError(f"{what}: out shares memory with base or x")
        nbytes = calls.pkv_adapter_workspace_bytes(T, max_tiles, plan.tile_rows, k, weights.rank,
                                                   weights._parts)
        # this call's own scratch, from the allocator's pool of the current stream (or of
        # the graph being captured): nothing is shared between calls
        ws = base.new_empty(nbytes, dtype=torch.uint8)
        rc = calls.pkv_adapter_apply(
            out.data_ptr(), out_stride, base.data_ptr(), base_stride, x.data_ptr(), x_stride,
            a.data_ptr(), weights._a_stride, weights.b.data_ptr(), weights.scales.data_ptr(),
            tiles.data_ptr(), plan.rows.data_ptr(), max_tiles, plan.tile_rows, T,
            weights.num_adapters, k, weights.rank, weights._parts, *weights._ns, epilogue,
            _native.DTYPE_CODES[dtype], ws.data_ptr(), nbytes, _native.stream_ptr(dev))
        if rc:
            _native.check(rc, what)
        if given:  # a graph that saved out finds it changed
            torch.autograd.graph.increment_version(out)
    finally:
        _native.restore(previous)
    return out


def adapter_add(base: torch.Tensor, x: torch.Tensor, weights: AdapterWeights, plan: AdapterPlan,
                out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """base [T, sum(out_features)] plus each row's adapter's product with x [T,
    in_features]; float32, float16 or bfloat16, sums in fp32, rounded once (between its
    two products a 16-bit type's A x is the sum of two values of the type). Rows without
    an adapter are base's. out: where to write, base itself (in place) or memory of no
    operand."""
    return _apply(base, x, weights, plan, out, weights._features, _native.EPILOGUE_NONE,
                  "adapter_add")


def adapter_swiglu(base: torch.Tensor, x: torch.Tensor, weights: AdapterWeights,
                   plan: AdapterPlan, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """silu(gate) * up [T, H] of adapter_add(base, ...) = [gate, up], base [T, 2 H],
    without rounding in between. Rows without an adapter are silu_mul of base."""
    outs = weights.out_features
    if len(outs) != 2 or outs[0] != outs[1]:
        raise ValueError("adapter_swiglu: the weights need two parts of one size (gate, up)")
    return _apply(base, x, weights, plan, out, outs[0], _native.EPILOGUE_SWIGLU, "adapter_swiglu")


# The adapted projections of a block: its module, the parts of its fused projection, and
# what the parts read and write, as attributes of the attention or the MLP
_PROJECTIONS = {"qkv": ("attn", ("q_proj", "k_proj", "v_proj")), "out": ("attn", ("out",)),
                "gate_up": ("mlp", ("gate_proj", "up_proj")), "down": ("mlp", ("down_proj",))}


class AdapterSet:
    """Adapters of a PagedTransformer, by index: layers[i] holds the AdapterWeights of
    layer i's fused projections ("qkv", "out", "gate_up", "down"), of those in
    `projections`."""

    def __init__(self, model, num_adapters: int, max_rank: int, projections=tuple(_PROJECTIONS)):
        unknown = set(projections) - set(_PROJECTIONS)
        if unknown:
            raise ValueError(f"AdapterSet: no projection {sorted(unknown)[0]!r}")
        self.num_adapters = int(num_adapters)
        self.layers = []
        for layer in model.layers:
            ws = {}
            for name in projections:
                owner, parts = _PROJECTIONS[name]
                lins = [getattr(getattr(layer, owner), p) for p in parts]
                ws[name] = AdapterWeights(lins[0].in_features, [m.out_features for m in lins],
                                          num_adapters, max_rank, dtype=lins[0].weight.dtype,
                                          device=lins[0].weight.device)
            self.layers.append(ws)

    def load(self, index: int, state: dict, scale: float = 1.0) -> None:
        """Puts an adapter in place `index`. state: for each adapted nn.Linear of the
        model, by its name ("layers.0.attn.q_proj"), "<name>.lora_A.weight" [r,
        in_features] and "<name>.lora_B.weight" [out_features, r]; scale is usually
        alpha / r. Linears that are not named have no adapter."""
        left = set(state)
        found = []
        for i, ws in enumerate(self.layers):
            for name, w in ws.items():
                owner, parts = _PROJECTIONS[name]
                pairs = []
                for p in parts:
                    keys = [f"layers.{i}.{owner}.{p}.lora_{m}.weight" for m in "AB"]
                    here = [k for k in keys if k in state]
                    if len(here) == 1:
                        raise ValueError(f"AdapterSet.load: {here[0]} comes without the other")
                    pairs.append(tuple(state[k] for k in keys) if here else None)
                    left -= set(here)
                found.append((w, pairs))
        if left:
            raise ValueError(f"AdapterSet.load: {sorted(left)[0]!r} is no projection of this set")
        for w, pairs in found:  # all before the first is changed
            w._check_parts(index, pairs)
        for w, pairs in found:
            w.load(index, pairs, scale)

    def clear(self, index: int) -> None:
        for ws in self.layers:
            for w in ws.values():
                w.clear(index)


@dataclass(frozen=True)
class StepAdapters:
    """The adapters of one step's rows."""
    weights: AdapterSet
    plan: AdapterPlan


def step_adapters(weights: AdapterSet, ids, query_start_loc, device) -> Optional[StepAdapters]:
    """The adapters of a ragged step from one id a sequence (-1: none) and the host's
    query_start_loc; None where no sequence has one."""
    ids = [int(i) for i in ids]
    if len(ids) != len(query_start_loc) - 1:
        raise ValueError(f"{len(ids)} adapter ids for {len(query_start_loc) - 1} sequences")
    for i in ids:
        if not -1 <= i < weights.num_adapters:
            raise ValueError(f"adapter {i} of {weights.num_adapters}")
    if all(i < 0 for i in ids):
        return None
    rows = [i for i, a, b in zip(ids, query_start_loc, query_start_loc[1:]) for _ in range(a, b)]
    return StepAdapters(weights, build_adapter_plan(
        torch.tensor(rows, dtype=_I32, device=device), weights.num_adapters))
