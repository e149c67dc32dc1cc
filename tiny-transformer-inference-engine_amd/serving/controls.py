"""What each request of a batch asks of its next token: penalties of tokens that are
there already, biases, a grammar's mask, and its own sampling parameters
(csrc/controls.hip). No counterpart in the reference, whose sample() takes one set of
parameters for all rows (sampling.py:94-137).

  logits = control_logits(logits, LogitControls(tokens=history, lens=lens, ...), out=logits)
  ids, logprobs = sample_each(logits, temperature, top_k, top_p, min_p)

Neither synchronises the host, so both can be captured in a HIP graph. RequestParams is
what a request of the Scheduler may ask for, draw_tokens its step over those requests.
"""
from __future__ import annotations

import math
from dataclasses import dataclass, field, fields
from typing import Optional, Protocol

import torch

from . import _native
from .adapters import _overlap, _rows
from .paged_meta import _status_ptr, raise_step_status

__all__ = ["LogitControls", "RequestParams", "Grammar", "TokenHistory", "control_logits",
           "sample_each", "pack_mask", "draw_tokens", "draw_rows"]

MAX_SAMPLE_VOCAB = 1 << 20


def _check(t, dtype, shape, name, what):
    if t.dtype != dtype or tuple(t.shape) != shape or not t.is_contiguous():
        raise ValueError(f"{what}: {name} must be contiguous {dtype} {list(shape)} "
                         f"(got {t.dtype} {list(t.shape)})")


@dataclass(frozen=True)
class LogitControls:
    """The controls of a batch's rows, on the device; each kind may be left out.

    tokens       int32 [rows, capacity] each row's tokens so far, the first lens[r]
    lens         int32 [rows]
    prompt_lens  int32 [rows] how many of them are the prompt (None: 0)
    repetition   float32 [rows] > 0: of a token that is there, x / r where x > 0, else x * r
    presence     float32 [rows] taken off a token that is there behind the prompt
    frequency    float32 [rows] the same, times how often it is there
    bias_ids, bias_values, bias_starts
                 int32 [n], float32 [n], int32 [rows + 1]: row r adds bias_values[e] to id
                 bias_ids[e], bias_starts[r] <= e < bias_starts[r + 1]; what is named
                 twice is added up
    masks        int32 [masks, ceil(vocab / 32)] bit id % 32 of word id / 32: id is allowed
    mask_rows    int32 [rows] the row's mask, -1 for none
    """
    tokens: Optional[torch.Tensor] = None
    lens: Optional[torch.Tensor] = None
    prompt_lens: Optional[torch.Tensor] = None
    repetition: Optional[torch.Tensor] = None
    presence: Optional[torch.Tensor] = None
    frequency: Optional[torch.Tensor] = None
    bias_ids: Optional[torch.Tensor] = None
    bias_values: Optional[torch.Tensor] = None
    bias_starts: Optional[torch.Tensor] = None
    masks: Optional[torch.Tensor] = None
    mask_rows: Optional[torch.Tensor] = None

    def __post_init__(self):
        what = "LogitControls"
        given = {f.name: getattr(self, f.name) for f in fields(self)
                 if getattr(self, f.name) is not None}
        if len({t.device for t in given.values()}) > 1:
            raise ValueError(f"{what}: the tensors must share a device")
        for group in (("tokens", "lens"), ("bias_ids", "bias_values", "bias_starts"),
                      ("masks", "mask_rows")):
            if len([n for n in group if n in given]) not in (0, len(group)):
                raise ValueError(f"{what}: {', '.join(group)} go together")
        history = [n for n in ("prompt_lens", "repetition", "presence", "frequency")
                   if n in given]
        if history and "tokens" not in given:
            raise ValueError(f"{what}: {history[0]} needs tokens and lens")
        rows = set()
        if "tokens" in given:
            t = self.tokens
            if t.dtype != torch.int32 or t.dim() != 2 or (t.numel() > 0 and (
                    t.stride(1) != 1 or (t.shape[0] > 1 and t.stride(0) < t.shape[1]))):
                raise ValueError(f"{what}: tokens must be int32 [rows, capacity] with unit "
                                 "column stride")
            rows.add(t.shape[0])
            _check(self.lens, torch.int32, (t.shape[0],), "lens", what)
            for n in history:
                _check(given[n], torch.int32 if n == "prompt_lens" else torch.float32,
                       (t.shape[0],), n, what)
        if "bias_ids" in given:
            n = self.bias_starts.numel() - 1
            _check(self.bias_starts, torch.int32, (n + 1,), "bias_starts", what)
            _check(self.bias_ids, torch.int32, (self.bias_ids.numel(),), "bias_ids", what)
            _check(self.bias_values, torch.float32, (self.bias_ids.numel(),), "bias_values", what)
            rows.add(n)
        if "masks" in given:
            if self.masks.dtype != torch.int32 or self.masks.dim() != 2 \
                    or not self.masks.is_contiguous():
                raise ValueError(f"{what}: masks must be contiguous int32 [masks, words]")
            _check(self.mask_rows, torch.int32, (self.mask_rows.numel(),), "mask_rows", what)
            rows.add(self.mask_rows.numel())
        if len(rows) > 1:
            raise ValueError(f"{what}: the tensors disagree on the rows ({sorted(rows)})")
        object.__setattr__(self, "_rows", rows.pop() if rows else None)
        # row stride and capacity, as the call hands them on
        t = self.tokens
        object.__setattr__(self, "_history", (0, 0) if t is None else (
            t.stride(0) if t.shape[0] > 1 else t.shape[1], t.shape[1]))
        object.__setattr__(self, "_device", next(iter(given.values())).device if given else None)


def control_logits(logits: torch.Tensor, controls: LogitControls,
                   out: Optional[torch.Tensor] = None,
                   status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """logits [rows, vocab] (float32, float16, bfloat16) with every row's penalties, then
    biases, then its mask (-infinity where an id is not allowed), in fp32 and rounded
    once; what finite operands carry past the range of fp32, or of the type at the end, is
    its largest value. out: where to write, logits itself or memory of no operand. `status` as in
    build_adapter_plan: ids outside the vocabulary, which are skipped, and lengths, offsets
    and mask rows outside their bounds. A mask may leave a row nothing: all -infinity."""
    what = "control_logits"
    _native.require_device(logits, what=what)
    code = _native.dtype_code(logits.dtype)
    if logits.dim() != 2:
        raise ValueError(f"{what}: expected [rows, vocab], got {tuple(logits.shape)}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(
            f"{what} is forward-only (inference); run it under torch.no_grad()")
    c, dev = controls, logits.device
    rows, vocab = logits.shape
    if c._rows is not None and (c._rows != rows or c._device != dev):
        raise ValueError(f"{what}: controls of {c._rows} rows on {c._device}, logits of {rows} "
                         f"on {dev}")
    masks, tokens, bias = c.masks, c.tokens, c.bias_ids
    if masks is not None and masks.shape[1] != -(-vocab // 32):
        raise ValueError(f"{what}: masks of {masks.shape[1]} words, {-(-vocab // 32)} needed")
    previous = _native.make_current(dev)
    try:
        src, stride = _rows(logits)
        in_place, given = out is logits, out is not None
        if out is None:
            out, out_stride = src.new_empty((rows, vocab)), vocab
        elif in_place and src is logits:
            out_stride = stride
        else:
            dst, out_stride = _rows(out) if out.dim() == 2 else (None, 0)
            if (dst is not out or out.shape != logits.shape or out.dtype != logits.dtype
                    or out.device != dev):
                raise ValueError(f"{what}: out must be {tuple(logits.shape)} {logits.dtype} on "
                                 f"{dev} with unit column stride and rows of its own")
            if out.requires_grad and torch.is_grad_enabled():
                raise NotImplementedError(f"{what} is forward-only (inference)")
            same = out.data_ptr() == src.data_ptr() and out_stride == stride
            if not same and _overlap(out, src):
                raise ValueError(f"{what}: out shares memory with logits")
        ptr = _native.ptr
        rc = _native.calls().pkv_control_logits(
            out.data_ptr(), out_stride, src.data_ptr(), stride, rows, vocab, ptr(tokens),
            *c._history, ptr(c.lens), ptr(c.prompt_lens),
            ptr(c.repetition), ptr(c.presence), ptr(c.frequency), ptr(bias), ptr(c.bias_values),
            ptr(c.bias_starts), 0 if bias is None else bias.numel(), ptr(masks),
            0 if masks is None else masks.shape[0], ptr(c.mask_rows), code,
            None if status is None else _status_ptr(status, dev, what), _native.stream_ptr(dev))
        if rc:
            _native.check(rc, what)
        if given:  # a graph that saved out finds it changed
            torch.autograd.graph.increment_version(out)
    finally:
        _native.restore(previous)
    return out


def sample_each(logits: torch.Tensor, temperature: torch.Tensor,
                top_k: Optional[torch.Tensor] = None, top_p: Optional[torch.Tensor] = None,
                min_p: Optional[torch.Tensor] = None, uniforms: Optional[torch.Tensor] = None,
                status: Optional[torch.Tensor] = None):
    """One draw a row of logits [rows, vocab] (up to 2^20 of them) with the row's
    temperature (float32 [rows], 0: the largest), top_k (int32, 0: off), top_p (float32, 1:
    off) and min_p (float32, 0: off; a share of the largest probability), by inverse CDF,
    ids ascending, at its uniform in [0, 1) (None: from torch's generator). top-k and top-p
    as in sampling.sample. Logits may be -infinity. Returns (ids int64 [rows], logprobs
    float32 [rows] of the distribution drawn from). A row that cannot be drawn has id -1
    and log-probability NaN, and is reported in `status` (PKV_STATUS_NONFINITE: NaN or
    +infinity; PKV_STATUS_BAD_DISTRIBUTION: all -infinity; PKV_STATUS_BAD_CONTROL: a
    parameter outside its range)."""
    what = "sample_each"
    _native.require_device(logits, what=what)
    code = _native.dtype_code(logits.dtype)
    if logits.dim() != 2 or not 0 < logits.shape[1] <= MAX_SAMPLE_VOCAB:
        raise ValueError(f"{what}: expected [rows, 1 to {MAX_SAMPLE_VOCAB}] logits, "
                         f"got {tuple(logits.shape)}")
    if logits.requires_grad and torch.is_grad_enabled():
        raise NotImplementedError(
            f"{what} is forward-only (inference); run it under torch.no_grad()")
    if temperature is None:
        raise ValueError(f"{what}: temperature must be given, float32 [{logits.shape[0]}]")
    rows, vocab = logits.shape
    dev = logits.device
    for t, dtype, name in ((temperature, torch.float32, "temperature"),
                           (top_k, torch.int32, "top_k"), (top_p, torch.float32, "top_p"),
                           (min_p, torch.float32, "min_p"),
                           (uniforms, torch.float32, "uniforms")):
        if t is not None:
            if t.device != dev:
                raise ValueError(f"{what}: {name} must be on {dev} (got {t.device})")
            _check(t, dtype, (rows,), name, what)
    previous = _native.make_current(dev)
    try:
        if uniforms is None:
            uniforms = torch.rand(rows, device=dev, dtype=torch.float32)
        src, stride = _rows(logits)
        ids = logits.new_empty(rows, dtype=torch.int64)
        logprobs = temperature.new_empty(rows)
        ptr = _native.ptr
        rc = _native.calls().pkv_sample_each(
            ids.data_ptr(), logprobs.data_ptr(), src.data_ptr(), rows, vocab, stride,
            temperature.data_ptr(), ptr(top_k), ptr(top_p), ptr(min_p), uniforms.data_ptr(), code,
            None if status is None else _status_ptr(status, dev, what), _native.stream_ptr(dev))
        if rc:
            _native.check(rc, what)
    finally:
        _native.restore(previous)
    return ids, logprobs


def pack_mask(allowed: torch.Tensor) -> torch.Tensor:
    """bool [..., vocab] -> int32 [..., ceil(vocab / 32)], the words of LogitControls.masks."""
    v = allowed.shape[-1]
    bits = torch.nn.functional.pad(allowed.bool(), (0, -v % 32)).view(*allowed.shape[:-1], -1, 32)
    weights = torch.tensor([1 << i for i in range(31)] + [-(1 << 31)], dtype=torch.int64,
                           device=allowed.device)
    return (bits * weights).sum(-1).to(torch.int32)


class Grammar(Protocol):
    """What a request's tokens may be: a state that its tokens advance."""

    def mask(self) -> torch.Tensor:
        """int32 [ceil(vocab / 32)] (pack_mask): the tokens allowed next."""

    def advance(self, token: int) -> None:
        """The request took `token`."""


def grammar_mask(grammar: Grammar, vocab: int) -> torch.Tensor:
    """The grammar's mask, refused where it is not one of `vocab` tokens."""
    mask, words = grammar.mask(), -(-vocab // 32)
    if not isinstance(mask, torch.Tensor) or tuple(mask.shape) != (words,):
        raise ValueError(f"the grammar's mask must be [{words}] words "
                         f"(got {list(getattr(mask, 'shape', ()))})")
    return mask


def _f32(x) -> float:
    return float(torch.tensor(float(x), dtype=torch.float32))


@dataclass(frozen=True)
class RequestParams:
    """What one request of a batch asks for beyond its prompt (Scheduler.add_request);
    the defaults ask for nothing but a draw at temperature 1. Numbers are checked as the
    float32 that the kernels get, when a request is added: what a step finds ends the request."""
    temperature: float = 1.0         # 0: the most likely token
    top_k: int = 0                   # 0: off
    top_p: float = 1.0
    min_p: float = 0.0
    repetition_penalty: float = 1.0
    presence_penalty: float = 0.0
    frequency_penalty: float = 0.0
    logit_bias: dict = field(default_factory=dict)  # id -> value (-infinity: never)
    grammar: Optional[Grammar] = None
    adapter: int = -1                # of the scheduler's AdapterSet

    def __post_init__(self):
        f32 = {f.name: _f32(getattr(self, f.name)) for f in fields(self)
               if isinstance(f.default, float)}
        if not math.isfinite(f32["temperature"]) or self.temperature < 0:
            raise ValueError("temperature must be finite and >= 0")
        if self.top_k < 0:
            raise ValueError("top_k must be >= 0")
        if not 0 < f32["top_p"] <= 1:
            raise ValueError("top_p must be in (0, 1]")
        if not 0 <= self.min_p <= 1:
            raise ValueError("min_p must be in [0, 1]")
        if not 0 < f32["repetition_penalty"] < math.inf:
            raise ValueError("repetition_penalty must be finite and > 0")
        if not (math.isfinite(f32["presence_penalty"]) and math.isfinite(f32["frequency_penalty"])):
            raise ValueError("presence_penalty and frequency_penalty must be finite")
        object.__setattr__(self, "logit_bias",
                           {int(i): float(v) for i, v in self.logit_bias.items()})
        for i, v in self.logit_bias.items():
            if not 0 <= i < 1 << 31 or not _f32(v) < math.inf:
                raise ValueError("logit_bias names an id below 0, or a value that is NaN or "
                                 f"infinity ({i}: {v})")

    @property
    def has_penalties(self) -> bool:
        return (self.repetition_penalty != 1.0 or self.presence_penalty != 0.0
                or self.frequency_penalty != 0.0)


class TokenHistory:
    """The tokens of running requests on the device, a row each: a step uploads the
    tokens that are new, not the histories."""

    def __init__(self, device):
        self.device = device
        self._buf = torch.zeros((0, 0), dtype=torch.int32, device=device)
        self._row: dict = {}    # request -> row
        self._len: dict = {}    # request -> (tokens, of which the prompt)
        self._free: list = []
        self._new: list = []    # (row, position, token) that are not on the device yet

    def put(self, key, tokens, prompt_len: int) -> None:
        """A request that starts, or starts again, with these tokens."""
        if key not in self._row:
            if not self._free:
                n = self._buf.shape[0]
                self._grow(max(8, 2 * n), self._buf.shape[1])
                self._free = list(range(self._buf.shape[0] - 1, n - 1, -1))
            self._row[key] = self._free.pop()
        r, n = self._row[key], len(tokens)
        self._fit(n)
        self._new = [e for e in self._new if e[0] != r]
        if n:
            self._buf[r, :n] = torch.tensor(tokens, dtype=torch.int32, device=self.device)
        self._len[key] = (n, int(prompt_len))

    def append(self, key, token: int) -> None:
        n, p = self._len[key]
        self._new.append((self._row[key], n, int(token)))
        self._len[key] = (n + 1, p)

    def drop(self, key) -> None:
        if key in self._row:
            r = self._row.pop(key)
            del self._len[key]
            self._new = [e for e in self._new if e[0] != r]
            self._free.append(r)

    def rows(self, keys):
        """(tokens [n, capacity], lens [n], prompt_lens [n]) of these requests; a request
        that was never put has none."""
        if self._new:
            self._fit(max(p for _, p, _ in self._new) + 1)
            row, pos, tok = torch.tensor(self._new, device=self.device).unbind(1)
            self._buf[row, pos] = tok.to(torch.int32)
            self._new = []
        lens = [self._len.get(k, (0, 0)) for k in keys]
        i = torch.tensor([[self._row.get(k, 0), *n] for k, n in zip(keys, lens)],
                         device=self.device)
        if self._buf.numel() == 0:
            tokens = torch.zeros((len(keys), 1), dtype=torch.int32, device=self.device)
        else:
            tokens = self._buf.index_select(0, i[:, 0])
        counts = i[:, 1:].to(torch.int32).t().contiguous()
        return tokens, counts[0], counts[1]

    def _fit(self, n):
        if n > self._buf.shape[1]:
            self._grow(self._buf.shape[0], max(n, 2 * self._buf.shape[1], 256))

    def _grow(self, rows, cap):
        buf = torch.zeros((rows, cap), dtype=torch.int32, device=self.device)
        buf[:self._buf.shape[0], :self._buf.shape[1]] = self._buf
        self._buf = buf


def draw_tokens(logits: torch.Tensor, params, history: TokenHistory, keys):
    """One token a row of logits [rows, vocab] on a ROCm device: row i by params[i]
    (RequestParams) with the tokens of request keys[i] in `history`. Returns (ids,
    log-probabilities) as lists; raises where a row has no token left to draw."""
    masks = {i: grammar_mask(p.grammar, logits.shape[1])
             for i, p in enumerate(params) if p.grammar is not None}
    ids, logprobs, _, status = _draw(logits, params, masks, history, keys)
    if status is not None:
        raise_step_status(status, "draw_tokens")
    return ids, logprobs


def draw_rows(logits: torch.Tensor, params, history: TokenHistory, keys):
    """draw_tokens for rows that have nothing to do with each other: (ids,
    log-probabilities, {row: why}), a row that cannot be drawn having id -1 and its reason
    (a text, or what its grammar's mask() raised) while the others have their tokens."""
    masks, broken = {}, {}
    for i, p in enumerate(params):
        if p.grammar is not None:
            try:
                masks[i] = grammar_mask(p.grammar, logits.shape[1])
            except Exception as e:
                broken[i] = e
    ids, logprobs, changed, status = _draw(logits, params, masks, history, keys)
    failed = {}
    for i in [i for i, tok in enumerate(ids) if tok < 0]:
        row = changed[i].float()
        failed[i] = ("the logits contain NaN or infinity" if not bool((row < math.inf).all())
                     else "there is no token left to draw" if bool((row == -math.inf).all())
                     else "a sampling parameter is outside its range")
    if status is not None and not failed:
        raise_step_status(status, "draw_rows")
    for i in broken:
        ids[i], logprobs[i] = -1, math.nan
    return ids, logprobs, {**failed, **broken}


def _draw(logits, params, masks, history, keys):
    """(ids, log-probabilities, the logits drawn from, the status word or None where it is
    0); masks {row: mask}"""
    n, dev, f32 = len(params), logits.device, torch.float32
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    # one upload of what is a number a row
    nums = torch.tensor([[p.temperature, p.top_p, p.min_p, p.repetition_penalty,
                          p.presence_penalty, p.frequency_penalty, min(p.top_k, 1 << 30)]
                         for p in params], dtype=torch.float64).t().contiguous().to(dev)
    temperature, top_p, min_p, rep, pres, freq = nums[:6].to(f32).unbind(0)
    kw = {}
    if any(p.has_penalties for p in params):
        tokens, lens, prompt_lens = history.rows(keys)
        kw.update(tokens=tokens, lens=lens, prompt_lens=prompt_lens, repetition=rep,
                  presence=pres, frequency=freq)
    if any(p.logit_bias for p in params):
        starts = [0]
        for p in params:
            starts.append(starts[-1] + len(p.logit_bias))
        flat = [(t, v) for p in params for t, v in p.logit_bias.items()]
        kw.update(bias_ids=torch.tensor([t for t, _ in flat], dtype=torch.int32, device=dev),
                  bias_values=torch.tensor([v for _, v in flat], dtype=f32, device=dev),
                  bias_starts=torch.tensor(starts, dtype=torch.int32, device=dev))
    if masks:
        rows = [-1] * n
        for m, i in enumerate(masks):
            rows[i] = m
        kw.update(masks=torch.stack([m.to(dev, torch.int32) for m in masks.values()]),
                  mask_rows=torch.tensor(rows, dtype=torch.int32, device=dev))
    if kw:
        logits = control_logits(logits, LogitControls(**kw), status=status)
    ids, logprobs = sample_each(logits, temperature, nums[6].to(torch.int32), top_p, min_p,
                                status=status)
    got = torch.cat([ids.double(), logprobs.double(), status.double()]).tolist()  # one copy
    return [int(i) for i in got[:n]], got[n:2 * n], logits, status if got[-1] else None
