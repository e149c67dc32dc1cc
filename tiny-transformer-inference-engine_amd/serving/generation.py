"""Paged generation loops — drop-in for serving/generation.py.

Entry points and their reference counterparts:
  generate_batched      serving/generation.py:112-148  greedy, token ids in
  generate_batched_text serving/generation.py:11-69    sampled, text in,
                                                       stops a row at EOS
  generate_paged        serving/generation.py:91-110   greedy, one sequence
  prefill_seq           serving/generation.py:71-77
  decode_step           serving/generation.py:80-88
  generate_speculative  no counterpart: generate_batched's tokens, several a
                        step, by verifying a drafting function's trees

The batched entry points share one driver (_drive): a _Cohort holds the
calls' sequences, feeds the model one prefill step of whole prompts and then
at most max_new_tokens - 1 decode steps of one token per running sequence,
and returns every block to the allocator when the call ends, normally or by
an exception. Per step the next tokens of the whole batch come from one
device call (one argmax kernel, or one sampling kernel) and one
device-to-host copy, instead of one per row. A row that samples
eos_token_id stops there; the EOS token is not part of its output, and the
decode steps after it leave that row out of the batch.
"""
from __future__ import annotations

import torch

from .batch import build_batch_step
from .paged_meta import DeviceTables, build_batch_meta, raise_step_status
from .sampling import greedy, sample
from .sequence import Sequence, blocks_for
from .tree_decode import MAX_TREE_NODES, build_tree_meta, tree_accept


class _Cohort:
    """The sequences of one batched call.

    rows      Sequence objects, in prompt order
    produced  tokens emitted per row so far
    running   indices of the rows still generating, ascending (the row order
              of the next decode batch)
    feed      the token each running row feeds to the next decode step
    """

    def __init__(self, id_lists, block_size, alloc, device):
        self.alloc = alloc
        self.device = device
        self.rows = [Sequence(n, list(ids), block_size) for n, ids in enumerate(id_lists)]
        self.produced = [[] for _ in self.rows]
        self.running = list(range(len(self.rows)))
        self.feed = {}

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for row in self.rows:
            row.release(self.alloc)
        return False

    def prefill_batch(self):
        for row in self.rows:
            row.ensure_blocks(self.alloc)
        return build_batch_step([(row, row.token_ids) for row in self.rows], self.device)

    def decode_batch(self):
        entries = []
        for n in self.running:
            row = self.rows[n]
            row.append_token(self.feed[n])
            row.ensure_blocks(self.alloc)
            entries.append((row, [self.feed[n]]))
        return build_batch_step(entries, self.device)

    def accept(self, tokens, stop_id):
        """tokens[i] is the pick of batch row i, i.e. of rows[running[i]]."""
        still = []
        for n, tok in zip(self.running, tokens):
            if stop_id is not None and tok == stop_id:
                continue
            self.produced[n].append(tok)
            self.feed[n] = tok
            still.append(n)
        self.running = still


def _drive(model, pool, cohort, max_new_tokens, pick, stop_id=None):
    cohort.accept(pick(model.forward_batch(cohort.prefill_batch(), pool)), stop_id)
    for _ in range(max_new_tokens - 1):
        if not cohort.running:
            break
        cohort.accept(pick(model.forward_batch(cohort.decode_batch(), pool)), stop_id)
    return cohort.produced


def _model_device(model):
    return next(model.parameters()).device


def _greedy_ids(logits):
    return greedy(logits)[:, 0].tolist()


@torch.no_grad()
def generate_batched(model, prompts_ids, max_new_tokens, pool, alloc, block_size=16):
    """prompts_ids: list of token-id lists. Returns the greedy continuation of
    each (max_new_tokens tokens, no EOS stop), in prompt order."""
    if max_new_tokens < 0:
        raise ValueError("max_new_tokens must be >= 0")
    if not prompts_ids:
        return []
    if not all(prompts_ids):
        raise ValueError("every prompt must contain at least one token")
    if max_new_tokens == 0:
        return [[] for _ in prompts_ids]
    with _Cohort(prompts_ids, block_size, alloc, _model_device(model)) as cohort:
        return _drive(model, pool, cohort, max_new_tokens, _greedy_ids)


def _draft_tree(draft, history, limit, depth, vocab):
    """draft(history) -> (tokens, parents), checked; the nodes below the root as
    (tokens, parents of the whole tree): the first `limit` of those fewer than
    `depth` levels below the root, deeper ones can add nothing."""
    tokens, parents = draft(history)
    tokens, parents = [int(t) for t in tokens], [int(p) for p in parents]
    if len(tokens) != len(parents):
        raise ValueError("a draft needs one parent per token")
    kept, above, node, level = [], [], [], [0]  # node: the place in the tree, None: left out
    for i, (t, p) in enumerate(zip(tokens, parents)):
        if not -1 <= p < i:
            raise ValueError(f"draft node {i}: parent {p} is neither -1 nor an earlier node")
        if not 0 <= t < vocab:
            raise ValueError(f"draft node {i}: token {t} is outside the vocabulary ({vocab})")
        up = 0 if p == -1 else node[p]
        if up is None or len(kept) == limit or level[up] + 1 >= depth:
            node.append(None)
            continue
        kept.append(t)
        above.append(up)
        level.append(level[up] + 1)
        node.append(len(kept))
    return kept, above


@torch.no_grad()
def generate_speculative(model, prompts_ids, max_new_tokens, pool, alloc, draft, block_size=16,
                         max_drafts=15, max_depth=8):
    """generate_batched on a ROCm device, several tokens a step. draft(token_ids)
    is called per row and step with the row's tokens so far and proposes a tree
    that goes on from the last of them: (tokens, parents), parents[i] the index of
    the proposed token that token i follows, -1 for those that follow the last
    token; at most max_drafts of them are used, and none too deep to be kept. The model verifies all rows' trees
    in one pass and keeps, per row, the longest path of its own greedy choices and
    the token after it, up to max_depth tokens: whatever is drafted, the tokens
    are greedy ones. Rejected drafts take no pool slots, so the pool and the positions
    needed are generate_batched's."""
    if max_new_tokens < 0:
        raise ValueError("max_new_tokens must be >= 0")
    if max_depth < 1 or not 0 <= max_drafts < MAX_TREE_NODES:
        raise ValueError(f"need max_depth >= 1 and 0 <= max_drafts < {MAX_TREE_NODES}")
    if not prompts_ids:
        return []
    if not all(prompts_ids):
        raise ValueError("every prompt must contain at least one token")
    if max_new_tokens == 0:
        return [[] for _ in prompts_ids]
    max_depth = min(max_depth, 1 + max_drafts, max_new_tokens)  # no path is longer
    device = _model_device(model)
    vocab = model.lm_head.out_features
    stock = []
    with _Cohort(prompts_ids, block_size, alloc, device) as cohort:
        first = _greedy_ids(model.forward_batch(cohort.prefill_batch(), pool))
        rows = [list(ids) + [tok] for ids, tok in zip(prompts_ids, first)]
        goal = [len(ids) + max_new_tokens for ids in prompts_ids]
        # no tree goes past its row's goal, and the last token takes no slot
        need = [blocks_for(g - 1, block_size) for g in goal]
        held = [len(r.block_table) for r in cohort.rows]
        try:
            stock = alloc.allocate_n(sum(need) - sum(held))
            tables = DeviceTables.from_host([r.block_table for r in cohort.rows],
                                            [len(ids) for ids in prompts_ids], stock, max(need),
                                            block_size, pool.num_blocks, device)
            status = torch.zeros(1, dtype=torch.int32, device=device)
            while any(len(r) < g for r, g in zip(rows, goal)):
                tokens, parents, starts = [], [], [0]
                for row, g in zip(rows, goal):
                    if len(row) < g:  # a finished row takes no nodes
                        t, p = _draft_tree(draft, list(row), max_drafts,
                                           min(max_depth, g - len(row)), vocab)
                        tokens += [row[-1]] + t
                        parents += [-1] + p
                    starts.append(len(tokens))
                i32 = torch.tensor(parents + starts, dtype=torch.int32, device=device)
                ids = torch.tensor(tokens, dtype=torch.long, device=device)
                tree = build_tree_meta(tables, i32[:len(parents)], i32[len(parents):],
                                       1 + max_drafts, max(len(r) for r in rows), status=status)
                logits, k_rows, v_rows = model.forward_tree(ids, pool, tree, status)
                accepted = tree_accept(greedy(logits)[:, 0], ids, tree, max_depth, status=status)
                meta, tables = build_batch_meta(tables, accepted.lens, len(rows) * max_depth,
                                                max_depth, status=status)
                pool.write_accepted(k_rows, v_rows, tree, accepted, meta)
                # one copy to the host: lengths and tokens of the whole batch
                new = torch.cat([accepted.lens[:, None].long(), accepted.tokens], 1).tolist()
                for row, (n, *toks) in zip(rows, new):
                    row += toks[:n]
            raise_step_status(status, "generate_speculative")
        finally:
            alloc.free(stock)
    return [row[len(ids):g] for row, ids, g in zip(rows, prompts_ids, goal)]


def _default_tokenizer():
    try:
        import tiktoken
    except ImportError as e:
        raise RuntimeError(
            "generate_batched_text needs a tokenizer: install tiktoken or pass tokenizer=") from e
    return tiktoken.get_encoding("gpt2")


@torch.no_grad()
def generate_batched_text(model, cfg, prompts, max_new_tokens, eos_token_id,
                          pool, alloc, temperature=1.0, top_k=32, top_p=0.9,
                          block_size=16, tokenizer=None):
    """Sampled batched generation from text prompts. Returns the token ids
    each prompt produced before it sampled eos_token_id (or before
    max_new_tokens). tokenizer: any object with encode_ordinary(str); the
    reference's tiktoken "gpt2" encoding when None."""
    if max_new_tokens < 0:
        raise ValueError("max_new_tokens must be >= 0")
    if not prompts:
        return []
    if temperature <= 0 or top_k < 0 or not 0 < top_p <= 1:
        raise ValueError("invalid sampling parameters")
    enc = tokenizer if tokenizer is not None else _default_tokenizer()
    id_lists = [enc.encode_ordinary(text) for text in prompts]
    if not all(id_lists):
        raise ValueError("every prompt must encode to at least one token")
    if max(len(ids) for ids in id_lists) + max_new_tokens > cfg.max_seq_len:
        raise ValueError("prompt plus requested generation exceeds max_seq_len")
    if max_new_tokens == 0:
        return [[] for _ in prompts]

    def pick(logits):
        return sample(logits, temperature=temperature, top_k=top_k, top_p=top_p)[:, 0].tolist()

    with _Cohort(id_lists, block_size, alloc, _model_device(model)) as cohort:
        return _drive(model, pool, cohort, max_new_tokens, pick, stop_id=eos_token_id)


def _last_position_argmax(model, seq, pool, new_ids):
    """Runs new_ids (the last len(new_ids) tokens of seq) through the
    single-sequence model call and returns the argmax at the last position."""
    x = torch.tensor([new_ids], dtype=torch.long, device=_model_device(model))
    logits = model(x, pool, seq.block_table, start=seq.num_tokens - len(new_ids))
    return int(logits[0, -1].argmax())


@torch.no_grad()
def prefill_seq(model, seq, pool, alloc):
    """Whole prompt of seq from position 0; returns its greedy next token."""
    seq.ensure_blocks(alloc)
    return _last_position_argmax(model, seq, pool, seq.token_ids)


@torch.no_grad()
def decode_step(model, seq, pool, alloc, token_id):
    """Appends token_id to seq, runs it at its position, returns the greedy
    next token."""
    seq.append_token(token_id)
    seq.ensure_blocks(alloc)
    return _last_position_argmax(model, seq, pool, [token_id])


@torch.no_grad()
def generate_paged(model, prompt_ids, max_new_tokens, pool, alloc, block_size=16):
    """Greedy single-sequence generation: one prefill call, then one decode
    call per further token."""
    if max_new_tokens < 0:
        raise ValueError("max_new_tokens must be >= 0")
    if not prompt_ids:
        raise ValueError("prompt must contain at least one token")
    if max_new_tokens == 0:
        return []
    seq = Sequence(0, list(prompt_ids), block_size)
    try:
        out = [prefill_seq(model, seq, pool, alloc)]
        while len(out) < max_new_tokens:
            out.append(decode_step(model, seq, pool, alloc, out[-1]))
        return out
    finally:
        seq.release(alloc)
