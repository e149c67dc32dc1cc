"""Restatement in 64 bits of the operators for batches whose requests differ — TEST
INFRASTRUCTURE ONLY, never used by the product: rows grouped by adapter, low-rank adapters
beside a projection, logit controls, and a draw with every row's own parameters."""
from __future__ import annotations

import numpy as np
import torch


def plan(ids, num_adapters, tile_rows):
    """(order, starts, tiles) of a step's adapter ids: rows sorted by adapter, in their
    own order within one, those without (any id outside [0, num_adapters)) last."""
    ids = np.asarray(ids, dtype=np.int64).reshape(-1)
    group = np.where((ids >= 0) & (ids < num_adapters), ids, num_adapters)
    order, starts, tiles = [], [0], []
    for g in range(num_adapters + 1):
        rows = np.nonzero(group == g)[0].tolist()
        for at in range(0, len(rows), tile_rows):
            tiles.append([g if g < num_adapters else -1, starts[-1] + at,
                          min(tile_rows, len(rows) - at), 0])
        order += rows
        starts.append(starts[-1] + len(rows))
    return order, starts, tiles


def adapted(base, x, a, b, scales, ids, parts, rank):
    """base + scale * B (A x) of every row, float64 tensors: a [N, parts * rank, k],
    b [N, n, rank]."""
    y = base.double().clone()
    for t, i in enumerate(ids):
        if not 0 <= i < a.shape[0]:
            continue
        low = float(scales[i]) * (a[i].double() @ x[t].double())
        at = 0
        for s, n in enumerate(parts):
            y[t, at:at + n] += b[i, at:at + n].double() @ low[s * rank:(s + 1) * rank]
            at += n
    return y


def adapted_bound(base, x, a, b, scales, ids, parts, rank):
    """The same with the magnitudes of every term: what rounding errors scale with."""
    return adapted(base.abs(), x.abs(), a.abs(), b.abs(), [abs(float(s)) for s in scales], ids,
                   parts, rank)


def swiglu(y):
    gate, up = y.chunk(2, 1)
    return gate * torch.sigmoid(gate) * up


def control(row, tokens, prompt, repetition, presence, frequency, biases, allowed):
    """One row of logits (float64 [vocab]): tokens the row's history, the first `prompt` of
    it the prompt; biases [(id, value)]; allowed None or a boolean array."""
    out = np.array(row, dtype=np.float64)
    vocab = len(out)
    inside = [int(t) for t in tokens if 0 <= t < vocab]
    made = [int(t) for t in tokens[prompt:] if 0 <= t < vocab]
    for t in set(inside):
        out[t] = out[t] / repetition if out[t] > 0 else out[t] * repetition
    for t in set(made):
        out[t] -= frequency * made.count(t) + presence
    for t, v in biases:
        if 0 <= t < vocab:
            out[t] += v
    if allowed is not None:
        out[~allowed] = -np.inf
    return out


def kept(row, temperature, top_k, top_p, min_p):
    """(weights of the kept ids, 0 elsewhere) of one row of logits, temperature > 0."""
    row = np.asarray(row, dtype=np.float64)
    order = np.lexsort((np.arange(len(row)), -row))
    e = np.exp((row[order] - row[order[0]]) / temperature)
    keep = np.ones(len(row), dtype=bool)
    if 0 < top_k < len(row):
        keep &= row[order] >= row[order[top_k - 1]]
    if top_p < 1:
        e_kept = np.where(keep, e, 0.0)
        before = np.cumsum(e_kept) - e_kept
        keep &= before <= top_p * e_kept.sum()
        keep[0] = True
    keep &= e >= min_p
    keep[0] = True
    out = np.zeros(len(row))
    out[order[keep]] = e[keep]
    return out


def draw(row, temperature, top_k, top_p, min_p, u):
    """(id, log-probability, distance of u to the nearest border as a share of the sum)."""
    if temperature == 0:
        return int(np.argmax(row)), 0.0, 1.0
    e = kept(row, temperature, top_k, top_p, min_p)
    c = np.cumsum(e)
    i = int(np.searchsorted(c, u * c[-1], side="right"))
    return i, float(np.log(e[i] / c[-1])), float(np.min(np.abs(c[e > 0] / c[-1] - u)))
