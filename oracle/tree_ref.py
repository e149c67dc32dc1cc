"""Plain implementations of the tree-verification step in 64 bits and on Python
lists — TEST INFRASTRUCTURE ONLY, never used by the product. No counterpart in
the reference (it drafts nothing); the definitions are the operators' own.
"""
from __future__ import annotations

import math

import numpy as np

NO_SLOT = -(1 << 63)


def visible_from_parents(parents):
    """[n, n] bool: node i sees j iff j is i or above it; a parent that is neither
    -1 nor an earlier node cuts there. Also the depths."""
    n = len(parents)
    vis, depth = np.zeros((n, n), dtype=bool), np.zeros(n, dtype=np.int64)
    for i in range(n):
        p = int(parents[i])
        if 0 <= p < i:
            vis[i], depth[i] = vis[p], depth[p] + 1
        vis[i, i] = True
    return vis, depth


def pack_masks(vis_list, total, words):
    """Per-sequence [n, n] visibilities, rows behind one another -> int64 [total, words]."""
    out = np.zeros((total, words), dtype=np.uint64)
    at = 0
    for vis in vis_list:
        for i in range(vis.shape[0]):
            for j in np.nonzero(vis[i])[0]:
                out[at + i, j >> 6] |= np.uint64(1) << np.uint64(j & 63)
        at += vis.shape[0]
    return out.view(np.int64)


def tree_attention(q, k, v, k_pool, v_pool, tables, ctx, qsl, vis_list, scale=None):
    """float64 arrays: q [T, hq, d], k / v [T, hkv, d], pools [nb, bs, hkv, d]; keys a row
    does not see are left out of its sums. Returns out, lse, and per row A = the
    softmax-weighted mean of |v| [T, hq, d], S = the largest scale * sum |q_i k_i|
    [T, hq] and V1 = sum of |v| over its keys [T, hq, d] (for tolerances)."""
    T, hq, d = q.shape
    bs, hkv = k_pool.shape[1], k_pool.shape[2]
    G = hq // hkv
    scale = scale if scale else 1.0 / math.sqrt(d)
    out, lse = np.zeros((T, hq, d)), np.full((T, hq), np.inf)
    A, S, V1 = np.zeros((T, hq, d)), np.zeros((T, hq)), np.zeros((T, hq, d))
    fk, fv = k_pool.reshape(-1, hkv, d), v_pool.reshape(-1, hkv, d)
    for s, vis in enumerate(vis_list):
        a, n = int(qsl[s]), vis.shape[0]
        pos = np.arange(int(ctx[s]))
        slots = np.asarray(tables[s], dtype=np.int64)[pos // bs] * bs + pos % bs
        for i in range(n):
            seen = np.nonzero(vis[i])[0] + a
            for h in range(hkv):
                kk = np.concatenate([fk[slots, h], k[seen, h]])
                vv = np.concatenate([fv[slots, h], v[seen, h]])
                if kk.shape[0] == 0:
                    continue
                qq = q[a + i, h * G:(h + 1) * G]
                with np.errstate(invalid="ignore", over="ignore"):
                    sc = scale * qq @ kk.T
                    m = sc.max(-1, keepdims=True)
                    p = np.exp(sc - m)
                    l = p.sum(-1, keepdims=True)
                    r = slice(h * G, (h + 1) * G)
                    out[a + i, r] = (p / l) @ vv
                    lse[a + i, r] = (m + np.log(l))[:, 0]
                    A[a + i, r] = (p / l) @ np.abs(vv)
                    S[a + i, r] = (scale * np.abs(qq) @ np.abs(kk).T).max(-1)
                    V1[a + i, r] = np.abs(vv).sum(0)
    return out, lse, A, S, V1


def build_step(tables, held, ctx, q, free, cursor, bs, num_blocks, num_tokens, max_q_len):
    """tables [N][max_blk] list (changed in place on success). Returns a dict of the
    state after, the metadata and the status bits' names."""
    n, width = len(tables), len(tables[0]) if tables else 0
    status, need = set(), []
    q = list(q)
    for s in range(n):
        if q[s] < 0 or q[s] > max_q_len or ctx[s] < 0 or held[s] < 0:
            status.add("qloc")
            q[s] = 0
        blocks = -(-(ctx[s] + q[s]) // bs) if q[s] else 0
        if q[s] and (blocks > width or held[s] > width):
            status.add("short")
            blocks = 0
        need.append(max(0, blocks - held[s]))
    if not 0 <= cursor <= len(free) or sum(need) > len(free) - cursor:
        status.add("blocks")
    if sum(q) > num_tokens:
        status.add("qloc")
    fails = bool(status)
    held_out, ctx_out, at = list(held), list(ctx), cursor
    if not fails:
        for s in range(n):
            for b in range(need[s]):
                tables[s][held[s] + b] = free[at]
                at += 1
            held_out[s] += need[s]
            ctx_out[s] += q[s]
    qsl = np.concatenate([[0], np.cumsum(q)]).astype(np.int64).tolist()
    positions, slots = [0] * num_tokens, [NO_SLOT] * num_tokens
    for s in range(n):
        for i in range(q[s]):
            t, p = qsl[s] + i, ctx[s] + i
            if t >= num_tokens:
                continue
            positions[t] = p
            if p // bs < min(held_out[s], width) and 0 < tables[s][p // bs] < num_blocks:
                slots[t] = tables[s][p // bs] * bs + p % bs
            elif not fails:
                status.add("block")
    return dict(held=held_out, ctx=ctx_out, cursor=at, qsl=qsl, positions=positions, slots=slots,
                seq_lens=[c + x if x else 0 for c, x in zip(ctx, q)],
                start_pos=[c if x else 0 for c, x in zip(ctx, q)], status=status)


def accept(picks, tokens, parents, qsl, max_depth):
    lens, path, out = [], [], []
    for s in range(len(qsl) - 1):
        a, b = int(qsl[s]), int(qsl[s + 1])
        walk = [0] if b > a else []
        while walk and len(walk) < max_depth:
            cur = walk[-1]
            nxt = [i for i in range(cur + 1, b - a)
                   if parents[a + i] == cur and tokens[a + i] == picks[a + cur]]
            if not nxt:
                break
            walk.append(nxt[0])
        lens.append(len(walk))
        path.append(walk + [-1] * (max_depth - len(walk)))
        out.append([int(picks[a + i]) for i in walk] + [-1] * (max_depth - len(walk)))
    return lens, path, out
