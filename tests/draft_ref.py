"""Plain implementations of the draft operators in 64 bits and more (numpy and Python integers), for
the tests: attention of draft trees, beam selection, and the moves of cache rows. Written from the
definitions in include/hardshell_b200.h."""

from __future__ import annotations

import numpy as np


def rescale(x: np.ndarray, m: int, s: int) -> np.ndarray:
    """floor((x m + 2^(s-1)) / 2^s) with Python integers, an exact 0 for s > 95 (int.rs:63-110)."""
    x = np.asarray(x)
    if s > 95:
        return np.zeros(x.shape, dtype=object)
    y = x.astype(object) * int(m)
    return y if s == 0 else (y + (1 << (s - 1))) >> s


def rescale_clamped(x: np.ndarray, m: int, s: int, lim: int) -> np.ndarray:
    return np.clip(rescale(x, m, s), -lim, lim).astype(np.int64)


def attend(q, k, v, seen, rule) -> np.ndarray:
    """One head: q [r, hd], k [n, hd], v [hd, n] (int8), seen [r, n] -> int8 [r, hd]."""
    table = np.asarray(rule["table"], dtype=np.int64)
    dot = q.astype(np.int64) @ k.astype(np.int64).T
    score = rescale_clamped(dot, rule["score_m"], rule["score_s"], 1 << 40)
    out = np.zeros((q.shape[0], v.shape[0]), dtype=np.int8)
    for r in range(q.shape[0]):
        at = np.flatnonzero(seen[r])
        if at.size == 0:
            continue
        d = np.minimum(score[r, at].max() - score[r, at], len(table) - 1)
        e = table[d]
        total = max(int(e.sum()), 1)
        p = (e << rule["P"]) // total
        acc = (p.astype(object) * v[:, at].astype(object)).sum(1)
        out[r] = rescale_clamped(acc, rule["out_m"], rule["out_s"], 127).astype(np.int8)
    return out


def tree_attention(k, v, q, seqs, mask, rule, n_kv, plane0, out) -> np.ndarray:
    """k [slots, planes, n_ctx, hd], v [slots, planes, hd, n_ctx], q [rows, heads, hd]; `out` as it was
    before the call (rows of no tree stay)."""
    out = out.copy()
    group = q.shape[1] // n_kv
    for first, count, slot, prefix in np.asarray(seqs).tolist():
        if count == 0:
            continue
        words = np.asarray(mask[first:first + count], dtype=np.uint32)
        bits = ((words[:, :, None] >> np.arange(32, dtype=np.uint32)) & 1).reshape(count, -1)[:, :count].astype(bool)
        seen = np.concatenate([np.ones((count, prefix), bool), bits], 1)
        n = prefix + count
        for h in range(q.shape[1]):
            pl = plane0 + h // group
            out[first:first + count, h] = attend(q[first:first + count, h], k[slot, pl, :n], v[slot, pl, :, :n], seen,
                                                 rule)
    return out


def norm_of(table, total: int) -> int:
    """The entries table[j] with table[j] * total > table[0]^2."""
    one = int(table[0]) ** 2
    return sum(1 for t in table if int(t) * total > one)


def beam_select(dist, tops, tile_shift, vocab, beams, keep, base, finished, table):
    """(parent, token, cost) of [groups, keep]; -1 in the place of no candidate."""
    table = [int(t) for t in table]
    last, groups = len(table) - 1, len(base) // beams
    out = [np.full((groups, keep), -1, dtype=np.int64) for _ in range(3)]
    for g in range(groups):
        found = []
        for b in range(beams):
            row = g * beams + b
            if base[row] < 0 or base[row] >= 1 << 62:
                continue
            if finished is not None and finished[row]:
                found.append((int(base[row]), b, -1))
                continue
            tr = [int(x) for x in tops[row][:((vocab - 1) >> tile_shift) + 1]]
            top = max(tr)
            d = [min(top - tr[s >> tile_shift] + int(dist[row][s]), last) for s in range(vocab)]
            n = norm_of(table, sum(table[x] for x in d))
            found += [(int(base[row]) + n + d[s], b, s) for s in range(vocab) if table[d[s]] > 0]
        for i, (c, b, s) in enumerate(sorted(found)[:keep]):
            out[0][g, i], out[1][g, i], out[2][g, i] = b, s, c
    return out


def reorder(k, v, slots, parents, rows, beams):
    k2, v2 = k.copy(), v.copy()
    for i, p in enumerate(np.asarray(parents).reshape(-1).tolist()):
        g, j = divmod(i, beams)
        if p == j or p < 0 or p == 0xFFFFFFFF:
            continue
        src, n = slots[g * beams + p], rows[g * beams + p]
        k2[slots[i], :, :n] = k[src, :, :n]
        v2[slots[i], :, :, :n] = v[src, :, :, :n]
    return k2, v2


def commit(k, v, seqs, path, lengths):
    k2, v2 = k.copy(), v.copy()
    for (_, _, slot, prefix), p, n in zip(np.asarray(seqs).tolist(), np.asarray(path).tolist(), lengths):
        for j in range(n):
            k2[slot, :, prefix + j] = k[slot, :, prefix + p[j]]
            v2[slot, :, :, prefix + j] = v[slot, :, :, prefix + p[j]]
    return k2, v2


def ancestors(parents, words: int) -> np.ndarray:
    """The masks of a tree given by parents (-1: the context): a node's bit and its ancestors'."""
    out = np.zeros((len(parents), words), dtype=np.uint32)
    for i, p in enumerate(parents):
        if p >= 0:
            out[i] = out[p]
        out[i, i >> 5] |= np.uint32(1 << (i & 31))
    return out
