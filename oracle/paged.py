"""Plain restatements in float64 of the paged-cache operators (test infrastructure only):
the cache append, attention of new tokens, accumulated weights and eviction, one sequence
and head at a time.  Layouts as in include/w4a8.h; caches as float64 arrays
[pages, KVH, page, D]."""

import numpy as np


def slots(table, b, n, page):
    """(page, row) of slots 0 .. n of sequence b."""
    j = np.arange(n)
    return table[b, j // page], j % page


def norm_rope(x, w, eps, cs, interleaved):
    """x f64 [rows, D]: RMS norm by w (or None), then the first rot dims turned by
    cs [rows, rot] (cosines | sines; rot may be 0)."""
    x = np.array(x, np.float64)
    if w is not None:
        x = x / np.sqrt((x ** 2).mean(1, keepdims=True) + eps) * w
    half = cs.shape[1] // 2
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    c, s = cs[:, :half], cs[:, half:]
    xa, xb = x[:, a].copy(), x[:, b].copy()
    x[:, a], x[:, b] = xa * c - xb * s, xb * c + xa * s
    return x


def attention(q, k, v, table, q_start, kv_len, scale, gate=None):
    """(o [T, H, D], lse [T, H]) in float64; rows that see nothing: 0 and -inf."""
    T, H, D = q.shape
    KVH, page = k.shape[1], k.shape[2]
    o, lse = np.zeros((T, H, D)), np.full((T, H), -np.inf)
    for b in range(len(kv_len)):
        n, L = q_start[b + 1] - q_start[b], kv_len[b]
        pg, row = slots(table, b, L, page)
        for i in range(n):
            m = L - n + i + 1
            if m <= 0:
                continue
            t = q_start[b] + i
            for h in range(H):
                kh = h // (H // KVH)
                s = k[pg[:m], kh, row[:m]] @ q[t, h] * scale
                top = s.max()
                e = np.exp(s - top)
                o[t, h] = e @ v[pg[:m], kh, row[:m]] / e.sum()
                lse[t, h] = top + np.log(e.sum())
    if gate is not None:
        o = o / (1 + np.exp(-gate.astype(np.float64)))
    return o, lse


def weights(q, lse, k, table, q_start, kv_len, scale, acc):
    """acc f64 [B, KVH, slots] plus the weight each slot received."""
    acc = np.array(acc, np.float64)
    H, KVH, page = q.shape[1], k.shape[1], k.shape[2]
    for b in range(len(kv_len)):
        n, L = q_start[b + 1] - q_start[b], kv_len[b]
        pg, row = slots(table, b, L, page)
        for i in range(n):
            m = L - n + i + 1
            if m <= 0:
                continue
            t = q_start[b] + i
            for h in range(H):
                kh = h // (H // KVH)
                acc[b, kh, :m] += np.exp(k[pg[:m], kh, row[:m]] @ q[t, h] * scale - lse[t, h])
    return acc


def evict(k, v, table, kv_len, acc, pos, keep, protect_from, sink):
    """(k, v, moves, acc, pos, len) after eviction; acc and pos lists per (sequence, head) of
    the new length."""
    k, v = k.copy(), v.copy()
    page = k.shape[2]
    acc_out, pos_out, lens = {}, {}, []
    for b in range(len(kv_len)):
        L = int(kv_len[b])
        n = min(L, int(keep[b]))
        lens.append(n)
        pg, row = slots(table, b, L, page)
        for h in range(k.shape[1]):
            a, p = acc[b, h, :L], pos[b, h, :L]
            safe = [p[j] < sink or p[j] >= protect_from[b] for j in range(L)]  # before any weight, by slot
            w = [0.0 if safe[j] else (-np.inf if np.isnan(a[j]) else a[j]) for j in range(L)]
            kept = set(sorted(range(L), key=lambda j: (not safe[j], -w[j], j))[:n])
            came = np.arange(n)
            came[[j for j in range(n) if j not in kept]] = sorted(j for j in kept if j >= n)
            for x in (k, v):
                x[pg[:n], h, row[:n]] = x[pg[came], h, row[came]]
            acc_out[b, h], pos_out[b, h] = a[came], p[came]
    return k, v, acc_out, pos_out, lens
