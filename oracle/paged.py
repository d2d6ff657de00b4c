"""Plain NumPy forms, in float64, of the paged key-value cache's operators and
of token log probabilities: what include/mtx.h says of mtx_kv_append_paged,
mtx_attn_decode_paged, mtx_kv_evict_paged, mtx_token_logprobs and
mtx_token_logprobs_bwd, row by row.

Pools are (n_pages, heads, page, D) arrays, tables (B, max_pages) page ids.
"""
from __future__ import annotations

import numpy as np


def page_row(pool, table, b, j):
    """(page, place) of row j of sequence b, or None where it is not there."""
    page = pool.shape[2]
    if not 0 <= j < table.shape[1] * page:
        return None
    at = int(table[b, j // page])
    return (at, j % page) if 0 <= at < pool.shape[0] else None


def append(k, pool, table, lengths, counts=None):
    """A copy of pool with the rows k (B, heads, T, D) appended."""
    pool = pool.copy()
    B, _, T, _ = k.shape
    for b in range(B):
        n = T if counts is None else min(int(counts[b]), T)
        for i in range(max(n, 0)):
            at = page_row(pool, table, b, int(lengths[b]) - n + i)
            if at is not None:
                pool[at[0], :, at[1]] = k[b, :, i]
    return pool


def rows(pool, table, b, n):
    """(heads, n, D) rows of sequence b in float64 (zeros where not there) and
    which of them are there."""
    out = np.zeros((pool.shape[1], n, pool.shape[3]))
    there = np.zeros(n, bool)
    for j in range(n):
        at = page_row(pool, table, b, j)
        if at is not None:
            out[:, j] = pool[at[0], :, at[1]]
            there[j] = True
    return out, there


def decode(q, k_pool, v_pool, table, lengths, scale):
    """(o, lse, weight each row got (B, Hkv, cap), and two magnitudes that
    error bounds are made of: sum |q||k| per score's row maximum, sum p |v|)."""
    B, H, _, D = q.shape
    Hkv, page = k_pool.shape[1], k_pool.shape[2]
    cap = table.shape[1] * page
    G = H // Hkv
    o, lse = np.zeros((B, H, D)), np.full((B, H), -np.inf)
    w = np.zeros((B, Hkv, cap))
    qk, pv = np.zeros((B, H)), np.zeros((B, H, D))
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cap)
        k, there = rows(k_pool, table, b, n)
        v, _ = rows(v_pool, table, b, n)
        if not there.any():
            continue
        for h in range(H):
            kh, vh = k[h // G][there], v[h // G][there]
            qh = q[b, h, 0].astype(np.float64)
            s = kh @ qh * scale
            m = s.max()
            p = np.exp(s - m)
            lse[b, h] = m + np.log(p.sum())
            p /= p.sum()
            o[b, h] = p @ vh
            w[b, h // G, np.flatnonzero(there)] += p
            qk[b, h] = (np.abs(kh) @ np.abs(qh)).max() * scale
            pv[b, h] = p @ np.abs(vh)
    return o[:, :, None], lse, w, qk, pv[:, :, None]


def evict(k_pool, v_pool, table, lengths, weights, to_table, keep, recent):
    """(new k_pool, v_pool, lengths, weights, slots)."""
    kp, vp = k_pool.copy(), v_pool.copy()
    B, Hkv, ld = weights.shape
    cap = table.shape[1] * k_pool.shape[2]
    new = np.zeros(B, np.int32)
    w_out = weights.copy()
    slots = np.full((B, Hkv, keep), -1, np.int32)
    for b in range(B):
        n = min(max(int(lengths[b]), 0), cap)
        new[b] = min(n, keep)
        for h in range(Hkv):
            if n <= keep:
                kept = list(range(n))
            else:
                old = weights[b, h, :n - recent].astype(np.float64)
                old = np.where(np.isnan(old), np.inf, old)
                nan = np.isnan(weights[b, h, :n - recent])
                order = sorted(range(n - recent), key=lambda j: (-int(nan[j]), -old[j], j))
                kept = sorted(order[:keep - recent]) + list(range(n - recent, n))
            w_out[b, h, :cap] = 0
            for i, j in enumerate(kept):
                slots[b, h, i] = j
                w_out[b, h, i] = weights[b, h, j]
                frm, to = page_row(k_pool, table, b, j), page_row(k_pool, to_table, b, i)
                if to is not None:
                    kp[to[0], h, to[1]] = 0 if frm is None else k_pool[frm[0], h, frm[1]]
                    vp[to[0], h, to[1]] = 0 if frm is None else v_pool[frm[0], h, frm[1]]
    return kp, vp, new, w_out, slots


def logprobs(logits, tokens, scale=1.0, top=0):
    """(logprob, entropy, lse, top_ids, top_logprobs, p) of logits (rows, V)."""
    x = logits.astype(np.float64) * scale
    R, V = x.shape
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(1)
        m0 = np.where(np.isneginf(m), 0.0, m)
        e = np.exp(x - m0[:, None])
        l = e.sum(1)
        lse = m0 + np.log(l)
        lp = np.where((l == 0)[:, None], -np.inf, x - lse[:, None])
        p = np.where((l == 0)[:, None], 0.0, np.exp(lp))
        entropy = -np.where(p == 0, 0.0, p * lp).sum(1)
    ids = np.zeros((R, top), np.int64)
    for r in range(R):
        nan = np.isnan(logits[r])
        key = np.where(nan, np.inf, logits[r].astype(np.float64))
        ids[r] = np.lexsort((np.arange(V), -key, ~nan))[:top]
    has = (tokens >= 0) & (tokens < V)
    t = np.where(has, tokens, 0)
    logprob = np.where(has, lp[np.arange(R), t], 0.0)
    return logprob, entropy, lse, ids, np.take_along_axis(lp, ids, 1), p


def logprobs_grad(logits, tokens, g, gh, scale=1.0):
    """The logits' gradient, g and gh those of logprob and entropy."""
    _, entropy, lse, _, _, p = logprobs(logits, tokens, scale)
    V = logits.shape[1]
    x = logits.astype(np.float64) * scale
    with np.errstate(invalid="ignore"):
        lp = np.where(p == 0, 0.0, x - lse[:, None])
    has = (tokens >= 0) & (tokens < V) & ~np.isneginf(lse)
    g = np.where(has, g.astype(np.float64), 0.0)
    d = -p * (g[:, None] + gh.astype(np.float64)[:, None] * (lp + entropy[:, None]))
    r = np.flatnonzero(has)
    d[r, tokens[r]] += g[r]
    return d * scale
