"""float64 oracle of the paged key/value cache: what is appended to it, and attention over it.

Written from the definitions, a token and a head at a time.  Arrays are numpy float64 (16-bit
values convert exactly); the plan (table, lengths, cu_q) is integers.
"""
import numpy as np


def positions(seq_lens, cu_q, n_tokens, capacity):
    """(sequence, position) of each packed token; sequence -1 for padding, position -1 for none."""
    out = []
    for t in range(n_tokens):
        b = -1
        for i in range(len(seq_lens)):
            if cu_q[i] <= t < cu_q[i + 1]:
                b = i
        p = -1 if b < 0 else int(seq_lens[b]) - int(cu_q[b + 1]) + t
        out.append((b, p if 0 <= p < capacity else -1))
    return out


def place(table, b, pos, page_size, num_pages):
    """(page, row) of a position, or None where no page is mapped."""
    page = int(table[b][pos // page_size])
    return (page, pos % page_size) if 0 <= page < num_pages else None


def rotate(x, cos, sin, interleaved):
    """x (heads, hs) with its first 2 len(cos) elements rotated in pairs."""
    y, half = x.copy(), len(cos)
    i = np.arange(half)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
    y[:, a] = x[:, a] * cos - x[:, b] * sin
    y[:, b] = x[:, b] * cos + x[:, a] * sin
    return y


def append(k, v, k_cache, v_cache, table, seq_lens, cu_q, q=None, cos=None, sin=None,
           interleaved=False):
    """(q rotated, k_cache, v_cache, written): new caches, and which rows of them were written."""
    pages, _, ps, _ = k_cache.shape
    k_cache, v_cache = k_cache.copy(), v_cache.copy()
    written = np.zeros((pages, ps), dtype=bool)
    q = None if q is None else q.copy()
    for t, (b, p) in enumerate(positions(seq_lens, cu_q, k.shape[0], len(table[0]) * ps)):
        if p < 0:
            continue
        kt = k[t]
        if cos is not None:
            q[t] = rotate(q[t], cos[p], sin[p], interleaved)
            kt = rotate(kt, cos[p], sin[p], interleaved)
        at = place(table, b, p, ps, pages)
        if at is not None:
            k_cache[at[0], :, at[1]] = kt
            v_cache[at[0], :, at[1]] = v[t]
            written[at] = True
    return q, k_cache, v_cache, written


def attention(q, k_cache, v_cache, table, seq_lens, cu_q, scale):
    """(O, L, A, dS): the results, and per element what error bounds are made of: A = sum p |v| / l
    and dS = the largest |scale| sum_d |q_d k_d| of a row's keys."""
    pages, nkv, ps, hs = k_cache.shape
    n, nh, _ = q.shape
    O, A = np.zeros((n, nh, hs)), np.zeros((n, nh, hs))
    L, dS = np.full((n, nh), -np.inf), np.zeros((n, nh))
    cap = len(table[0]) * ps if len(table) else 0
    for t, (b, _) in enumerate(positions(seq_lens, cu_q, n, cap)):
        # the positions behind a sequence's pages hold no key; a query there sees those in front
        keys = 0 if b < 0 else min(max(int(seq_lens[b]) - int(cu_q[b + 1]) + t + 1, 0), cap)
        at = [a for a in (place(table, b, j, ps, pages) for j in range(keys)) if a]
        if not at:
            continue
        page, row = np.array(at).T
        for h in range(nh):
            g = h // (nh // nkv)
            k, v = k_cache[page, g, row], v_cache[page, g, row]
            s = scale * (k @ q[t, h])
            m = s.max()
            e = np.exp(s - m)
            O[t, h], L[t, h] = (e @ v) / e.sum(), m + np.log(e.sum())
            A[t, h] = (e @ np.abs(v)) / e.sum()
            dS[t, h] = abs(scale) * (np.abs(k) @ np.abs(q[t, h])).max()
    return O, L, A, dS
