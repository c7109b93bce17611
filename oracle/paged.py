"""Plain restatements, in 64 bits and request by request, of the operators over a paged key/value cache.

They have no counterpart in the reference; each follows the formulas at its entry point in ``include/aoto_hip.h``.
"""

from __future__ import annotations

import numpy as np


def tables(context, new, block_tables, counts, free, start, page, max_tokens):
    """``(query_start, kv_lens, positions, slots, block_tables, counts, start, error)`` of a step."""

    requests, blocks = block_tables.shape
    block_tables = block_tables.copy()
    query_start, kv_lens, counts_out = [0], [], []
    positions, slots = np.zeros(max_tokens, np.int64), np.full(max_tokens, -1, np.int64)
    at, error = max(int(start), 0), 0
    taken = False
    for r in range(requests):
        held = min(max(int(context[r]), 0), 2 ** 30)
        want = max(int(new[r]), 0)
        n = min(want, max_tokens - query_start[-1])
        error |= 1 if n < want else 0
        kv = held + n
        full = -(-kv // page)
        error |= 4 if full > blocks else 0
        count = min(max(int(counts[r]), 0), blocks)
        for j in range(count, max(count, min(full, blocks))):
            if at < len(free):
                block_tables[r, j] = free[at]
                at, count, taken = at + 1, count + 1, True
            else:
                block_tables[r, j] = -1
                error |= 2
        for i in range(n):
            t, position = query_start[-1] + i, held + i
            positions[t] = position
            block = position // page
            entry = int(block_tables[r, block]) if block < count else -1
            slots[t] = entry * page + position % page if entry >= 0 else -1
        query_start.append(query_start[-1] + n)
        kv_lens.append(kv)
        counts_out.append(count)
    return (np.array(query_start, np.int32), np.array(kv_lens, np.int32), positions, slots, block_tables,
            np.array(counts_out, np.int32), np.array([at if taken else start], np.int32), error)


def rope(x, cos, sin):
    """``(x * cos + rotate_half(x) * sin, |x * cos| + |rotate_half(x) * sin|)`` over the last dimension."""

    half = x.shape[-1] // 2
    other = np.concatenate([-x[..., half:], x[..., :half]], -1)
    return x * cos + other * sin, np.abs(x * cos) + np.abs(other * sin)


def attention(q, keys, values, block_tables, query_start, kv_lens, causal=True, scale=None):
    """``(out [T, Hq * D], sum_j p_j |v_j|, rows written [T])``; keys, values ``[P, Hkv, page, D]``."""

    tokens, heads, dim = q.shape
    pages, kv_heads, page, _ = keys.shape
    scale = dim ** -0.5 if scale is None else scale
    group = heads // kv_heads
    out, size = np.zeros((tokens, heads, dim)), np.zeros((tokens, heads, dim))
    written = np.zeros(tokens, bool)
    for r in range(len(kv_lens)):
        first, last = int(query_start[r]), int(query_start[r + 1])
        length = max(0, min(int(kv_lens[r]), block_tables.shape[1] * page))
        entries = block_tables[r, np.arange(length) // page]
        there = (entries >= 0) & (entries < pages)
        at = np.where(there, entries, 0)
        k = keys[at, :, np.arange(length) % page].astype(np.float64)   # [L, Hkv, D]
        v = values[at, :, np.arange(length) % page].astype(np.float64)
        for t in range(first, last):
            written[t] = True
            seen = there & (np.arange(length) <= int(kv_lens[r]) - (last - first) + (t - first)) if causal else there
            if not seen.any():
                continue
            for h in range(heads):
                score = scale * (k[seen, h // group] @ q[t, h].astype(np.float64))
                p = np.exp(score - score.max())
                p /= p.sum()
                out[t, h] = p @ v[seen, h // group]
                size[t, h] = p @ np.abs(v[seen, h // group])
    return out.reshape(tokens, -1), size.reshape(tokens, -1), written


def law(z, temperature):
    """The weights of a row of logits, normalized (all 0 for a row without a number above -inf)."""

    z = np.where(np.isnan(z), -np.inf, z.astype(np.float64))
    top = z.max()
    if top == -np.inf:
        return np.zeros_like(z)
    if not temperature > 0:
        w = np.zeros_like(z)
        w[int(np.argmax(z))] = 1.0
        return w
    if top == np.inf:  # shared by its equals, at every temperature
        w = (z == top).astype(np.float64)
    else:
        w = np.where(z == -np.inf, 0.0, np.exp((np.maximum(z, -1e300) - top) / np.float64(temperature)))
    return w / w.sum()


def verify(logits, draft_tokens, query_start, uniforms, draft_logits=None, temperature=None):
    """``(tokens [R, K + 1], accepted [R])``."""

    requests, drafts = draft_tokens.shape
    tokens = np.full((requests, drafts + 1), -1, np.int64)
    accepted = np.zeros(requests, np.int32)
    for r in range(requests):
        rows = logits[query_start[r]: query_start[r + 1]]
        heat = 0.0 if temperature is None else float(temperature[r])
        if not len(rows):
            continue
        count = min(len(rows) - 1, drafts)
        for i in range(count + 1):
            p = law(rows[i], heat)
            w = p
            if i == count:
                break
            x = int(draft_tokens[r, i])
            known = 0 <= x < len(p)
            if not heat > 0:
                stands = known and p[x] > 0
            elif draft_logits is None:
                stands = known and float(uniforms[r, i]) < p[x]
                w = p.copy()
                if known:
                    w[x] = 0.0
            else:
                q = law(draft_logits[r, i], heat)
                stands = known and float(uniforms[r, i]) * q[x] < p[x]
                w = np.maximum(p - q, 0.0)
            if not stands:
                w = w if w.sum() > 0 else p
                break
            tokens[r, i] = x
            accepted[r] = i + 1
        sums = np.cumsum(w)
        if sums[-1] > 0:
            above = np.nonzero(sums > float(uniforms[r, drafts]) * sums[-1])[0] if heat > 0 else [int(np.argmax(w))]
            tokens[r, accepted[r]] = above[0] if len(above) else np.nonzero(w)[0][-1]
        else:
            tokens[r, accepted[r]] = 0
    return tokens, accepted
