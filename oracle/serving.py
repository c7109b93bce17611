"""Plain restatements, in 64 bits, of the operators over a 4-bit paged cache, on pages and on logits.

They have no counterpart in the reference; each follows the formulas at its entry point in ``include/aoto_hip.h``.
"""

from __future__ import annotations

import numpy as np

#: magnitudes of the codes 0 .. 7
MAGNITUDES = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def mx4_scale_byte(most):
    """The scale bytes of groups of these largest magnitudes."""

    most = np.asarray(most, np.float64)
    byte = np.full(most.shape, 255, np.int64)
    for i in np.ndindex(most.shape):
        if np.isfinite(most[i]):
            b = 1
            while b < 252 and most[i] > 7 * 2.0 ** (b - 127):
                b += 1
            byte[i] = b
    return byte


def mx4_pack(x):
    """f64 ``[..., D]`` -> ``(codes [..., D / 2], scale bytes [..., D / 32])``, uint8."""

    x = np.asarray(x, np.float64)
    groups = x.reshape(*x.shape[:-1], -1, 32)
    most = np.abs(groups).max(-1)
    byte = mx4_scale_byte(np.where(np.isnan(most), np.inf, most))
    bad = byte == 255
    size = np.where(bad[..., None], 0.0, np.abs(groups)) / 2.0 ** (byte - 127.0)[..., None]
    far = np.abs(size[..., None] - MAGNITUDES)
    nearest = far.min(-1, keepdims=True) == far
    even = nearest & (np.arange(8) % 2 == 0)
    code = np.where(even.any(-1), even.argmax(-1), nearest.argmax(-1))
    code = np.where(bad[..., None], 0, code | (np.signbit(groups) << 3)).reshape(x.shape)
    return (code[..., 0::2] | code[..., 1::2] << 4).astype(np.uint8), byte.astype(np.uint8)


def mx4_unpack(codes, scales):
    """f64 values of codes and scale bytes."""

    code = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    value = np.where(code & 8, -1.0, 1.0) * MAGNITUDES[code & 7]
    scale = np.where(scales > 252, np.nan, 2.0 ** (scales.astype(np.float64) - 127))
    return value * np.repeat(scale, 32, -1)


def fork(parents, lens, tables, counts, shares, free, start, page):
    """``(lens, counts, start, source, target, tables, shares, error)``."""

    requests, blocks = tables.shape
    before, tables, left, shares = tables, tables.copy(), shares.copy(), shares.copy()
    lens_out, counts_out = np.array(lens, np.int32), np.array(counts, np.int32)
    source, target = np.full(requests, -1, np.int32), np.full(requests, -1, np.int32)
    at, taken, error = max(int(start), 0), False, 0
    for r, p in enumerate(parents):
        if p >= requests or (p >= 0 and counts[r] > 0):
            error |= 64 if p >= requests else 32
            p = -1
        of = r if p < 0 else p
        n = min(max(int(lens[of]), 0), min(max(int(counts[of]), 0), blocks) * page)
        full = n // page
        if p < 0:
            # a row that stays: its page in progress is to be its own
            own = int(before[r, full]) if n % page else -1
            if 0 <= own < len(shares) and left[own] > 0:
                taken = True
                if at < len(free) and 0 <= free[at] < len(shares):
                    source[r], target[r], tables[r, full] = own, free[at], free[at]
                    shares[own] -= 1
                else:
                    error |= 2 | 512
                left[own] -= 1
                at = min(at + 1, max(len(free), at))
            continue
        tables[r, :full] = before[p, :full]
        for entry in before[p, :full]:
            if 0 <= entry < len(shares):
                shares[entry] += 1
        count = full
        if n % page:
            taken = True
            if at < len(free):
                source[r], target[r] = before[p, full], free[at]
                tables[r, full] = free[at]
                at, count = at + 1, full + 1
            else:
                error |= 2
                n = full * page
        lens_out[r], counts_out[r] = n, count
    return lens_out, counts_out, np.array([at if taken else start], np.int32), source, target, tables, shares, error


def release(keep, tables, counts, shares, free, start, page):
    """``(counts, start, free, shares, error)``."""

    counts_out, holders, free = np.array(counts, np.int32), shares.astype(np.int64) + 1, free.copy()
    for r, n in enumerate(keep):
        if n < 0:
            continue
        count = min(max(int(counts[r]), 0), tables.shape[1])
        stays = min(count, -(-int(n) // page))
        for entry in tables[r, stays:count]:
            if 0 <= entry < len(holders):
                holders[entry] -= 1
        counts_out[r] = stays
    at, error = min(max(int(start), 0), len(free)), 0
    listed = np.isin(np.arange(len(holders)), free[at:])
    if (listed & (holders <= 0)).any():               # given back before
        error |= 128
        holders[listed & (holders <= 0)] = 1
    gone = np.nonzero(holders <= 0)[0]
    for p in gone:
        error |= 128 if holders[p] < 0 else 0
        at -= 1
        if at >= 0:
            free[at] = p
        else:
            error |= 256
    holders[gone] = 1
    return (counts_out, np.array([max(at, 0) if len(gone) else start], np.int32), free, (holders - 1).astype(np.int32),
            error)


def compact(tables, counts, shares, free, start):
    """``(source, target, count, tables, shares, free, error)``."""

    tables, shares, free = tables.copy(), shares.copy(), free.copy()
    pages, first = len(shares), min(max(int(start), 0), len(free))
    rows = [min(max(int(n), 0), tables.shape[1]) for n in counts]
    held = {int(p) for r, n in enumerate(rows) for p in tables[r, :n] if 0 <= p < pages}
    spare = {int(p) for p in free[first:] if 0 <= p < pages}
    every = sorted(held | spare)
    low = every[: len(held)]
    source = [p for p in every[len(held):] if p in held]
    target = [p for p in low if p not in held]
    now = dict(zip(source, target))
    for a, b in now.items():
        shares[b], shares[a] = shares[a], 0
    for r, n in enumerate(rows):
        tables[r, :n] = [now.get(int(p), p) for p in tables[r, :n]]
    rest = every[len(held):]
    error = 128 if held & spare or first + len(rest) < len(free) else 0
    free[first: first + len(rest)] = rest
    free[first + len(rest):] = -1
    out = np.full((2, pages), -1, np.int32)
    out[0, : len(source)], out[1, : len(target)] = source, target
    return out[0], out[1], np.array([len(source)], np.int32), tables, shares, free, error


def adjust(logits, query_start=None, history=None, history_lens=None, prompt_lens=None, draft_tokens=None,
           repetition=None, presence=None, frequency=None, bias_tokens=None, bias_values=None, allowed=None):
    """``(out [T, V], sum of the terms' magnitudes, rows written [T])``."""

    rows, vocab = logits.shape
    out, size = logits.astype(np.float64), np.abs(logits.astype(np.float64))
    written = np.zeros(rows, bool)
    start = np.arange(rows + 1) if query_start is None else np.clip(query_start, 0, rows)
    for r in range(len(start) - 1):
        text = []
        if history is not None:
            n = history.shape[1] if history_lens is None else min(max(int(history_lens[r]), 0), history.shape[1])
            text = [int(x) for x in history[r, :n]]
        answer = text[max(0, int(prompt_lens[r])):] if prompt_lens is not None else list(text)
        bias = {}
        if bias_tokens is not None:
            bias = {int(x): float(b) for x, b in zip(bias_tokens[r], bias_values[r]) if 0 <= x < vocab}
        for t in range(start[r], max(start[r], start[r + 1])):
            written[t] = True
            i = t - start[r]
            drafts = [] if draft_tokens is None else [int(x) for x in draft_tokens[r, :i]]
            said = np.zeros(vocab)
            known = np.zeros(vocab, bool)
            for x in text + drafts:
                if 0 <= x < vocab:
                    known[x] = True
            for x in answer + drafts:
                if 0 <= x < vocab:
                    said[x] += 1
            z = out[t]
            if repetition is not None:
                f = float(repetition[r])
                z = np.where(known, np.where(z > 0, z / f, z * f), z)
            less = (0.0 if frequency is None else float(frequency[r])) * said
            less = less + (0.0 if presence is None else float(presence[r])) * (said > 0)
            z = z - less
            size[t] = np.abs(z) + 2 * np.abs(less) + size[t]
            for x, b in bias.items():
                z[x] += b
                size[t, x] += 2 * abs(b)
            if allowed is not None:
                bits = np.unpackbits(np.ascontiguousarray(allowed[t]).view(np.uint8), bitorder="little")[:vocab]
                z = np.where(bits == 0, -np.inf, z)
            out[t] = z
    return out, size, written
