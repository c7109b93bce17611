"""Performance cases of the operators beside the paged cache's: a cache held in 4 bits, the pages' own upkeep, and what
is done to logits before drafts are verified.

Kinds (a case's ``"kind"``; its other entries are that kind's sizes and options):

``append``     one layer's q/k/v rows: RoPE of q and k, the new keys and values written to a 4-bit cache
               (``ops.paged_rope_append_mx4``), and that cache read back (``ops.paged_unpack_mx4``)
``attention``  one layer's attention of each request's new tokens over its pages of a 4-bit cache
               (``ops.paged_attention_mx4``): one token (decode), a few (drafted tokens), a chunk of a prompt, or all
``fork``       requests that go on in several ways: their full pages shared, the page in progress copied in all layers
               (``ops.paged_fork``, ``ops.paged_copy``)
``release``    requests that ended, and drafts that did not stand: their pages back to the free list
               (``ops.paged_release``)
``compact``    a pool whose requests came and went: the pages in use moved together (``ops.paged_compact``,
               ``ops.paged_copy``)
``logits``     penalties for repeated tokens, biases and grammar masks of each request's rows (``ops.adjust_logits``)

The 4-bit format: groups of 32 dims share a scale 2^(byte - 127), the smallest power of two of which the group's largest
magnitude is at most 7; a code is a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6, the nearest, ties to the even code.

Head counts, head sizes, layers and vocabularies are those of the two decoder shapes the benchmark runs (14 / 2 heads of
64, 24 layers, 151936 tokens; 32 / 8 heads of 128, 32 layers, 128256 tokens), and generic ones beside them. The lengths
of a case's requests come from its own ``"lens"`` number, their order and every value from the seed.

Where ``own`` is false, ``run`` computes the same in elementary torch operations.
"""

from __future__ import annotations

import random

import numpy as np
import torch

own = False

BF16 = torch.bfloat16
#: what the codes stand for, before their group's scale
VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


# ----------------------------------------------------------------------------- the listed cases
def listed():
    return [
        # the rows of a decode step of the 4096-wide decoder: latency and launches
        dict(name="append_decode_32", kind="append", heads=32, kv_heads=8, dim=128, page=16, tokens=32, positions=2304),
        # a 2048-token prompt chunk of the 4096-wide decoder
        dict(name="append_chunk_2048", kind="append", heads=32, kv_heads=8, dim=128, page=64, tokens=2048,
             positions=8192),
        # one request of the 896-wide decoder inside its 192-key bucket: the smallest call
        dict(name="attention_decode_1", kind="attention", heads=14, kv_heads=2, dim=64, page=16, requests=1,
             context=191, new=1, chunks=0, lens=3),
        # a decode step of 64 requests of very different lengths, up to the long ones a small cache is for
        dict(name="attention_decode_64", kind="attention", heads=32, kv_heads=8, dim=128, page=16, requests=64,
             context=16000, new=1, chunks=0, lens=4),
        # four drafted tokens and the one before them for each of 16 requests, beside one 300-token prompt chunk
        dict(name="attention_mixed_17", kind="attention", heads=14, kv_heads=2, dim=64, page=32, requests=17,
             context=4000, new=300, chunks=1, lens=5),
        # one 2048-token chunk deep in a long prompt: matrix products
        dict(name="attention_chunk_2048", kind="attention", heads=32, kv_heads=8, dim=128, page=64, requests=1,
             context=6000, new=2048, chunks=1, lens=6),
        # one prompt of the 896-wide decoder answered four times
        dict(name="fork_samples_4", kind="fork", kv_heads=2, dim=64, layers=24, page=16, requests=8, context=700,
             children=3, parents=1, lens=7),
        # beams of the 4096-wide decoder: 16 requests go on in four ways each, every layer's page in progress copied
        dict(name="fork_beams_64", kind="fork", kv_heads=8, dim=128, layers=32, page=16, requests=68, context=1000,
             children=48, parents=16, lens=8),
        # a busy server's step: requests that ended, drafts that fell, shared prompts among them
        dict(name="release_256", kind="release", page=16, requests=256, context=8192, lens=9),
        # a pool three quarters free after a busy hour, made small again
        dict(name="compact_pool", kind="compact", kv_heads=8, dim=128, layers=4, page=16, requests=32, context=1500,
             spare=3.0, lens=10),
        # one request with a long text behind it, three drafted tokens
        dict(name="logits_long_1", kind="logits", requests=1, drafts=3, vocab=151936, dtype="bf16", history=6000,
             biases=4, masked=False, lens=11),
        # 64 requests, up to four drafted tokens each, some held to a grammar
        dict(name="logits_grammar_64", kind="logits", requests=64, drafts=4, vocab=128256, dtype="bf16", history=2000,
             biases=16, masked=True, lens=12),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""

    return min(high, int(low * (high / low) ** rng.random() * (1 + 1e-9)))


def draw(rng):
    kind = rng.choice(["append", "attention", "attention", "attention", "fork", "release", "compact", "logits",
                       "logits"])
    lens = rng.randrange(1, 1 << 20)
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (32, 8, 128), (8, 8, 64), (28, 4, 128), (8, 1, 128), (16, 2, 64)])
    page = rng.choice([8, 16, 16, 20, 32, 64, 128])
    if kind == "append":
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, tokens=_log(rng, 1, 2048),
                    positions=_log(rng, 2100, 9000))
    if kind == "attention":
        form = rng.choice(["decode", "verify", "chunk", "mixed"])
        if form == "chunk":
            requests, new = rng.randrange(1, 4), _log(rng, 24, 680)
            return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests,
                        context=_log(rng, 16, 6000), new=new, chunks=requests, lens=lens)
        requests = _log(rng, 2, 16) if form == "mixed" else _log(rng, 1, 64)
        new = 1 if form == "decode" else rng.randrange(2, 9) if form == "verify" else _log(rng, 16, 300)
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests,
                    context=_log(rng, 16, 16000 if form == "decode" else 4000), new=new,
                    chunks=1 if form == "mixed" else 0, lens=lens)
    if kind == "fork":
        parents = _log(rng, 1, 16)
        children = _log(rng, 1, 48)
        return dict(kind=kind, kv_heads=kv_heads, dim=dim, layers=rng.randint(1, min(32, 512 // page)), page=page,
                    requests=parents + children + rng.randrange(0, 5), context=_log(rng, 8, 1000), children=children,
                    parents=parents, lens=lens)
    if kind == "release":
        return dict(kind=kind, page=page, requests=_log(rng, 1, 500), context=_log(rng, 16, 8192), lens=lens)
    if kind == "compact":
        return dict(kind=kind, kv_heads=kv_heads, dim=dim, layers=rng.randint(1, 4), page=page,
                    requests=_log(rng, 1, 32), context=_log(rng, 16, 1500), spare=rng.choice([0.5, 1.0, 2.0, 3.0]),
                    lens=lens)
    return dict(kind=kind, requests=_log(rng, 1, 64), drafts=rng.randrange(0, 5), vocab=_log(rng, 1000, 128256),
                dtype=rng.choice(["bf16", "bf16", "f32"]), history=_log(rng, 16, 2000), biases=_log(rng, 1, 100),
                masked=rng.random() < 0.5, lens=lens)


# ----------------------------------------------------------------------------- lengths
def _ceil(a, b):
    return -(-a // b)


def _lengths(case):
    """``(context, new)`` of each request; ``release``: what stays of it; ``fork``: its part. The case's alone."""

    rng = random.Random(case["lens"])
    kind, requests = case["kind"], case["requests"]
    if kind == "logits":
        # the token before the drafts, then 0 .. drafts of them; one request has them all
        new = [1 + (case["drafts"] if i == 0 else rng.randint(0, case["drafts"])) for i in range(requests)]
        context = [_log(rng, max(1, case["history"] // 16), case["history"]) for _ in new]
        context[0] = case["history"]
        return context, new
    context = [_log(rng, max(1, case["context"] // 16), case["context"]) for _ in range(requests)]
    context[0] = case["context"]
    if kind == "attention":
        if case["chunks"] == 0 or case["chunks"] == requests:
            return context, [case["new"]] * requests
        return context, [case["new"] if i < case["chunks"] else rng.choice([1, 5]) for i in range(requests)]
    if kind == "release":
        # what stays of each: nothing, all but a few drafted tokens, all
        return context, [rng.choice([0, max(1, n - rng.randint(0, 40)), n]) for n in context]
    if kind == "fork":
        parents, children = case["parents"], case["children"]
        role = [1] * parents + [2] * children + [0] * (requests - parents - children)
        return [0 if i == 2 else n for i, n in zip(role, context)], role
    return context, [0] * requests


def _shuffled(case, seed):
    pairs = list(zip(*_lengths(case)))
    random.Random(seed).shuffle(pairs)
    return [list(x) for x in zip(*pairs)]


# ----------------------------------------------------------------------------- the 4-bit format, in elementary steps
def _pack(x):
    """f32 ``[..., D]`` -> codes ``[..., D / 2]`` and scale bytes ``[..., D / 32]`` (uint8)."""

    grouped = x.float().unflatten(-1, (-1, 32))
    bits = grouped.abs().amax(-1).view(torch.int32)
    byte = ((bits + 0x1FFFFF) >> 23) - 2
    byte = byte.clamp(1, 252)
    size = (grouped / (byte << 23).view(torch.float32)[..., None]).abs()
    code = ((size > 0.25).int() + (size >= 0.75) + (size > 1.25) + (size >= 1.75) + (size > 2.5) + (size >= 3.5)
            + (size > 5.0)) | (grouped.signbit().int() << 3)
    code = code.flatten(-2)
    return (code[..., 0::2] | code[..., 1::2] << 4).to(torch.uint8), byte.to(torch.uint8)


def _unpack(codes, scales):
    """What codes and scale bytes stand for, f32 ``[..., D]``."""

    table = torch.tensor(VALUES, device=codes.device)
    both = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()
    scale = torch.exp2(scales.float() - 127.0)
    return (table[both].unflatten(-1, (-1, 32)) * scale[..., None]).flatten(-2)


# ----------------------------------------------------------------------------- the inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values, dtype=torch.int32):
    return torch.tensor(np.asarray(values), dtype=dtype, device="cuda")


def prepare(case, seed):
    return {"append": _prepare_append, "attention": _prepare_attention, "fork": _prepare_fork,
            "release": _prepare_release, "compact": _prepare_compact,
            "logits": _prepare_logits}[case["kind"]](case, seed)


def _cache4(pool, kv_heads, page, dim, g):
    """A pool of pages with keys and values of a model's spread: a few dims of the keys far larger than the rest."""

    wide = 1.0 + 4.0 * (torch.rand((kv_heads, 1, dim), generator=g, device="cuda") < 0.05)
    keys = _pack(torch.randn((pool, kv_heads, page, dim), generator=g, device="cuda") * wide)
    values = _pack(torch.randn((pool, kv_heads, page, dim), generator=g, device="cuda"))
    return dict(keys=keys[0], key_scales=keys[1], values=values[0], value_scales=values[1])


def _prepare_append(case, seed):
    g, rng = _generator(seed), np.random.default_rng(seed)
    tokens, page, dim = case["tokens"], case["page"], case["dim"]
    pool = 2 * _ceil(tokens, page) + 8
    if tokens <= 64:  # a decode step: one token of each request, wherever its last page has room
        order = rng.permutation(pool * page)[:tokens]
        positions = rng.integers(0, case["positions"], tokens)
    else:  # a chunk of one prompt: whole pages in the free list's order, from the middle of the first
        first = int(rng.integers(0, page))
        at = first + np.arange(tokens)
        order = rng.permutation(pool)[at // page] * page + at % page
        positions = int(rng.integers(0, case["positions"] - tokens)) + np.arange(tokens)
    angle = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * (
        10000.0 ** (-2.0 * (torch.arange(dim, device="cuda", dtype=torch.float64) % (dim // 2)) / dim))
    width = (case["heads"] + 2 * case["kv_heads"]) * dim
    return dict(case=case, qkv=torch.randn((tokens, width), generator=g, device="cuda").to(BF16),
                positions=_ints(positions, torch.int64), slots=_ints(order, torch.int64),
                cos=angle.cos().to(BF16), sin=angle.sin().to(BF16), **_cache4(pool, case["kv_heads"], page, dim, g))


def _prepare_attention(case, seed):
    context, new = _shuffled(case, seed)
    g, rng = _generator(seed), np.random.default_rng(seed)
    page, requests = case["page"], case["requests"]
    kv = np.array(context) + np.array(new)
    counts = (kv + page - 1) // page
    pool = int(counts.sum()) + 16
    blocks = _ceil(case["context"] + case["new"], page)
    tables = np.full((requests, blocks), -1, np.int32)
    tables[np.arange(blocks)[None, :] < counts[:, None]] = rng.permutation(pool)[: counts.sum()]
    q = torch.randn((sum(new), case["heads"], case["dim"]), generator=g, device="cuda").to(BF16)
    return dict(case=case, q=q, tables=_ints(tables), start=_ints(np.concatenate([[0], np.cumsum(new)])), kv=_ints(kv),
                longest=max(new), most=int(kv.max()), **_cache4(pool, case["kv_heads"], page, case["dim"], g))


def _held(case, context, rng, spare):
    """Tables of requests over a pool in no order: ``(tables, counts, free pages)``."""

    page = case["page"]
    counts = np.array([_ceil(c, page) for c in context])
    blocks = _ceil(case["context"], page) + 1
    pool = int(counts.sum()) + spare
    pages = rng.permutation(pool).astype(np.int32)
    tables = np.full((len(context), blocks), -1, np.int32)
    tables[np.arange(blocks)[None, :] < counts[:, None]] = pages[: counts.sum()]
    return tables, counts, pages[counts.sum():]


def _layers(case, pool, g):
    """Keys and values of all layers, bf16 ``[layers, 2, pages, Hkv, page, D]``."""

    return torch.randn((case["layers"], 2, pool, case["kv_heads"], case["page"], case["dim"]), generator=g,
                       device="cuda", dtype=BF16)


def _prepare_fork(case, seed):
    context, role = _shuffled(case, seed)  # rows in any order: parents (1), those that get one (2), others (0)
    rng = np.random.default_rng(seed)
    role = np.array(role)
    parents = np.full(case["requests"], -1, np.int32)
    parents[role == 2] = np.flatnonzero(role == 1)[np.arange(case["children"]) % case["parents"]]
    tables, counts, free = _held(case, context, rng, case["children"] + 16)
    start = int(rng.integers(0, 9))
    pool = int(counts.sum()) + free.size
    free = np.concatenate([np.full(start, -1, np.int32), free, np.full(8 - start, -1, np.int32)])
    return dict(case=case, parents=_ints(parents), lens=_ints(context), tables=_ints(tables), counts=_ints(counts),
                shares=torch.zeros(pool, dtype=torch.int32, device="cuda"), free=_ints(free), start=_ints([start]),
                cache=_layers(case, pool, _generator(seed)))


def _prepare_pool(case, context, rng, spare):
    """A pool with shared prompts: tables, counts, shares, the free list at the end of a pool's room, its start."""

    tables, counts, free = _held(case, context, rng, spare)
    pool = int(counts.sum()) + free.size
    shares = np.zeros(pool, np.int32)
    # a fifth of the requests began from another's prompt: its first pages are theirs too, their own are nobody's
    for r in range(1, case["requests"]):
        if r % 5 == 0:
            n = min(counts[r], counts[r - 1]) // 2
            free = np.concatenate([free, tables[r, :n]])
            tables[r, :n] = tables[r - 1, :n]
            np.add.at(shares, tables[r, :n], 1)
    free = np.concatenate([np.full(pool - free.size, -1, np.int32), free])
    return dict(tables=_ints(tables), counts=_ints(counts), shares=_ints(shares), free=_ints(free),
                start=_ints([int((free < 0).sum())]))


def _prepare_release(case, seed):
    context, keep = _shuffled(case, seed)
    return dict(case=case, keep=_ints(keep),
                **_prepare_pool(case, context, np.random.default_rng(seed), 64 + 2 * case["requests"]))


def _prepare_compact(case, seed):
    context, _ = _shuffled(case, seed)
    in_use = sum(_ceil(c, case["page"]) for c in context)
    pool = _prepare_pool(case, context, np.random.default_rng(seed), int(in_use * case["spare"]) + 1)
    return dict(case=case, cache=_layers(case, pool["shares"].numel(), _generator(seed)), **pool)


def _prepare_logits(case, seed):
    context, new = _shuffled(case, seed)
    g, rng = _generator(seed), np.random.default_rng(seed)
    requests, vocab, drafts = case["requests"], case["vocab"], case["drafts"]
    rows = sum(new)
    dtype = BF16 if case["dtype"] == "bf16" else torch.float32
    logits = torch.randn((rows, vocab), generator=g, device="cuda")
    logits = (2.0 * logits + 4.0 * (logits - 3.0).clamp(min=0)).to(dtype)
    # a text's tokens: most of them few and frequent
    longest = max(context)
    history, draft = (torch.rand((requests, n), generator=g, device="cuda").pow(4.0).mul(vocab).long()
                      .clamp(max=vocab - 1) for n in (longest, drafts))
    biases = min(case["biases"], vocab)
    tokens = np.stack([rng.choice(vocab, biases, replace=False) for _ in range(requests)])
    tokens[rng.random(tokens.shape) < 0.2] = -1  # requests have lists of their own length
    allowed = None
    if case["masked"]:
        words = _ceil(vocab, 32)
        allowed = torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device="cuda").int()
        allowed &= torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device="cuda").int()
        allowed[torch.rand(rows, generator=g, device="cuda") < 0.5] = -1  # no grammar
    uniform = lambda low, high: _ints(rng.uniform(low, high, requests), torch.float32)  # noqa: E731
    return dict(case=case, logits=logits, start=_ints(np.concatenate([[0], np.cumsum(new)])), history=history,
                lens=_ints(context), prompts=_ints([int(c * f) for c, f in zip(context, rng.random(requests))]),
                drafts=draft, repetition=uniform(1.0, 1.4), presence=uniform(0.0, 0.8), frequency=uniform(0.0, 0.3),
                bias_tokens=_ints(tokens, torch.int64),
                bias_values=torch.randn((requests, biases), generator=g, device="cuda") * 4.0, allowed=allowed)


# ----------------------------------------------------------------------------- one pass
def run(state):
    return {"append": _run_append, "attention": _run_attention, "fork": _run_fork, "release": _run_release,
            "compact": _run_compact, "logits": _run_logits}[state["case"]["kind"]](state)


def _own_cache(s):
    from aotolith_amd import ops

    return ops.PagedMx4(s["keys"], s["values"], s["key_scales"], s["value_scales"])


def _run_append(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if own:
        from aotolith_amd import ops

        cache = _own_cache(s)
        q = ops.paged_rope_append_mx4(s["qkv"], s["positions"], s["slots"], s["cos"], s["sin"], cache,
                                      query_heads=heads)
        keys, values = ops.paged_unpack_mx4(cache)
        return dict(q=q, keys=keys, values=values)
    x = s["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    cos, sin = s["cos"][s["positions"]].float()[:, None, :], s["sin"][s["positions"]].float()[:, None, :]
    turned = x[:, : heads + kv_heads]
    half = torch.cat([-turned[..., dim // 2:], turned[..., : dim // 2]], -1)
    turned = turned * cos + half * sin
    at = (s["slots"] // page, slice(None), s["slots"] % page)
    s["keys"][at], s["key_scales"][at] = _pack(turned[:, heads:])
    s["values"][at], s["value_scales"][at] = _pack(x[:, heads + kv_heads:])
    return dict(q=turned[:, :heads].to(BF16), keys=_unpack(s["keys"], s["key_scales"]).to(BF16),
                values=_unpack(s["values"], s["value_scales"]).to(BF16))


def _run_attention(s):
    c = s["case"]
    if own:
        from aotolith_amd import ops

        # a server knows its requests' lengths; the bounds choose the launch, the lengths are read on the GPU
        return ops.paged_attention_mx4(s["q"], _own_cache(s), s["tables"], s["start"], s["kv"],
                                       max_query_len=s["longest"], max_kv_len=s["most"])
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    start, kv, tokens = s["start"].long(), s["kv"].long(), s["q"].shape[0]
    new = start[1:] - start[:-1]
    # every request padded to the longest: [R, Hkv, G * N, D] against [R, Hkv, L, D]
    i = torch.arange(s["longest"], device="cuda")
    q = s["q"][(start[:-1, None] + i).clamp(max=tokens - 1)].float()
    q = q.view(-1, i.numel(), kv_heads, heads // kv_heads, dim).permute(0, 2, 3, 1, 4)
    j = torch.arange(s["most"], device="cuda")
    at = (s["tables"].long().clamp(min=0)[:, j // page], slice(None), j % page)
    keys, values = (_unpack(s[x][at], s[y][at]).transpose(1, 2).contiguous()
                    for x, y in (("keys", "key_scales"), ("values", "value_scales")))
    flat = q.reshape(q.shape[0], kv_heads, -1, dim)
    score = torch.matmul(flat, keys.transpose(2, 3).contiguous()) * dim ** -0.5
    del keys
    score = score.view(*q.shape[:4], j.numel())
    keep = j[None, None, :] <= (kv - new)[:, None, None] + i[None, :, None]
    score = score.masked_fill(~keep[:, None, None], float("-inf"))
    p = torch.exp(score - score.amax(-1, keepdim=True))
    del score
    out = torch.matmul(p.view(*flat.shape[:3], -1), values) / p.sum(-1).view(*flat.shape[:3], 1)
    out = out.view(q.shape).permute(0, 3, 1, 2, 4).reshape(-1, i.numel(), heads * dim).to(BF16)
    t = torch.arange(tokens, device="cuda")
    r = torch.searchsorted(start[1:], t, right=True)
    return out[r, t - start[r]]


def _run_fork(s):
    page, cache = s["case"]["page"], s["cache"]
    if own:
        from aotolith_amd import ops

        # lengths, counts and the list's start come back in tensors of their own: the same pages at every pass
        fork = ops.paged_fork(s["parents"], s["lens"], s["tables"], s["counts"], s["shares"], s["free"], s["start"],
                              page_size=page)
        ops.paged_copy(cache, fork.source, fork.target, dim=2)
        return dict(lens=fork.context_lens, counts=fork.page_counts, start=fork.free_start, source=fork.source,
                    target=fork.target, tables=s["tables"], shares=s["shares"], cache=cache)
    parents, lens, counts, tables = s["parents"].long(), s["lens"].long(), s["counts"].long(), s["tables"]
    of = parents.clamp(min=0)
    child = (parents >= 0) & (counts == 0)
    length = torch.where(child, torch.minimum(lens[of], counts[of] * page), 0)
    full, part = length // page, length % page > 0
    fresh = s["free"][s["start"].long() + torch.cumsum(part.long(), 0) - part.long()]
    j = torch.arange(tables.shape[1], device="cuda")[None, :]
    theirs = tables[of]
    shared = j < full[:, None]
    begun = part[:, None] & (j == full[:, None])
    source = torch.where(part, theirs.gather(1, full[:, None])[:, 0], -1)
    target = torch.where(part, fresh, -1)
    tables.copy_(torch.where(shared, theirs, torch.where(begun, fresh[:, None], tables)))
    s["shares"].scatter_add_(0, theirs.clamp(min=0).long().flatten(), shared.int().flatten())
    # rows that copy nothing repeat one that does
    one = part.long().argmax()
    cache[:, :, torch.where(part, target, target[one]).long()] = \
        cache[:, :, torch.where(part, source, source[one]).long()]
    return dict(lens=torch.where(child, length, lens).int(), counts=torch.where(child, full + part, counts).int(),
                start=(s["start"] + part.sum()).int(), source=source.int(), target=target.int(), tables=tables,
                shares=s["shares"], cache=cache)


def _run_release(s):
    page = s["case"]["page"]
    if own:
        from aotolith_amd import ops

        # counts and the list's start come back in tensors of their own: the same pages are given back at every pass
        counts, start = ops.paged_release(s["keep"], s["tables"], s["counts"], s["shares"], s["free"], s["start"],
                                          page_size=page)
        return dict(counts=counts, start=start, free=s["free"], shares=s["shares"])
    counts, keep, tables, free = s["counts"].long(), s["keep"].long(), s["tables"], s["free"]
    stays = torch.where(keep < 0, counts, torch.minimum((keep + page - 1) // page, counts))
    j = torch.arange(tables.shape[1], device="cuda")[None, :]
    dropped = (j >= stays[:, None]) & (j < counts[:, None])
    held = s["shares"].scatter_add(0, tables.clamp(min=0).long().flatten(), -dropped.int().flatten())
    freed = held < 0
    at = torch.where(freed, s["start"].long() - torch.cumsum(freed.long(), 0), free.numel())
    pages = torch.arange(held.numel(), dtype=torch.int32, device="cuda")
    free.copy_(torch.nn.functional.pad(free, (0, 1)).scatter(0, at, pages)[:-1])
    s["shares"].copy_(held.clamp(min=0))
    return dict(counts=stays.int(), start=(s["start"] - freed.sum()).int(), free=free, shares=s["shares"])


def _run_compact(s):
    cache = s["cache"]
    # kept as they are, so that the pass can be repeated
    tables, shares, free = s["tables"].clone(), s["shares"].clone(), s["free"].clone()
    if own:
        from aotolith_amd import ops

        moves = ops.paged_compact(tables, s["counts"], shares, free, s["start"])
        ops.paged_copy(cache, moves.source, moves.target, count=moves.count, dim=2)
        return dict(source=moves.source, target=moves.target, count=moves.count, tables=tables, shares=shares,
                    free=free, cache=cache)
    pages, start = shares.numel(), s["start"].long()
    j = torch.arange(tables.shape[1], device="cuda")[None, :]
    entries = j < s["counts"].long()[:, None]
    held = torch.zeros(pages, dtype=torch.bool, device="cuda")
    held[tables[entries].long()] = True
    spare = torch.zeros(pages, dtype=torch.bool, device="cuda")
    spare[free[start:].long()] = True
    place = torch.cumsum((held | spare).long(), 0) - 1
    first = place < held.sum()
    page = torch.arange(pages, dtype=torch.int32, device="cuda")
    movers, holes = page[held & ~first], page[spare & first]
    now = page.clone()
    now[movers.long()] = holes
    tables[entries] = now[tables[entries].long()]
    behind = (held | spare) & ~first
    free[start + place[behind] - held.sum()] = page[behind]
    shares[holes.long()] = shares[movers.long()]
    shares[movers.long()] = 0
    cache[:, :, holes.long()] = cache[:, :, movers.long()]
    source, target = (torch.nn.functional.pad(x, (0, pages - x.numel()), value=-1) for x in (movers, holes))
    return dict(source=source, target=target,
                count=_ints([movers.numel()]), tables=tables, shares=shares, free=free, cache=cache)


def _run_logits(s):
    if own:
        from aotolith_amd import ops

        return ops.adjust_logits(s["logits"], s["start"], history=s["history"], history_lens=s["lens"],
                                 prompt_lens=s["prompts"], draft_tokens=s["drafts"], repetition=s["repetition"],
                                 presence=s["presence"], frequency=s["frequency"], bias_tokens=s["bias_tokens"],
                                 bias_values=s["bias_values"], allowed=s["allowed"])
    logits, start, drafts = s["logits"], s["start"].long(), s["drafts"]
    rows, vocab = logits.shape
    requests = start.numel() - 1
    t = torch.arange(rows, device="cuda")
    r = torch.searchsorted(start[1:], t, right=True)
    j = torch.arange(s["history"].shape[1], device="cuda")[None, :]
    told = j < s["lens"].long()[:, None]
    seen = torch.zeros((requests, vocab), dtype=torch.int32, device="cuda")
    seen.scatter_add_(1, s["history"], told.int())
    said = torch.zeros((requests, vocab), dtype=torch.int32, device="cuda")
    said.scatter_add_(1, s["history"], (told & (j >= s["prompts"].long()[:, None])).int())
    before = (torch.arange(drafts.shape[1], device="cuda")[None, :] < (t - start[r])[:, None]).int()
    seen = seen[r].scatter_add(1, drafts[r], before)
    said = said[r].scatter_add(1, drafts[r], before)
    z = logits.float()
    times = s["repetition"][r][:, None]
    z = torch.where(seen > 0, torch.where(z > 0, z / times, z * times), z)
    z = z - s["frequency"][r][:, None] * said - s["presence"][r][:, None] * (said > 0)
    bias = torch.zeros((requests, vocab + 1), device="cuda")
    bias.scatter_(1, torch.where(s["bias_tokens"] < 0, vocab, s["bias_tokens"]), s["bias_values"])
    z = z + bias[r, :vocab]
    if s["allowed"] is not None:
        v = torch.arange(vocab, device="cuda")
        z = z.masked_fill((s["allowed"][:, v // 32] >> (v % 32) & 1) == 0, float("-inf"))
    return z.to(logits.dtype)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["kind"] == "append":
        heads, kv_heads, dim, tokens = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
        packed = dim // 2 + dim // 32
        # rows in, q out, table rows and maps, codes written; then the pool read and its values written
        pool = (2 * _ceil(tokens, case["page"]) + 8) * case["page"]
        return {"bytes": tokens * (2 * dim * (2 * heads + 2 * kv_heads + 2) + 2 * kv_heads * packed + 16)
                + 2 * pool * kv_heads * (packed + 2 * dim),
                "flops": 3 * tokens * (heads + kv_heads) * dim}
    context, new = _lengths(case)
    if case["kind"] == "attention":
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(context, new))
        keys = sum(c + n for c, n in zip(context, new))
        return {"bytes": keys * kv_heads * (dim + dim // 16) + 4 * sum(new) * heads * dim
                + 4 * sum(_ceil(c + n, case["page"]) for c, n in zip(context, new)),
                "flops": 4 * pairs * heads * dim}
    if case["kind"] == "fork":
        # each child: its row read and written, its pages' shares, one page of every layer copied
        page = case["page"]
        entries = sum(context[i % case["parents"]] // page for i in range(case["children"]))
        data = 4 * case["layers"] * case["kv_heads"] * page * case["dim"]
        return {"bytes": 16 * entries + 28 * case["requests"] + 2 * case["children"] * data, "flops": 0}
    if case["kind"] == "release":
        gone = sum(_ceil(c, case["page"]) - min(_ceil(k, case["page"]), _ceil(c, case["page"]))
                   for c, k in zip(context, new))
        pool = sum(_ceil(c, case["page"]) for c in context) + 64 + 2 * case["requests"]
        return {"bytes": 4 * gone + 8 * pool + 16 * len(new), "flops": 0}
    if case["kind"] == "compact":
        # the tables read and written, marks, lists and shares of the pool; about spare / (1 + spare) of the pages move
        in_use = sum(_ceil(c, case["page"]) for c in context)
        pool = in_use + int(in_use * case["spare"]) + 1
        data = 4 * case["layers"] * case["kv_heads"] * case["page"] * case["dim"]
        moved = int(in_use * case["spare"] / (1 + case["spare"]))
        return {"bytes": 8 * in_use + 24 * pool + 2 * moved * data, "flops": 0}
    size = 2 if case["dtype"] == "bf16" else 4
    rows, vocab = sum(new), case["vocab"]
    return {"bytes": 2 * rows * vocab * size + (rows * 4 * _ceil(vocab, 32) if case["masked"] else 0)
            + 8 * sum(context) + 12 * len(new) * case["biases"], "flops": 4 * rows * vocab}


# ----------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    return {"append": _exact_append, "attention": _exact_attention, "fork": _exact_fork, "release": _exact_release,
            "compact": _exact_compact, "logits": _exact_logits}[case["kind"]](prepare(case, seed))


def _stands_for(codes, scales):
    """f64 values of codes and scale bytes, dim by dim."""

    table = torch.tensor(VALUES, dtype=torch.float64, device=codes.device)
    out = torch.empty((*codes.shape[:-1], 2 * codes.shape[-1]), dtype=torch.float64, device=codes.device)
    out[..., 0::2], out[..., 1::2] = table[(codes % 16).long()], table[(codes // 16).long()]
    for g in range(scales.shape[-1]):
        out[..., 32 * g: 32 * g + 32] *= torch.pow(2.0, scales[..., g: g + 1].double() - 127)
    return out


def _nearest(x):
    """The nearest values of the format to f64 ``x [..., D]``: the distance to each, the even code where two tie."""

    x = x.unflatten(-1, (-1, 32))
    most = x.abs().amax(-1, keepdim=True)
    scale = torch.pow(2.0, torch.ceil(torch.log2(most / 7)).clamp(-126, 125))
    # the logarithm's own rounding, next to a power of two
    scale = torch.where(most > 7 * scale, 2 * scale, torch.where(most <= 3.5 * scale, scale / 2, scale))
    scale = scale.clamp(2.0 ** -126, 2.0 ** 125)
    size = x.abs() / scale
    best, far = torch.zeros_like(size), size.clone()
    for code in (2, 4, 6, 1, 3, 5, 7):  # an odd one has to be nearer
        off = (size - VALUES[code]).abs()
        nearer = off < far if code % 2 else off <= far
        best, far = torch.where(nearer, VALUES[code], best), torch.where(nearer, off, far)
    return (torch.copysign(best, x) * scale).flatten(-2)


def _exact_append(s):
    c = s["case"]
    dim, half = c["dim"], c["dim"] // 2
    x = s["qkv"].double().reshape(s["qkv"].shape[0], -1, dim)
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
    low, high = x[..., :half], x[..., half:]
    turned = torch.empty_like(x)
    turned[..., :half] = low * cos[:, None, :half] - high * sin[:, None, :half]
    turned[..., half:] = high * cos[:, None, half:] + low * sin[:, None, half:]
    keys, values = _stands_for(s["keys"], s["key_scales"]), _stands_for(s["values"], s["value_scales"])
    for h in range(c["kv_heads"]):
        for cache, rows in ((keys, turned[:, c["heads"] + h]), (values, x[:, c["heads"] + c["kv_heads"] + h])):
            one = cache[:, h].reshape(-1, dim)
            one[s["slots"]] = _nearest(rows)
            cache[:, h] = one.view(cache.shape[0], -1, dim)
    return dict(q=turned[:, : c["heads"]].contiguous(), keys=keys, values=values)


def _exact_attention(s):
    c = s["case"]
    group, page, dim = c["heads"] // c["kv_heads"], c["page"], c["dim"]
    out = torch.zeros((s["q"].shape[0], c["heads"], dim), dtype=torch.float64, device="cuda")
    start, kv = s["start"].tolist(), s["kv"].tolist()
    for r, length in enumerate(kv):
        first, count = start[r], start[r + 1] - start[r]
        held = s["tables"][r, : _ceil(length, page)].long()
        seen = torch.arange(length, device="cuda")[None, :] < torch.arange(length - count + 1, length + 1,
                                                                            device="cuda")[:, None]
        for h in range(c["kv_heads"]):
            keys = _stands_for(s["keys"][held, h], s["key_scales"][held, h]).reshape(-1, dim)[:length]
            values = _stands_for(s["values"][held, h], s["value_scales"][held, h]).reshape(-1, dim)[:length]
            for head in range(h * group, (h + 1) * group):
                score = s["q"][first: first + count, head].double() @ keys.T.contiguous() / dim ** 0.5
                out[first: first + count, head] = torch.softmax(score.masked_fill(~seen, -torch.inf), -1) @ values
    return out.reshape(-1, c["heads"] * dim)


def _exact_fork(s):
    page = s["case"]["page"]
    parents, lens, counts, free = (s[k].tolist() for k in ("parents", "lens", "counts", "free"))
    tables, shares = s["tables"].cpu().numpy(), s["shares"].cpu().numpy()
    cache, at = s["cache"].clone(), int(s["start"])
    old_lens, old_counts, old = list(lens), list(counts), tables.copy()
    source, target = [-1] * len(parents), [-1] * len(parents)
    for r, p in enumerate(parents):
        if p < 0 or old_counts[r]:
            continue
        lens[r] = min(old_lens[p], old_counts[p] * page)
        for block in range(_ceil(lens[r], page)):
            if (block + 1) * page <= lens[r]:
                tables[r, block] = old[p, block]
                shares[old[p, block]] += 1
            else:
                source[r], target[r] = int(old[p, block]), free[at]
                tables[r, block] = free[at]
                cache[:, :, target[r]] = s["cache"][:, :, source[r]]
                at += 1
        counts[r] = _ceil(lens[r], page)
    i32 = lambda x: np.array(x, np.int32)  # noqa: E731
    return dict(lens=i32(lens), counts=i32(counts), start=i32([at]), source=i32(source), target=i32(target),
                tables=tables, shares=shares, cache=cache.double() if cache.numel() < 1 << 30 else None)


def _exact_release(s):
    page = s["case"]["page"]
    keep, counts, free = (s[k].tolist() for k in ("keep", "counts", "free"))
    tables, holders, at = s["tables"].tolist(), [x + 1 for x in s["shares"].tolist()], int(s["start"])
    gone = set()
    for r, n in enumerate(counts):
        while keep[r] >= 0 and (counts[r] - 1) * page >= keep[r] and counts[r]:
            counts[r] -= 1
            holders[tables[r][counts[r]]] -= 1
            gone.add(tables[r][counts[r]])
    for p in sorted(p for p in gone if holders[p] == 0):
        at, holders[p] = at - 1, 1
        free[at] = p
    i32 = lambda x: np.array(x, np.int32)  # noqa: E731
    return dict(counts=i32(counts), start=i32([at]), free=i32(free), shares=i32([x - 1 for x in holders]))


def _exact_compact(s):
    counts, free, start = s["counts"].tolist(), s["free"].tolist(), int(s["start"])
    tables, shares = s["tables"].cpu().numpy().copy(), s["shares"].cpu().numpy().copy()
    held = sorted({int(tables[r, b]) for r, n in enumerate(counts) for b in range(n)})
    every = sorted(held + free[start:])
    low = set(every[: len(held)])
    source = [p for p in held if p not in low]
    target = [p for p in every[: len(held)] if p not in set(held)]
    now = dict(zip(source, target))
    cache = s["cache"].clone()
    for a, b in now.items():
        shares[b], shares[a] = shares[a], 0
        cache[:, :, b] = s["cache"][:, :, a]
    for r, n in enumerate(counts):
        for b in range(n):
            tables[r, b] = now.get(int(tables[r, b]), tables[r, b])
    free[start:] = every[len(held):]
    i32 = lambda x: np.array(x, np.int32)  # noqa: E731
    pad = [-1] * (shares.size - len(source))
    return dict(source=i32(source + pad), target=i32(target + pad), count=i32([len(source)]), tables=tables,
                shares=shares, free=i32(free), cache=cache.double() if cache.numel() < 1 << 30 else None)


def _exact_logits(s):
    start, lens, prompts = (s[k].tolist() for k in ("start", "lens", "prompts"))
    out = s["logits"].double()
    vocab = out.shape[1]
    for r in range(len(lens)):
        times, presence, frequency = (float(s[k][r]) for k in ("repetition", "presence", "frequency"))
        bias = torch.zeros(vocab, dtype=torch.float64, device="cuda")
        listed_ = s["bias_tokens"][r] >= 0
        bias[s["bias_tokens"][r][listed_]] = s["bias_values"][r][listed_].double()
        for t in range(start[r], start[r + 1]):
            drafts = s["drafts"][r, : t - start[r]]
            text = torch.cat([s["history"][r, : lens[r]], drafts])
            said = torch.bincount(torch.cat([s["history"][r, prompts[r]: lens[r]], drafts]), minlength=vocab).double()
            known = torch.bincount(text, minlength=vocab) > 0
            z = out[t]
            z = torch.where(known, torch.where(z > 0, z / times, z * times), z)
            z = z - frequency * said - presence * (said > 0) + bias
            if s["allowed"] is not None:
                words = s["allowed"][t].cpu().numpy().view(np.uint32)
                bits = np.unpackbits(words.view(np.uint8), bitorder="little")[:vocab]
                z[torch.from_numpy(bits == 0).cuda()] = -torch.inf
            out[t] = z
    return out
