"""Performance cases of the operators that serve requests over a paged key/value cache, call by call.

Kinds (a case's ``"kind"``; its other entries are that kind's sizes and options):

``tables``     the bookkeeping of a step on the GPU: pages taken from the free list for the requests' new tokens, the
               block tables they extend, and each token's position and cache slot (``ops.paged_tables``)
``append``     one layer's q/k/v rows: RoPE of q and k, the new keys and values written to their cache slots
               (``ops.paged_rope_append``)
``attention``  one layer's attention of each request's new tokens over its pages (``ops.paged_attention``): one token
               (decode), a few (drafted tokens under verification), a chunk of a prompt, or requests of all these
``verify``     the drafted tokens of each request against the target's logits and given random numbers: how many
               stand, and the token that follows them (``ops.verify_draft``)

Head counts, head sizes, widths and vocabularies are those of the two decoder shapes the benchmark runs (14 / 2
heads of 64 with 151936 tokens, 32 / 8 heads of 128 with 128256 tokens), and generic ones beside them. The lengths
of a case's requests come from its own ``"lens"`` number, their order and every value from the seed.

Where ``own`` is false, ``run`` computes the same in elementary torch operations.
"""

from __future__ import annotations

import random

import numpy as np
import torch

own = False

BF16 = torch.bfloat16


# ----------------------------------------------------------------------------- the listed cases
def listed():
    return [
        # bookkeeping of one decode step of a few requests: the smallest call, latency and launches
        dict(name="tables_decode_8", kind="tables", requests=8, page=16, context=2048, new=1, lens=1),
        # bookkeeping of a busy server's step: prompt chunks beside decodes and idle rows, 16384 tokens at most
        dict(name="tables_chunks_256", kind="tables", requests=256, page=16, context=8192, new=64, lens=2),
        # the rows of a decode step of the 4096-wide decoder
        dict(name="append_decode_32", kind="append", heads=32, kv_heads=8, dim=128, page=16, tokens=32, positions=2304),
        # a 2048-token prompt chunk of the 4096-wide decoder
        dict(name="append_chunk_2048", kind="append", heads=32, kv_heads=8, dim=128, page=64, tokens=2048,
             positions=8192),
        # one request of the 896-wide decoder inside its 192-key bucket: latency and launches
        dict(name="attention_decode_1", kind="attention", heads=14, kv_heads=2, dim=64, page=16, requests=1,
             context=191, new=1, chunks=0, lens=3),
        # a decode step of 32 requests of very different lengths: the pages of all of them are read once
        dict(name="attention_decode_32", kind="attention", heads=32, kv_heads=8, dim=128, page=16, requests=32,
             context=8100, new=1, chunks=0, lens=4),
        # four drafted tokens and the one before them for each of 16 requests
        dict(name="attention_verify_16", kind="attention", heads=32, kv_heads=8, dim=128, page=32, requests=16,
             context=4000, new=5, chunks=0, lens=5),
        # decodes beside one 500-token prompt chunk, as a server that never stops for a prompt runs them
        dict(name="attention_mixed_25", kind="attention", heads=14, kv_heads=2, dim=64, page=16, requests=25,
             context=3000, new=500, chunks=1, lens=6),
        # one 2048-token chunk deep in a long prompt: matrix products
        dict(name="attention_chunk_2048", kind="attention", heads=32, kv_heads=8, dim=128, page=64, requests=1,
             context=6000, new=2048, chunks=1, lens=7),
        # one greedy request, three drafted tokens found in its own text: latency
        dict(name="verify_greedy_1", kind="verify", requests=1, drafts=3, vocab=151936, dtype="bf16", draft=False,
             temperature="greedy", lens=8),
        # 16 requests that sample, up to four drafted tokens found in their own text
        dict(name="verify_lookup_16", kind="verify", requests=16, drafts=4, vocab=151936, dtype="bf16", draft=False,
             temperature="sampled", lens=9),
        # 64 requests, some greedy, up to five drafted tokens of a draft model with its own logits
        dict(name="verify_draft_64", kind="verify", requests=64, drafts=5, vocab=128256, dtype="bf16", draft=True,
             temperature="mixed", lens=10),
    ]


def _log(rng, low, high):
    """A whole number spread over the logarithm of [low, high]."""

    return min(high, int(low * (high / low) ** rng.random() * (1 + 1e-9)))


def draw(rng):
    kind = rng.choice(["tables", "append", "attention", "attention", "attention", "verify", "verify"])
    lens = rng.randrange(1, 1 << 20)
    heads, kv_heads, dim = rng.choice([(14, 2, 64), (32, 8, 128), (32, 8, 64), (16, 16, 64), (28, 4, 128), (8, 1, 128)])
    page = rng.choice([8, 16, 16, 24, 32, 64, 128])
    if kind == "tables":
        requests = _log(rng, 1, 500)
        new = 1 if rng.random() < 0.3 else _log(rng, 1, max(1, min(1024, 16384 // requests)))
        return dict(kind=kind, requests=requests, page=page, context=_log(rng, 16, 8192), new=new, lens=lens)
    if kind == "append":
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, tokens=_log(rng, 1, 2048),
                    positions=_log(rng, 2100, 9000))
    if kind == "attention":
        form = rng.choice(["decode", "verify", "chunk", "mixed"])
        if form == "chunk":
            requests, new = rng.randrange(1, 4), _log(rng, 24, 680)
            return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests,
                        context=_log(rng, 16, 6000), new=new, chunks=requests, lens=lens)
        requests = _log(rng, 2, 16) if form == "mixed" else _log(rng, 1, 32)
        new = 1 if form == "decode" else rng.randrange(2, 9) if form == "verify" else _log(rng, 16, 300)
        return dict(kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, page=page, requests=requests,
                    context=_log(rng, 16, 8100 if form == "decode" else 4000), new=new,
                    chunks=1 if form == "mixed" else 0, lens=lens)
    return dict(kind=kind, requests=_log(rng, 1, 64), drafts=rng.randrange(1, 6), vocab=_log(rng, 1000, 128256),
                dtype=rng.choice(["bf16", "bf16", "f32"]), draft=rng.random() < 0.4,
                temperature=rng.choice(["greedy", "sampled", "sampled", "mixed"]), lens=lens)


# ----------------------------------------------------------------------------- lengths
def _lengths(case):
    """``(context, new)`` of each request: the case's alone."""

    rng = random.Random(case["lens"])
    if case["kind"] == "verify":
        # the token before the drafts, then 0 .. drafts of them; one request has them all
        new = [1 + (case["drafts"] if i == 0 else rng.randint(0, case["drafts"])) for i in range(case["requests"])]
        return [0] * len(new), new
    context = [_log(rng, max(1, case["context"] // 16), case["context"]) for _ in range(case["requests"])]
    context[0] = case["context"]
    if case["kind"] == "tables":
        # idle rows, decodes and chunks of all lengths
        new = [case["new"] if i == 0 else rng.choice([0, 1, rng.randint(1, case["new"]), case["new"]])
               for i in range(case["requests"])]
    elif case["chunks"] == 0 or case["chunks"] == case["requests"]:
        new = [case["new"]] * case["requests"]
    else:
        new = [case["new"] if i < case["chunks"] else 1 for i in range(case["requests"])]
    return context, new


def _shuffled(case, seed):
    pairs = list(zip(*_lengths(case)))
    random.Random(seed).shuffle(pairs)
    return [list(x) for x in zip(*pairs)]


def _ceil(a, b):
    return -(-a // b)


# ----------------------------------------------------------------------------- the inputs
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def prepare(case, seed):
    return {"tables": _prepare_tables, "append": _prepare_append, "attention": _prepare_attention,
            "verify": _prepare_verify}[case["kind"]](case, seed)


def _prepare_tables(case, seed):
    context, new = _shuffled(case, seed)
    rng = np.random.default_rng(seed)
    page, requests = case["page"], case["requests"]
    # a request may hold one page more than its tokens need: drafted tokens that did not stand
    counts = np.array([_ceil(c, page) for c in context]) + rng.integers(0, 2, requests)
    blocks = _ceil(case["context"] + case["new"], page) + 1
    tables = np.full((requests, blocks), -1, np.int32)
    pages = rng.permutation(int(counts.sum()) + requests * (_ceil(case["new"], page) + 1) + 64).astype(np.int32)
    held = np.arange(blocks)[None, :] < counts[:, None]
    tables[held] = pages[: counts.sum()]
    start = int(rng.integers(0, 32))
    free = np.concatenate([np.full(start, -1, np.int32), pages[counts.sum():]])
    return dict(case=case, context=_ints(context), new=_ints(new), tables=_ints(tables), counts=_ints(counts),
                free=_ints(free), start=_ints([start]), tokens=requests * case["new"])


def _pages(pool, kv_heads, page, dim, g):
    return (torch.randn((pool, kv_heads, page, dim), generator=g, device="cuda").to(BF16),
            torch.randn((pool, kv_heads, page, dim), generator=g, device="cuda").to(BF16))


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
    keys, values = _pages(pool, case["kv_heads"], page, dim, g)
    angle = torch.arange(case["positions"], device="cuda", dtype=torch.float64)[:, None] * (
        10000.0 ** (-2.0 * (torch.arange(dim, device="cuda", dtype=torch.float64) % (dim // 2)) / dim))
    width = (case["heads"] + 2 * case["kv_heads"]) * dim
    return dict(case=case, qkv=torch.randn((tokens, width), generator=g, device="cuda").to(BF16),
                positions=_ints(positions, torch.int64), slots=_ints(order, torch.int64), keys=keys, values=values,
                cos=angle.cos().to(BF16), sin=angle.sin().to(BF16))


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
    keys, values = _pages(pool, case["kv_heads"], page, case["dim"], g)
    q = torch.randn((sum(new), case["heads"], case["dim"]), generator=g, device="cuda").to(BF16)
    return dict(case=case, q=q, keys=keys, values=values, tables=_ints(tables),
                start=_ints(np.concatenate([[0], np.cumsum(new)])), kv=_ints(kv), longest=max(new),
                most=int(kv.max()))


def _prepare_verify(case, seed):
    _, new = _shuffled(case, seed)
    g, rng = _generator(seed), np.random.default_rng(seed)
    requests, drafts, vocab = case["requests"], case["drafts"], case["vocab"]
    dtype = BF16 if case["dtype"] == "bf16" else torch.float32
    start = np.concatenate([[0], np.cumsum(new)])
    # a model's logits: a wide bulk and a few far above it
    logits = torch.randn((sum(new), vocab), generator=g, device="cuda")
    logits = (2.0 * logits + 4.0 * (logits - 3.0).clamp(min=0)).to(dtype)
    greedy = {"greedy": np.ones(requests), "sampled": np.zeros(requests),
              "mixed": (np.arange(requests) % 3 == 0)}[case["temperature"]]
    temperature = np.where(greedy, 0.0, rng.uniform(0.6, 1.3, requests)).astype(np.float32)
    # the row that judges draft i of request r (the last row again where the request has fewer)
    row = np.minimum(start[:-1, None] + np.arange(drafts)[None, :], start[1:, None] - 1)
    judged = logits[_ints(row, torch.int64)].float()
    draft_logits = None
    if case["draft"]:
        draft_logits = (judged + torch.randn(judged.shape, generator=g, device="cuda")).to(dtype)
        heat = torch.tensor(temperature, device="cuda").clamp(min=0.05)[:, None, None]
        noise = torch.rand(judged.shape, generator=g, device="cuda").clamp(min=1e-20)
        tokens = (draft_logits.float() / heat - torch.log(-torch.log(noise))).argmax(-1)
    else:
        some = torch.randint(0, vocab, (requests, drafts), generator=g, device="cuda")
        tokens = torch.where(torch.rand((requests, drafts), generator=g, device="cuda") < 0.75, judged.argmax(-1), some)
    uniforms = torch.rand((requests, drafts + 1), generator=g, device="cuda")
    return dict(case=case, logits=logits, tokens=tokens.contiguous(), start=_ints(start), uniforms=uniforms,
                draft_logits=draft_logits, temperature=torch.tensor(temperature, device="cuda"))


# ----------------------------------------------------------------------------- one pass
def run(state):
    return {"tables": _run_tables, "append": _run_append, "attention": _run_attention,
            "verify": _run_verify}[state["case"]["kind"]](state)


def _run_tables(s):
    page = s["case"]["page"]
    if own:
        from aotolith_amd import ops

        # the entries that a step adds are the same at every call with the same lengths and counts
        step = ops.paged_tables(s["context"], s["new"], s["tables"], s["counts"], s["free"], s["start"],
                                page_size=page, max_tokens=s["tokens"])
        return dict(query_start=step.query_start, kv_lens=step.kv_lens, positions=step.positions, slots=step.slots,
                    tables=s["tables"], counts=step.page_counts, start=step.free_start)
    context, new, counts, tables = s["context"].long(), s["new"].long(), s["counts"].long(), s["tables"]
    start = torch.nn.functional.pad(torch.cumsum(new, 0), (1, 0))
    kv = context + new
    need = torch.maximum((kv + page - 1) // page, counts)
    taken = torch.cumsum(need - counts, 0)
    j = torch.arange(tables.shape[1], device=tables.device)[None, :]
    at = s["start"].long() + (taken - (need - counts))[:, None] + j - counts[:, None]
    fresh = s["free"][at.clamp(0, s["free"].numel() - 1)]
    tables = torch.where((j >= counts[:, None]) & (j < need[:, None]), fresh, tables)
    t = torch.arange(s["tokens"], device=tables.device)
    r = torch.searchsorted(start[1:], t, right=True).clamp(max=context.numel() - 1)
    real = t < start[-1]
    positions = torch.where(real, context[r] + t - start[r], 0)
    slots = torch.where(real, tables[r, positions // page].long() * page + positions % page, -1)
    return dict(query_start=start.int(), kv_lens=kv.int(), positions=positions, slots=slots, tables=tables,
                counts=need.int(), start=(s["start"].long() + taken[-1]).int())


def _run_append(s):
    c = s["case"]
    heads, kv_heads, dim, page = c["heads"], c["kv_heads"], c["dim"], c["page"]
    if own:
        from aotolith_amd import ops

        q = ops.paged_rope_append(s["qkv"], s["positions"], s["slots"], s["cos"], s["sin"], s["keys"], s["values"],
                                  query_heads=heads)
        return dict(q=q, keys=s["keys"], values=s["values"])
    x = s["qkv"].float().view(-1, heads + 2 * kv_heads, dim)
    cos, sin = s["cos"][s["positions"]].float()[:, None, :], s["sin"][s["positions"]].float()[:, None, :]
    turned = x[:, : heads + kv_heads]
    half = torch.cat([-turned[..., dim // 2:], turned[..., : dim // 2]], -1)
    turned = (turned * cos + half * sin).to(BF16)
    at = (s["slots"] // page, slice(None), s["slots"] % page)
    s["keys"][at] = turned[:, heads:]
    s["values"][at] = s["qkv"].view(-1, heads + 2 * kv_heads, dim)[:, heads + kv_heads:]
    return dict(q=turned[:, :heads], keys=s["keys"], values=s["values"])


def _run_attention(s):
    c = s["case"]
    if own:
        from aotolith_amd import ops

        # a server knows its requests' lengths; the bounds choose the launch, the lengths are read on the GPU
        return ops.paged_attention(s["q"], s["keys"], s["values"], s["tables"], s["start"], s["kv"],
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
    keys, values = (x[at].float().transpose(1, 2).contiguous() for x in (s["keys"], s["values"]))
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


def _run_verify(s):
    c = s["case"]
    if own:
        from aotolith_amd import ops

        tokens, accepted = ops.verify_draft(s["logits"], s["tokens"], s["start"], s["uniforms"],
                                            draft_logits=s["draft_logits"], temperature=s["temperature"])
        return dict(tokens=tokens, accepted=accepted)
    # 64 bits: a token is where a sum over the vocabulary passes a random number
    drafts, start, u, x = c["drafts"], s["start"].long(), s["uniforms"].double(), s["tokens"]
    requests = x.shape[0]
    r = torch.arange(requests, device="cuda")
    count = start[1:] - start[:-1] - 1
    greedy = s["temperature"] == 0
    heat = torch.where(greedy, 1.0, s["temperature"]).double()
    t = torch.arange(s["logits"].shape[0], device="cuda")
    owner = torch.searchsorted(start[1:], t, right=True)
    logits = s["logits"].double()
    p = torch.exp((logits - logits.amax(-1, keepdim=True)) / heat[owner][:, None])
    p /= p.sum(-1, keepdim=True)
    best = (logits == logits.amax(-1, keepdim=True)).int().argmax(-1)
    i = torch.arange(drafts, device="cuda")
    row = (start[:-1, None] + i).clamp(max=t.numel() - 1)
    there = i[None, :] < count[:, None]
    q = None
    chance = torch.ones((requests, drafts), dtype=torch.float64, device="cuda")
    if s["draft_logits"] is not None:
        z = s["draft_logits"].double()
        q = torch.exp((z - z.amax(-1, keepdim=True)) / heat[:, None, None])
        q /= q.sum(-1, keepdim=True)
        chance = q.gather(2, x[..., None])[..., 0]
    stands = torch.where(greedy[:, None], best[row] == x, u[:, :drafts] * chance < p[row, x]) & there
    accepted = torch.cumprod(stands.long(), 1).sum(1)
    last = start[:-1] + accepted
    at = accepted.clamp(max=drafts - 1)
    w = p[last]
    if q is None:
        rest = w.scatter(1, x[r, at][:, None], 0.0)
    else:
        rest = (w - q[r, at]).clamp(min=0)
    rest = torch.where((accepted < count)[:, None] & (rest.sum(-1, keepdim=True) > 0), rest, w)
    cdf = torch.cumsum(rest, -1)
    drawn = (cdf > u[:, drafts:] * cdf[:, -1:]).int().argmax(-1)
    follows = torch.where(greedy, best[last], drawn)
    k = torch.arange(drafts + 1, device="cuda")[None, :]
    padded = torch.nn.functional.pad(x, (0, 1))
    tokens = torch.where(k < accepted[:, None], padded, torch.where(k == accepted[:, None], follows[:, None], -1))
    return dict(tokens=tokens, accepted=accepted.int())


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    context, new = _lengths(case) if case["kind"] != "append" else (None, None)
    if case["kind"] == "tables":
        page = case["page"]
        fresh = sum(max(0, _ceil(c + n, page) - _ceil(c, page)) for c, n in zip(context, new))
        # the lengths and counts; taken pages read and entered; starts, lengths, counts; positions and slots
        return {"bytes": 24 * len(new) + 8 * fresh + 16 * case["requests"] * case["new"], "flops": 0}
    if case["kind"] == "append":
        row, tokens = 2 * case["dim"], case["tokens"]
        moved = 2 * (case["heads"] + 2 * case["kv_heads"]) + 2
        return {"bytes": tokens * (moved * row + 16),
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * case["dim"]}
    if case["kind"] == "attention":
        heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
        pairs = sum(n * c + n * (n + 1) // 2 for c, n in zip(context, new))
        keys = sum(c + n for c, n in zip(context, new))
        return {"bytes": 4 * keys * kv_heads * dim + 4 * sum(new) * heads * dim
                + 4 * sum(_ceil(c + n, case["page"]) for c, n in zip(context, new)),
                "flops": 4 * pairs * heads * dim}
    size = 2 if case["dtype"] == "bf16" else 4
    rows = sum(new)
    drafted = sum(new) - len(new) if case["draft"] else 0
    return {"bytes": (rows + drafted) * case["vocab"] * size + 20 * case["requests"] * (case["drafts"] + 1),
            "flops": 3 * (rows + drafted) * case["vocab"]}


# ----------------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    return {"tables": _exact_tables, "append": _exact_append, "attention": _exact_attention,
            "verify": _exact_verify}[case["kind"]](prepare(case, seed))


def _exact_tables(s):
    page = s["case"]["page"]
    context, new, counts = (s[k].tolist() for k in ("context", "new", "counts"))
    free, at = s["free"].tolist(), int(s["start"])
    tables = s["tables"].cpu().numpy().copy()
    start, positions, slots = [0], [], []
    for r, (c, n) in enumerate(zip(context, new)):
        while counts[r] * page < c + n:
            tables[r, counts[r]] = free[at]
            counts[r], at = counts[r] + 1, at + 1
        for position in range(c, c + n):
            positions.append(position)
            slots.append(int(tables[r, position // page]) * page + position % page)
        start.append(start[-1] + n)
    behind = s["tokens"] - len(slots)
    return dict(query_start=np.array(start, np.int32), kv_lens=np.array([c + n for c, n in zip(context, new)], np.int32),
                positions=np.array(positions + [0] * behind, np.int64), slots=np.array(slots + [-1] * behind, np.int64),
                tables=tables, counts=np.array(counts, np.int32), start=np.array([at], np.int32))


def _exact_append(s):
    c = s["case"]
    dim, half = c["dim"], c["dim"] // 2
    x = s["qkv"].double().reshape(s["qkv"].shape[0], -1, dim)
    cos, sin = s["cos"].double()[s["positions"]], s["sin"].double()[s["positions"]]
    low, high = x[..., :half], x[..., half:]
    turned = torch.empty_like(x)
    turned[..., :half] = low * cos[:, None, :half] - high * sin[:, None, :half]
    turned[..., half:] = high * cos[:, None, half:] + low * sin[:, None, half:]
    keys, values = s["keys"].double(), s["values"].double()
    for h in range(c["kv_heads"]):
        for cache, rows in ((keys, turned[:, c["heads"] + h]), (values, x[:, c["heads"] + c["kv_heads"] + h])):
            one = cache[:, h].reshape(-1, dim)
            one[s["slots"]] = rows
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
            keys = s["keys"][held, h].double().reshape(-1, dim)[:length]
            values = s["values"][held, h].double().reshape(-1, dim)[:length]
            for head in range(h * group, (h + 1) * group):
                score = s["q"][first: first + count, head].double() @ keys.T.contiguous() / dim ** 0.5
                out[first: first + count, head] = torch.softmax(score.masked_fill(~seen, -torch.inf), -1) @ values
    return out.reshape(-1, c["heads"] * dim)


def _exact_verify(s):
    c = s["case"]
    tokens = np.full((c["requests"], c["drafts"] + 1), -1, np.int64)
    accepted = np.zeros(c["requests"], np.int32)
    start, heat, u, x = (s[k].tolist() for k in ("start", "temperature", "uniforms", "tokens"))
    for r in range(c["requests"]):
        rows = s["logits"][start[r]: start[r + 1]].double().cpu().numpy()
        drafted = None if s["draft_logits"] is None else s["draft_logits"][r].double().cpu().numpy()

        def law(z):
            if heat[r] == 0:
                w = np.zeros_like(z)
                w[int(z.argmax())] = 1.0
                return w
            w = np.exp((z - z.max()) / heat[r])
            return w / w.sum()

        count = len(rows) - 1
        for i in range(count + 1):
            w = law(rows[i])
            if i == count:
                break
            q = np.zeros_like(w)
            if drafted is None or heat[r] == 0:
                q[x[r][i]] = 1.0
            else:
                q = law(drafted[i])
            if u[r][i] * q[x[r][i]] >= w[x[r][i]]:
                rest = np.maximum(w - q, 0.0)
                w = rest if rest.sum() > 0 else w
                break
            tokens[r, i] = x[r][i]
            accepted[r] = i + 1
        sums = np.cumsum(w)
        tokens[r, accepted[r]] = int(np.argmax(sums > u[r][c["drafts"]] * sums[-1]))
    return dict(tokens=tokens, accepted=accepted)
