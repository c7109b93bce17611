"""GPU parity of the operators over a paged key/value cache with their 64-bit restatements (``oracle/paged.py``)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as oracle
from tests.helpers import bf16_normal, from_gpu_bf16, to_gpu_bf16

pytestmark = pytest.mark.gpu

HALF = 2.0 ** -8  # a rounding to bf16, relative to the value: half a step of 2^-7


def _ops():
    from aotolith_amd import ops

    return ops


def _i32(values):
    return torch.tensor(np.asarray(values, np.int32), device="cuda")


def _i64(values):
    return torch.tensor(np.asarray(values, np.int64), device="cuda")


def _np(tensor):
    return tensor.cpu().numpy()


# ---------------------------------------------------------------- block tables and slot maps
def _tables_state(rng, context, new, page, *, blocks=None, spare=16, surplus=False):
    context, new = np.asarray(context), np.asarray(new)
    counts = -(-np.maximum(context, 0) // page) + (rng.integers(0, 2, len(context)) if surplus else 0)
    blocks = blocks or int(max(1, (-(-(np.maximum(context, 0) + np.maximum(new, 0)) // page)).max(), counts.max()))
    pages = rng.permutation(int(counts.sum() + (np.maximum(new, 0) // page + 2).sum() + spare)).astype(np.int32)
    tables = np.full((len(context), blocks), -1, np.int32)
    at = 0
    for r, count in enumerate(counts):
        count = min(int(count), blocks)
        tables[r, :count] = pages[at: at + count]
        at += count
    free = np.concatenate([np.full(5, -7, np.int32), pages[at:]])
    return tables, counts.astype(np.int32), free, np.array([5], np.int32)


def _check_tables(context, new, tables, counts, free, start, page, max_tokens, in_place=False):
    expected = oracle.tables(context, new, tables, counts, free, start[0], page, max_tokens)
    device_tables, error = _i32(tables), torch.zeros(1, dtype=torch.int32, device="cuda")
    device_counts, device_start = _i32(counts), _i32(start)
    step = None
    if in_place:
        ops = _ops()
        step = ops.PagedStep(*(torch.full((n,), -9, dtype=d, device="cuda") for n, d in (
            (len(context) + 1, torch.int32), (len(context), torch.int32), (max_tokens, torch.int64),
            (max_tokens, torch.int64))), device_counts, device_start)
    got = _ops().paged_tables(_i32(context), _i32(new), device_tables, device_counts, _i32(free), device_start,
                              page_size=page, max_tokens=max_tokens, step=step, error=error)
    for name, a, e in (("query_start", got.query_start, expected[0]), ("kv_lens", got.kv_lens, expected[1]),
                       ("positions", got.positions, expected[2]), ("slots", got.slots, expected[3]),
                       ("tables", device_tables, expected[4]), ("counts", got.page_counts, expected[5]),
                       ("start", got.free_start, expected[6])):
        np.testing.assert_array_equal(_np(a), e, err_msg=name)
    assert int(error) == expected[7]
    return got


@pytest.mark.parametrize("page", [1, 5, 16, 64])
@pytest.mark.parametrize("requests", [1, 3, 70, 1024, 1025, 2500])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables_of_ragged_requests(page, requests, in_place):
    rng = np.random.default_rng(page * 10000 + requests)
    context = rng.integers(0, 90, requests)
    new = rng.choice([0, 1, 1, 7, 40], requests)
    state = _tables_state(rng, context, new, page, surplus=True)
    _check_tables(context, new, *state, page, int(new.sum()) + 13, in_place)


@pytest.mark.parametrize("max_tokens", [4096, 4097, 20000])
def test_tables_on_both_sides_of_the_second_launch(max_tokens):
    rng = np.random.default_rng(max_tokens)
    context, new = rng.integers(0, 300, 37), rng.integers(0, 110, 37)
    new[5] = max_tokens - new.sum() + new[5] - 3
    state = _tables_state(rng, context, new, 16)
    _check_tables(context, new, *state, 16, max_tokens)


def test_tables_of_a_page_boundary_and_of_nothing():
    # a context that ends on a page, one token short of it, one past it; an idle row; no rows at all
    rng = np.random.default_rng(3)
    context, new = np.array([32, 31, 33, 0, 16]), np.array([1, 1, 1, 0, 16])
    state = _tables_state(rng, context, new, 16)
    _check_tables(context, new, *state, 16, 19)
    _check_tables(context, np.zeros(5, int), *state, 16, 0)
    _check_tables(context, np.zeros(5, int), *state, 16, 4)


@pytest.mark.parametrize("big", [False, True])  # one launch, two launches
def test_tables_flag_what_does_not_fit(big):
    rng = np.random.default_rng(4)
    room = 5000 if big else 64
    context, new = np.array([20, 0, 100, 7]), np.array([30, 3, 8, 40])
    tables, counts, free, start = _tables_state(rng, context, new, 8)
    _check_tables(context, new, tables, counts, free, start, 8, 50 if not big else room)   # 81 tokens: cut
    _check_tables(context, new, tables, counts, free[:8], start, 8, room + 40)             # three pages left
    _check_tables(context, new, tables, counts, free[:0], np.array([0], np.int32), 8, room + 40)
    _check_tables(context, new, tables, counts, free, np.array([9999], np.int32), 8, room + 40)
    _check_tables(context, new, tables[:, :5], counts, free, start, 8, room + 40)          # rows too short
    _check_tables(np.array([-4, 0, 100, 7]), np.array([3, -3, 8, 1]), tables, np.maximum(counts - 99, -1), free, start,
                  8, room + 40)


def test_tables_replay_in_a_graph():
    # decode steps captured once: the counts, the free list's start and the lengths move on in device memory
    rng = np.random.default_rng(5)
    context, new = np.array([5, 16, 0, 31]), np.array([1, 1, 0, 1])
    tables, counts, free, start = _tables_state(rng, context, new, 16, blocks=6, spare=64)
    ops = _ops()
    d = [_i32(v) for v in (context, new, tables, counts, free, start)]
    step = ops.paged_tables(*d, page_size=16, max_tokens=6)
    for t, v in zip(d, (context, new, tables, counts, free, start)):
        t.copy_(torch.from_numpy(v.astype(np.int32)))
    step = step._replace(page_counts=d[3], free_start=d[5])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_tables(*d, page_size=16, max_tokens=6, step=step)
        d[0].copy_(step.kv_lens)
    for t, v in zip(d, (context, new, tables, counts, free, start)):
        t.copy_(torch.from_numpy(v.astype(np.int32)))
    for i in range(40):
        if i == 20:
            new = np.array([0, 3, 2, 1])
            d[1].copy_(torch.from_numpy(new.astype(np.int32)))
        want = oracle.tables(context, new, tables, counts, free, start[0], 16, 6)
        graph.replay()
        torch.cuda.synchronize()
        for got, expected in zip((step.query_start, step.kv_lens, step.positions, step.slots, d[2], d[3], d[5]), want):
            np.testing.assert_array_equal(_np(got), expected)
        context, tables, counts, start = want[1], want[4], want[5], want[6]


# ---------------------------------------------------------------- RoPE and the cache write
def _cache(rng, pages, kv_heads, page, dim, layout):
    """Keys and values [P, Hkv, page, D] in one of three layouts, and their values."""

    host = [bf16_normal(rng, (pages, kv_heads, page, dim)) for _ in range(2)]
    if layout == "dense":
        return [to_gpu_bf16(x) for x in host], host
    if layout == "tokens":  # [P, page, Hkv, D] seen per head
        return [to_gpu_bf16(np.ascontiguousarray(x.transpose(0, 2, 1, 3))).transpose(1, 2) for x in host], host
    both = torch.zeros((pages, kv_heads, page, 2 * dim + 16), dtype=torch.bfloat16, device="cuda")  # rows side by side
    out = [both[..., 8: 8 + dim], both[..., dim + 16:]]
    for t, x in zip(out, host):
        t.copy_(to_gpu_bf16(x))
    return out, host


@pytest.mark.parametrize("hq,hkv,dim", [(14, 2, 64), (32, 8, 128), (5, 5, 16), (6, 1, 96), (3, 1, 80)])
@pytest.mark.parametrize("tokens,page", [(1, 16), (7, 1), (33, 24), (130, 64)])
@pytest.mark.parametrize("layout", ["dense", "tokens", "rows"])
def test_rope_append(hq, hkv, dim, tokens, page, layout):
    rng = np.random.default_rng(hq + dim + tokens)
    pages = -(-2 * tokens // page) + 1
    (keys, values), (k0, v0) = _cache(rng, pages, hkv, page, dim, layout)
    width = (hq + 2 * hkv) * dim
    qkv = bf16_normal(rng, (tokens, width))
    cos, sin = bf16_normal(rng, (50, dim)), bf16_normal(rng, (50, dim))
    positions = rng.integers(0, 50, tokens)
    slots = rng.permutation(pages * page)[:tokens].astype(np.int64)
    slots[rng.random(tokens) < 0.2] = -1
    if layout == "rows":  # the projection's rows inside wider ones
        wide = torch.zeros((tokens, width + 40), dtype=torch.bfloat16, device="cuda")
        wide[:, 16: 16 + width] = to_gpu_bf16(qkv)
        x = wide[:, 16: 16 + width]
    else:
        x = to_gpu_bf16(qkv)
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = torch.full((tokens, hq, dim), 7.0, dtype=torch.bfloat16, device="cuda")
    got = _ops().paged_rope_append(x, _i64(positions), _i64(slots), to_gpu_bf16(cos), to_gpu_bf16(sin), keys, values,
                                   query_heads=hq, q_out=q_out, error=error)
    heads = qkv.astype(np.float64).reshape(tokens, hq + 2 * hkv, dim)
    turned, size = oracle.rope(heads[:, : hq + hkv], cos.astype(np.float64)[positions][:, None],
                               sin.astype(np.float64)[positions][:, None])
    # one rounding to bf16; before it the products of two bf16 are exact in f32 and their sum is rounded once or twice
    bound = HALF * np.abs(turned) + 2.0 ** -22 * size
    live = slots >= 0
    q = from_gpu_bf16(got).astype(np.float64)
    assert (np.abs(q - turned[:, :hq]) <= bound[:, :hq])[live].all()
    assert (q[~live] == 7.0).all()
    k1, v1 = from_gpu_bf16(keys).astype(np.float64), from_gpu_bf16(values).astype(np.float64)
    at = (slots[live] // page, slice(None), slots[live] % page)
    assert (np.abs(k1[at] - turned[live, hq:]) <= bound[live, hq:]).all()
    np.testing.assert_array_equal(v1[at], heads[live, hq + hkv:])
    k0, v0 = k0.astype(np.float64), v0.astype(np.float64)  # the rest of the cache is as it was
    k0[at], v0[at] = k1[at], v1[at]
    np.testing.assert_array_equal(k1, k0)
    np.testing.assert_array_equal(v1, v0)
    assert int(error) == 0


@pytest.mark.parametrize("slot,position,flag", [(64, 0, 8), (-2, 0, 8), (2 ** 40, 0, 8), (3, 50, 16), (3, -1, 16)])
def test_rope_append_leaves_bad_rows_out(slot, position, flag):
    rng = np.random.default_rng(1)
    (keys, values), (k0, v0) = _cache(rng, 4, 2, 16, 64, "dense")
    table = to_gpu_bf16(bf16_normal(rng, (50, 64)))
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = torch.full((2, 2, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    _ops().paged_rope_append(to_gpu_bf16(bf16_normal(rng, (2, 6 * 64))), _i64([position, 0]), _i64([slot, 5]), table,
                             table, keys, values, query_heads=2, q_out=q_out, error=error)
    assert int(error) == flag
    assert bool((q_out[0] == 7.0).all()) and not bool((q_out[1] == 7.0).any())
    same = np.ones((4, 2, 16), bool)
    same[0, :, 5] = False
    np.testing.assert_array_equal(from_gpu_bf16(keys)[same], k0[same])
    np.testing.assert_array_equal(from_gpu_bf16(values)[same], v0[same])


# ---------------------------------------------------------------- attention
def _requests(rng, lengths, hq, hkv, dim, page, *, layout="dense", spare=3, tail=0, blocks=None):
    """Inputs of paged_attention for (rows, keys) of each request, with `tail` rows behind the last."""

    new, kv = np.array([n for n, _ in lengths]), np.array([k for _, k in lengths])
    counts = -(-kv // page)
    pages = int(counts.sum()) + spare
    blocks = blocks or max(1, int(counts.max()))
    tables = np.full((len(lengths), blocks), -1, np.int32)
    order, at = rng.permutation(pages), 0
    for r, count in enumerate(counts):
        tables[r, :count] = order[at: at + count]
        at += count
    device, host = _cache(rng, pages, hkv, page, dim, layout)
    q = bf16_normal(rng, (int(new.sum()) + tail, hq, dim))
    return dict(q=q, keys=host[0], values=host[1], tables=tables, start=np.concatenate([[0], np.cumsum(new)]), kv=kv,
                device=device)


def _attend(s, *, q=None, **kwargs):
    q = to_gpu_bf16(s["q"]) if q is None else q
    out = torch.full((q.shape[0], q.shape[1] * q.shape[2]), 5.0, dtype=torch.bfloat16, device="cuda")
    got = _ops().paged_attention(q, *s["device"], _i32(s["tables"]), _i32(s["start"]), _i32(s["kv"]), out=out, **kwargs)
    assert got is out
    return out


def attention_bound(want, size):
    return HALF * (1 + 2 * HALF) * (2 * np.abs(want) + size) + 4e-5 * size


def _check_attention(s, got, **kwargs):
    want, size, written = oracle.attention(s["q"], s["keys"], s["values"], s["tables"], s["start"], s["kv"], **kwargs)
    got = from_gpu_bf16(got).astype(np.float64)
    # out = sum p' v / sum p' with p' = p (1 + d), |d| <= HALF, the weights rounded to bf16 for the product (and, in wide
    # tiles, for the sum): off by sum p d (v - want) / sum p' <= HALF (size + |want|) / (1 - HALF); the result is rounded
    # once more, HALF of itself. Scores of |s| < 100 in f32 add 100 * 2^-23 to log p, exponentials and sums less: 2e-5
    # of sum p |v| and of |want|, which is no larger
    bound = attention_bound(want, size)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad[written].any(), (np.argwhere(bad & written[:, None])[:5], np.abs(got - want)[bad & written[:, None]][:5])
    assert (got[~written] == 5.0).all()


HEADS = [(14, 2, 64), (32, 8, 128), (4, 4, 64), (8, 1, 128), (28, 4, 64), (3, 1, 128), (20, 1, 64), (40, 2, 128)]


@pytest.mark.parametrize("hq,hkv,dim", HEADS)
@pytest.mark.parametrize("page", [1, 16, 24, 64, 256])
def test_attention_of_single_tokens(hq, hkv, dim, page):
    rng = np.random.default_rng(hq * dim + page)
    s = _requests(rng, [(1, 1), (1, 2), (1, 15), (0, 9), (1, 16), (1, 17), (1, 129), (1, 700)], hq, hkv, dim, page, tail=3)
    _check_attention(s, _attend(s))
    _check_attention(s, _attend(s, max_query_len=1, max_kv_len=700))


@pytest.mark.parametrize("hq,hkv,dim", HEADS)
@pytest.mark.parametrize("page", [1, 8, 48, 256])
def test_attention_of_chunks(hq, hkv, dim, page):
    rng = np.random.default_rng(hq * dim + page)
    s = _requests(rng, [(5, 5), (1, 200), (70, 133), (2, 31), (0, 0), (131, 131), (9, 300)], hq, hkv, dim, page, tail=2)
    _check_attention(s, _attend(s))
    _check_attention(s, _attend(s, causal=False), causal=False)


@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33, 65])
def test_attention_of_a_few_rows(rows):
    rng = np.random.default_rng(rows)
    s = _requests(rng, [(rows, rows), (rows, rows + 1), (rows, 333)], 8, 2, 64, 16)
    _check_attention(s, _attend(s, max_query_len=rows))
    _check_attention(s, _attend(s))


@pytest.mark.parametrize("layout", ["tokens", "rows"])
@pytest.mark.parametrize("lengths", [[(1, 90), (1, 41)], [(40, 90), (3, 41)]])
def test_attention_of_strided_operands(layout, lengths):
    rng = np.random.default_rng(7)
    s = _requests(rng, lengths, 8, 4, 128, 16, layout=layout)
    # the queries where the projection left them, heads of a row with a gap between them
    wide = torch.zeros((s["q"].shape[0], 8, 160), dtype=torch.bfloat16, device="cuda")
    wide[..., 16:144] = to_gpu_bf16(s["q"])
    _check_attention(s, _attend(s, q=wide[..., 16:144]))


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_over_long_requests_is_split_and_joined(rows):
    rng = np.random.default_rng(rows)
    s = _requests(rng, [(rows, 9000), (1, 3), (rows, 5000), (1, 1)], 4, 1, 64, 16)
    _check_attention(s, _attend(s))
    _check_attention(s, _attend(s, max_query_len=rows, max_kv_len=9000))


@pytest.mark.parametrize("rows", [1, 30])
def test_attention_bounds_choose_the_launch_and_not_the_result(rows):
    # bounds that are not true: the lengths on the GPU decide
    rng = np.random.default_rng(rows)
    s = _requests(rng, [(rows, 700), (rows, 70)], 8, 2, 128, 16)
    for most, keys in ((1, 1), (1, 0), (0, 64), (500, 5000)):
        _check_attention(s, _attend(s, max_query_len=most, max_kv_len=keys))


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_without_keys_gives_zero(rows):
    rng = np.random.default_rng(8)
    s = _requests(rng, [(rows, 40), (rows, 40), (rows, 40)], 8, 2, 64, 16)
    s["kv"] = np.array([0, 40, rows // 2])  # no keys; all; fewer than rows: the first see none
    _check_attention(s, _attend(s))
    s["kv"] = np.array([-5, 40, 40])
    s["tables"][1] = -1                     # no page is known
    _check_attention(s, _attend(s))


@pytest.mark.parametrize("rows", [1, 20])
@pytest.mark.parametrize("keys", [60, 3000])  # whole items, items that are cut and joined
def test_attention_leaves_rows_before_the_first_request(rows, keys):
    rng = np.random.default_rng(17)
    s = _requests(rng, [(rows, keys), (rows, 40)], 8, 2, 64, 16)
    s["q"] = np.concatenate([bf16_normal(rng, (5, 8, 64)), s["q"]])
    s["start"] = s["start"] + 5
    got = _attend(s, max_query_len=rows, max_kv_len=keys)
    assert bool((got[:5] == 5.0).all())
    _check_attention(s, got)


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_leaves_out_entries_that_name_no_page(rows):
    rng = np.random.default_rng(9)
    s = _requests(rng, [(rows, 400), (rows, 300)], 8, 2, 128, 16)
    s["tables"][0, 3], s["tables"][0, 11], s["tables"][1, 0] = -1, 10 ** 6, -(2 ** 31)
    s["tables"][1, 18] = 2 ** 31 - 1  # the last entry, with the rows' own keys
    _check_attention(s, _attend(s))
    s["kv"] = np.array([10 ** 9, 300])      # longer than the table row
    _check_attention(s, _attend(s))


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_keeps_what_it_may_not_see_out(rows):
    # NaN and infinities in the pages' unused rows and in pages of other requests
    rng = np.random.default_rng(10)
    s = _requests(rng, [(rows, 37), (rows, 100)], 8, 2, 64, 16, spare=4)
    used = np.zeros(s["keys"].shape[0::2][:2], bool)
    for r, length in enumerate(s["kv"]):
        j = np.arange(length)
        used[s["tables"][r, j // 16], j % 16] = True
    for host, device, value in ((s["keys"], s["device"][0], np.nan), (s["values"], s["device"][1], np.inf)):
        host.transpose(0, 2, 1, 3)[~used] = value
        device.copy_(to_gpu_bf16(host))
    _check_attention(s, _attend(s))


def _check_special_values(s, marks, **bounds):
    """Place (request, key, value) in two dims of the request's own each: rows that see the key have the value there."""

    hq, dim = s["q"].shape[1:]
    page = s["keys"].shape[2]
    for i, (r, j, value) in enumerate(marks):
        s["values"][s["tables"][r, j // page], :, j % page, 3 * i: 3 * i + 2] = value
    s["device"][1].copy_(to_gpu_bf16(s["values"]))
    got = from_gpu_bf16(_attend(s, **bounds)).astype(np.float64)
    plain = {**s, "values": np.where(np.isfinite(s["values"]), s["values"], 0.0)}
    want, size, written = oracle.attention(plain["q"], plain["keys"], plain["values"], s["tables"], s["start"], s["kv"])
    special = np.zeros(want.shape)
    for i, (r, j, value) in enumerate(marks):
        rows = s["start"][r + 1] - s["start"][r]
        seen = s["start"][r] + np.arange(rows)[s["kv"][r] - rows + np.arange(rows) >= j]
        for h in range(hq):
            special[seen[:, None], dim * h + 3 * i + np.arange(2)] = value
    odd = special != 0
    assert odd.any()
    np.testing.assert_array_equal(got[odd], special[odd])
    assert (np.abs(got - want) <= attention_bound(want, size))[~odd & written[:, None]].all()


@pytest.mark.parametrize("rows", [1, 5, 40])
def test_attention_of_infinite_values(rows):
    # an infinite value reaches the rows that see its key, in its own dims, and no others
    s = _requests(np.random.default_rng(16), [(rows, 333), (rows, rows), (rows, 64)], 8, 2, 64, 16)
    last = s["kv"] - 1
    _check_special_values(s, [(0, 200, np.inf), (1, last[1], -np.inf), (2, last[2] - rows // 2, np.nan)])


#: kernel, query heads, kv heads, head dim, most rows of a request, requests
FORMS = [("d64_n1", 8, 4, 64, 8, 5), ("d64_n2", 8, 4, 64, 16, 5), ("d64_w", 14, 2, 64, 150, 7),
         ("d128_n1", 8, 2, 128, 4, 5), ("d128_n2", 8, 2, 128, 8, 5), ("d128_w", 12, 2, 128, 150, 5),
         ("d128_w", 32, 8, 128, 80, 20), ("d128_w", 128, 1, 128, 64, 9), ("d64_w", 128, 1, 64, 7, 3)]


@pytest.mark.parametrize("kernel,hq,hkv,dim,most,requests", FORMS)
@pytest.mark.parametrize("keys", [700, 1500])  # within one item, over several
def test_attention_of_every_form(kernel, hq, hkv, dim, most, requests, keys):
    rng = np.random.default_rng(hq + most + keys)
    rows = rng.integers(0, most + 1, requests)
    rows[1], rows[2], rows[-1] = most, most - 1, most
    lengths = [(int(n), int(n) + int(rng.integers(0, 400))) for n in rows]
    lengths[2] = (most - 1, keys)
    s = _requests(rng, lengths, hq, hkv, dim, 16, tail=3)
    bounds = dict(max_query_len=most, max_kv_len=keys)
    with _ops().recording_launches() as take:
        got = _attend(s, **bounds)
        assert "aoto_paged_attention_" + kernel in take()
    _check_attention(s, got)
    _check_attention(s, _attend(s, causal=False, **bounds), causal=False)
    kv = s["kv"].copy()
    s["kv"][1], s["kv"][-1] = most // 2, 0       # the first rows see no key; no row sees one
    _check_attention(s, _attend(s, **bounds))
    s["kv"] = kv
    last = s["kv"] - 1
    _check_special_values(s, [(1, last[1], np.inf), (2, keys - most, -np.inf), (2, last[2] - most // 2, np.nan),
                              (2, 0, -np.inf)], **bounds)
    s["values"] = np.where(np.isfinite(s["values"]), s["values"], 0.0)
    s["device"][1].copy_(to_gpu_bf16(s["values"]))
    s["tables"][2, 3], s["tables"][2, -(-keys // 16) - 1], s["tables"][1, 0] = -1, 10 ** 6, -(2 ** 31)
    _check_attention(s, _attend(s, **bounds))


def _form_requests(rng, hq, hkv, dim, most, requests, keys):
    """Requests of a form of ``FORMS``: the second and the last of ``most`` rows, the third over ``keys`` keys."""

    rows = rng.integers(0, most + 1, requests)
    rows[1], rows[2], rows[-1] = most, most - 1, most
    lengths = [(int(n), int(n) + int(rng.integers(0, 400))) for n in rows]
    lengths[2] = (most - 1, keys)
    return _requests(rng, lengths, hq, hkv, dim, 16, tail=3)


def _form_attend(s, kernel, most, keys, cut):
    """The call with that kernel, its items whole or cut and joined."""

    with _ops().recording_launches() as take:
        # a bound that is not true keeps the items whole
        got = _attend(s, max_query_len=most, max_kv_len=keys if cut else 64)
        launches = take()
    assert "aoto_paged_attention_" + kernel in launches
    return got, any("join" in name for name in launches)


def _check_attention_pattern(s, got):
    """NaN where the definition has it, everything else within the bound."""

    with np.errstate(invalid="ignore"):
        want, size, written = oracle.attention(s["q"], s["keys"], s["values"], s["tables"], s["start"], s["kv"])
    got = from_gpu_bf16(got).astype(np.float64)
    odd = np.isnan(want)
    assert odd.any() and not odd[written].all()
    np.testing.assert_array_equal(np.isnan(got), odd)
    assert (np.abs(got - want) <= attention_bound(want, size))[~odd & written[:, None]].all()
    assert (got[~written] == 5.0).all()


@pytest.mark.parametrize("kernel,hq,hkv,dim,most,requests", FORMS)
@pytest.mark.parametrize("cut", [False, True])
def test_attention_of_nan_and_infinite_scores(kernel, hq, hkv, dim, most, requests, cut):
    # a query that is NaN makes its row NaN, a key that is NaN the rows that see it; a score of +inf the row it is in
    # (inf - inf), one of -inf weighs nothing
    rng = np.random.default_rng(hq + most)
    s = _form_requests(rng, hq, hkv, dim, most, requests, 1500)
    first, rows, kv = s["start"][:-1], np.diff(s["start"]), s["kv"]

    def key(r, j):
        return s["keys"][s["tables"][r, j // 16], :, j % 16]

    s["q"][first[2] + 1, 0, 5] = np.nan                  # all scores of one head's row
    key(1, kv[1] - 1 - rows[1] // 2)[hkv - 1, 7] = np.nan  # a key that the later rows of one kv head see
    key(2, 700)[0, 3] = np.nan if hkv > 1 else np.inf    # inside the long request, in one part of it
    key(requests - 1, kv[-1] - 1)[0, 0] = np.inf         # +inf or -inf, as the last row's query has it
    s["device"][0].copy_(to_gpu_bf16(s["keys"]))
    got, joined = _form_attend(s, kernel, most, 1500, cut)
    if not cut:
        assert not joined
    _check_attention_pattern(s, got)


def _vanishing(rng, s, r, keys):
    """Keys of request r whose weights are below 2^-150 of their rows' largest: queries near 1, these keys -16."""

    first, last = s["start"][r], s["start"][r + 1]
    s["q"][first:last] = from_gpu_bf16(to_gpu_bf16(1 + 0.1 * bf16_normal(rng, s["q"][first:last].shape)))
    for j in keys:
        s["keys"][s["tables"][r, j // 16], :, j % 16] = -16.0
    s["device"][0].copy_(to_gpu_bf16(s["keys"]))


@pytest.mark.parametrize("kernel,hq,hkv,dim,most,requests", FORMS)
@pytest.mark.parametrize("cut", [False, True])
def test_attention_of_large_values_that_weigh_nothing(kernel, hq, hkv, dim, most, requests, cut):
    # values near the largest number, hidden from a row or next to it of no weight, leave the row as it is
    rng = np.random.default_rng(hq + most + 1)
    s = _form_requests(rng, hq, hkv, dim, most, requests, 1500)
    low = [*range(600), 700, 1023, 1024, 1490 - most]
    _vanishing(rng, s, 2, low)
    for i, j in enumerate((0, 300, *low[600:])):
        s["values"][s["tables"][2, j // 16], :, j % 16, 4 * i: 4 * i + 2] = -3e38 if i % 2 else 3e38
    last = s["kv"][1] - 1   # the key of the second request's last row
    s["values"][s["tables"][1, last // 16], :, last % 16, 40: 50] = 3e38
    s["device"][1].copy_(to_gpu_bf16(s["values"]))
    s["values"] = from_gpu_bf16(s["device"][1]).copy()
    got = from_gpu_bf16(_form_attend(s, kernel, most, 1500, cut)[0]).astype(np.float64)
    want, size, written = oracle.attention(s["q"], s["keys"], s["values"], s["tables"], s["start"], s["kv"])
    written[s["start"][2] - 1] = False
    # scores of up to 16 * 128^(1/2) = 181 in f32 add 181 * 2^-23 = 2.2e-5 to log p, of the few that matter 2e-6
    assert (np.abs(got - want) <= attention_bound(want, size))[written].all()


@pytest.mark.parametrize("kernel,hq,hkv,dim,most,requests", FORMS)
@pytest.mark.parametrize("cut", [False, True])
def test_attention_of_infinite_values_that_weigh_nothing(kernel, hq, hkv, dim, most, requests, cut):
    # a weight is above 0 however small, and infinite with an infinite value: in whole tiles, in parts whose keys all
    # weigh nothing beside the others', before and after the running maximum
    rng = np.random.default_rng(hq + most + 2)
    s = _form_requests(rng, hq, hkv, dim, most, requests, 1500)
    _vanishing(rng, s, 2, [*range(600), 700, 1023, 1024, 1490 - most])
    bounds = dict(max_query_len=most, max_kv_len=1500 if cut else 64)
    _check_special_values(s, [(2, 0, np.inf), (2, 300, -np.inf), (2, 700, np.inf), (2, 1024, np.nan), (2, 1023, -np.inf),
                              (1, s["kv"][1] - 1, np.inf)], **bounds)


@pytest.mark.parametrize("kernel,hq,hkv,dim,most,requests", FORMS)
@pytest.mark.parametrize("cut", [False, True])
def test_attention_of_scores_that_are_all_minus_infinity(kernel, hq, hkv, dim, most, requests, cut):
    # 0 / 0 is NaN for rows that see such keys alone; beside others they weigh nothing; rows without keys are 0
    rng = np.random.default_rng(hq + most + 3)
    s = _form_requests(rng, hq, hkv, dim, most, requests, 1500)
    s["q"][s["start"][1]: s["start"][3], :, 0] = -1.0
    for r, keys in ((1, range(s["kv"][1])), (2, range(640))):
        for j in keys:
            s["keys"][s["tables"][r, j // 16], :, j % 16, 0] = np.inf
    s["device"][0].copy_(to_gpu_bf16(s["keys"]))
    s["kv"][-1] = 0
    _check_attention_pattern(s, _form_attend(s, kernel, most, 1500, cut)[0])
    s["tables"][1] = -1     # without pages it sees none of them
    _check_attention(s, _form_attend(s, kernel, most, 1500, cut)[0])


@pytest.mark.parametrize("requests", [8, 32, 33, 128, 129, 256, 257, 600])
@pytest.mark.parametrize("most", [1, 40])        # narrow tiles; wide ones beside them
@pytest.mark.parametrize("cut", [False, True])
def test_attention_of_many_requests(requests, most, cut):
    # a thread of the dealing takes a share of a request's tiles, a request, or several of them
    rng = np.random.default_rng(requests + most)
    rows = rng.choice([0, 1, 1, 3, most], requests)
    rows = np.minimum(rows, most)
    rows[-1] = most
    kv = rows + rng.integers(0, 60, requests)
    kv[::9] += rng.integers(0, 1300, len(kv[::9]))
    s = _requests(rng, list(zip(rows.tolist(), kv.tolist())), 4, 1, 64, 16, tail=1, blocks=90)
    got, joined = _form_attend(s, "d64_w" if most > 1 else "d64_n1", most, 1440, cut)
    assert joined == (cut and (most == 1 or requests < 256))
    _check_attention(s, got)


def narrow_bound(want, size):
    # a weight is its upper 8 bits and what they leave, less than 2^-7 of it, rounded to bf16: off by 2^-7 HALF, and by
    # as much of sum p |v|; the sum is of the weights as they were, the result is rounded once, and f32 adds what it
    # does in _check_attention
    return HALF * (1 + HALF) * np.abs(want) + (1 + HALF) * (2.0 ** -7 * HALF + 4e-5) * size


@pytest.mark.parametrize("hq,hkv,dim", [h for h in HEADS if h[0] // h[1] <= 16])
@pytest.mark.parametrize("most", [1, 200])       # narrow tiles alone, and beside wide ones
def test_attention_of_single_tokens_keeps_16_bits_of_the_weights(hq, hkv, dim, most):
    rng = np.random.default_rng(hq * dim + most)
    s = _requests(rng, [(1, 1), (1, 2), (0, 9), (1, 16), (1, 129), (1, 700), (1, 1500)], hq, hkv, dim, 16, tail=2)
    got = from_gpu_bf16(_attend(s, max_query_len=most)).astype(np.float64)
    want, size, written = oracle.attention(s["q"], s["keys"], s["values"], s["tables"], s["start"], s["kv"])
    assert (np.abs(got - want) <= narrow_bound(want, size))[written].all()


@pytest.mark.parametrize("hq,hkv,dim", [(8, 2, 64), (8, 2, 128), (16, 4, 128)])
def test_attention_of_drafted_rows_keeps_16_bits_of_the_weights(hq, hkv, dim):
    rng = np.random.default_rng(hq * dim)
    s = _requests(rng, [(5, 5), (8, 40), (0, 9), (1, 16), (7, 129), (8, 700), (3, 1500)], hq, hkv, dim, 16, tail=2)
    got = from_gpu_bf16(_attend(s, max_query_len=8)).astype(np.float64)
    want, size, written = oracle.attention(s["q"], s["keys"], s["values"], s["tables"], s["start"], s["kv"])
    assert (np.abs(got - want) <= narrow_bound(want, size))[written].all()


@pytest.mark.parametrize("kernel,hq,hkv,dim,most,requests", FORMS)
@pytest.mark.parametrize("cut", [False, True])
def test_attention_of_large_values_as_scores_rise(kernel, hq, hkv, dim, most, requests, cut):
    # a value near the largest number, its weight 200 times that of the keys before it and a tenth of the row's
    rng = np.random.default_rng(hq + most + 4)
    s = _form_requests(rng, hq, hkv, dim, most, requests, 1500)
    s["q"][s["start"][2]: s["start"][3]] = 1.0
    for j in range(1500):
        s["keys"][s["tables"][2, j // 16], :, j % 16] = 5.3 / dim ** 0.5 if j == 700 else 0.0
    s["values"][s["tables"][2, 700 // 16], :, 700 % 16, :9] = -3e38
    for host, device in zip((s["keys"], s["values"]), s["device"]):
        device.copy_(to_gpu_bf16(host))
    s["keys"], s["values"] = (from_gpu_bf16(device).copy() for device in s["device"])
    _check_attention(s, _form_attend(s, kernel, most, 1500, cut)[0])


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_of_large_scores(rows):
    # one key far above the others, scores to +-90: the running maximum moves, nothing overflows
    rng = np.random.default_rng(11)
    s = _requests(rng, [(rows, 300), (rows, 64)], 8, 2, 64, 16)
    s["q"] *= 16
    s["q"][:, ::2] *= -1
    _check_attention(s, _attend(s), scale=None)
    _check_attention(s, _attend(s, scale=1e-3), scale=1e-3)


@pytest.mark.parametrize("rows", [1, 20])
def test_attention_past_31_bits_of_cache(rows):
    # 2^31 elements and more before the pages in use
    page, hkv, dim = 16, 8, 128
    pages = 2 ** 31 // (page * hkv * dim) + 8
    rng = np.random.default_rng(12)
    s = _requests(rng, [(rows, 100)], 8, hkv, dim, page, spare=0)
    keys = torch.zeros((pages, hkv, page, dim), dtype=torch.bfloat16, device="cuda")
    values = torch.zeros_like(keys)
    keys[-8:][: s["keys"].shape[0]], values[-8:][: s["values"].shape[0]] = s["device"]
    s["device"] = (keys, values)
    got = _ops().paged_attention(to_gpu_bf16(s["q"]), keys, values, _i32(s["tables"] + pages - 8), _i32(s["start"]),
                                 _i32(s["kv"]))
    _check_attention(s, got)
    slots = _i64([pages * page - 3])
    x = to_gpu_bf16(bf16_normal(rng, (1, 3 * hkv * dim)))
    table = torch.ones((1, dim), dtype=torch.bfloat16, device="cuda")
    _ops().paged_rope_append(x, _i64([0]), slots, table, torch.zeros_like(table), keys, values, query_heads=hkv)
    torch.testing.assert_close(values[-1, :, -3], x[0].view(-1, dim)[2 * hkv:], rtol=0, atol=0)


def test_attention_replays_in_graphs_that_share_a_workspace():
    rng = np.random.default_rng(13)
    ops = _ops()
    graphs = []
    shapes = [[(1, 900), (1, 40), (1, 2000)], [(20, 900), (1, 40), (4, 1500)]]
    sizes = [ops.paged_attention_workspace(sum(n for n, _ in x), 3, 125, 16, 8, 2, 64, device="cuda").numel() for x in shapes]
    workspace = torch.empty(max(sizes), dtype=torch.uint8, device="cuda")
    for lengths in shapes:
        s = _requests(rng, lengths, 8, 2, 64, 16, blocks=125)
        s["in"] = [to_gpu_bf16(s["q"]), *s["device"], _i32(s["tables"]), _i32(s["start"]), _i32(s["kv"])]
        s["out"] = torch.full((s["q"].shape[0], 512), 5.0, dtype=torch.bfloat16, device="cuda")
        ops.paged_attention(*s["in"], out=s["out"], workspace=workspace)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_attention(*s["in"], out=s["out"], workspace=workspace)
        graphs.append((graph, s))
    for i in range(4):
        for graph, s in graphs:
            if i:  # the requests in another order of lengths, and shorter
                s["kv"] = np.maximum(s["kv"] - 37 * i, np.diff(s["start"]))
                s["in"][5].copy_(_i32(s["kv"]))
            s["out"].fill_(5.0)
            graph.replay()
        for graph, s in graphs:
            _check_attention(s, s["out"])


def test_attention_on_another_stream_and_with_a_small_workspace():
    rng = np.random.default_rng(14)
    s = _requests(rng, [(1, 3000), (1, 50)], 8, 2, 64, 16)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = _attend(s, workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    stream.synchronize()
    _check_attention(s, got)


def test_attention_on_two_streams_at_once():
    # each call has a workspace of its own
    rng = np.random.default_rng(18)
    ops, streams, runs = _ops(), [torch.cuda.Stream(), torch.cuda.Stream()], []
    for lengths in ([(1, 3000), (1, 50), (1, 4100)], [(150, 2000), (1, 900), (7, 7)]):
        s = _requests(rng, lengths, 8, 2, 64, 16)
        runs.append((s, [to_gpu_bf16(s["q"]), *s["device"], _i32(s["tables"]), _i32(s["start"]), _i32(s["kv"])], []))
    torch.cuda.synchronize()
    for _ in range(10):
        for (_, inputs, outs), stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                outs.append(ops.paged_attention(*inputs))
    torch.cuda.synchronize()
    for s, _, outs in runs:
        _check_attention(s, outs[0])
        assert all(bool((o == outs[0]).all()) for o in outs)


def test_attention_is_the_same_every_time():
    rng = np.random.default_rng(15)
    s = _requests(rng, [(1, 3000), (40, 2500), (3, 50)], 8, 2, 64, 16)
    first = _attend(s)
    for _ in range(3):
        assert torch.equal(first, _attend(s))


# ---------------------------------------------------------------- verification of drafted tokens
def _logits(rng, shape, dtype):
    z = rng.standard_normal(shape).astype(np.float32) * 3
    t = torch.tensor(z, device="cuda").to(dtype)
    return t, _np(t.float())


def _drafted(rng, counts, drafts, vocab, dtype, with_law):
    start = np.concatenate([[0], np.cumsum(np.array(counts) + 1)])
    logits, host = _logits(rng, (int(start[-1]), vocab), dtype)
    requests = len(counts)
    tokens = rng.integers(0, vocab, (requests, drafts))
    law = law_host = None
    if with_law:
        law, law_host = _logits(rng, (requests, drafts, vocab), dtype)
    for r in range(requests):
        for i in range(counts[r]):
            if rng.random() < 0.7:
                tokens[r, i] = int(np.argmax(host[start[r] + i]))
            if with_law and rng.random() < 0.7:  # a draft model that is nearly the target
                row = host[start[r] + i] + rng.standard_normal(vocab).astype(np.float32) * 0.3
                law[r, i] = torch.tensor(row, device="cuda").to(dtype)
                law_host[r, i] = _np(law[r, i].float())
    return start, logits, host, tokens, law, law_host, rng.random((requests, drafts + 1)).astype(np.float32)


def _check_verify(start, logits, host, tokens, law, law_host, uniforms, temperature):
    want, count = oracle.verify(host, tokens, start, uniforms, law_host, temperature)
    heat = None if temperature is None else torch.tensor(np.asarray(temperature, np.float32), device="cuda")
    got, accepted = _ops().verify_draft(logits, _i64(tokens), _i32(start), torch.tensor(uniforms, device="cuda"),
                                        draft_logits=law, temperature=heat)
    np.testing.assert_array_equal(_np(accepted), count)
    np.testing.assert_array_equal(_np(got), want)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [1, 2, 255, 1000, 2047, 2049, 8191, 8192, 8193, 50001, 200003])
@pytest.mark.parametrize("with_law", [False, True])
def test_verify_of_ragged_drafts(dtype, vocab, with_law):
    rng = np.random.default_rng(vocab)
    drafts = _drafted(rng, [3, 0, 1, 3, 2, 3, 3, 1], 3, vocab, dtype, with_law)
    _check_verify(*drafts, None)
    _check_verify(*drafts, [0.0, 1.0, 0.7, 1.3, 0.0, 0.2, 2.5, 1.0])
    _check_verify(*drafts, np.linspace(0.05, 4, 8))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [262143, 262144, 262145, 300001, 600000])
@pytest.mark.parametrize("with_law", [False, True])
def test_verify_of_large_vocabularies(dtype, vocab, with_law):
    # more chunks than a wave keeps in registers; laws whose weight is all behind them, a drafted token among it
    rng = np.random.default_rng(vocab)
    start, logits, host, tokens, law, law_host, uniforms = _drafted(rng, [2, 0, 1, 2], 2, vocab, dtype, with_law)
    behind = min(262144, vocab - 1)
    for t in (logits[1], logits[3], logits[4:6], *(() if law is None else (law[0], law[2]))):
        t[..., :behind] -= 40.0
    tokens[0, 0], tokens[2, 0] = vocab - 1, behind
    if with_law:                    # both fall: the draft is all but sure of them
        law[0, 0, vocab - 1], law[2, 0, behind] = 60.0, 60.0
        law_host = _np(law.float())
    host = _np(logits.float())
    for row in (uniforms, np.full_like(uniforms, 1 - 2.0 ** -24), np.full_like(uniforms, 0.5)):
        state = start, logits, host, tokens, law, law_host, row
        _check_verify(*state, [1.0, 0.7, 1.3, 0.0])
    _check_verify(*state, None)


@pytest.mark.parametrize("drafts", [0, 1, 5, 62])
@pytest.mark.parametrize("with_law", [False, True])
def test_verify_of_any_number_of_drafts(drafts, with_law):
    rng = np.random.default_rng(drafts)
    counts = [drafts, 0, drafts // 2]
    state = _drafted(rng, counts, drafts, 300, torch.float32, with_law)
    _check_verify(*state, None)
    _check_verify(*state, [1.0, 0.5, 0.3])
    small = (state[6] * 1e-3).astype(np.float32)  # nearly everything stands
    _check_verify(*state[:6], small, [1.0, 0.5, 0.3])


def test_verify_of_the_ends_of_the_random_numbers():
    rng = np.random.default_rng(2)
    state = list(_drafted(rng, [2, 2, 2, 2], 2, 20000, torch.bfloat16, True))
    for value in (0.0, np.float32(1 - 2 ** -24), 1.0):
        state[6] = np.full((4, 3), value, np.float32)
        _check_verify(*state, [0.5, 1.0, 1.0, 3.0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_verify_of_infinite_and_missing_logits(dtype):
    rng = np.random.default_rng(3)
    start, logits, host, tokens, _, _, uniforms = _drafted(rng, [1] * 8, 1, 9000, dtype, False)
    rows = [np.nan, -np.inf, np.inf]
    for r, value in enumerate(rows):
        logits[2 * r], logits[2 * r + 1, ::2] = value, value           # whole rows; every other token
    logits[6, 17], logits[8, 8999], logits[10, 3] = np.inf, np.nan, -np.inf
    logits[12, :8192], logits[14, 8192:] = -np.inf, np.nan             # a chunk without any
    host = _np(logits.float())
    tokens[:, 0] = [5, 5, 5, 17, 8999, 3, 8995, 2]
    law, _ = _logits(rng, (8, 1, 9000), dtype)
    law[2], law[5, 0, 3] = -np.inf, -np.inf
    for heat in (None, [1.0] * 8, [np.inf] * 8, [1e-30] * 8, [np.nan, -1.0, -np.inf, 0.0] * 2):
        _check_verify(start, logits, host, tokens, None, None, uniforms, heat)
        _check_verify(start, logits, host, tokens, law, _np(law.float()), uniforms, heat)


def test_verify_of_ties_takes_the_first():
    logits = torch.zeros((4, 20000), dtype=torch.bfloat16, device="cuda")
    logits[0, [300, 9000, 19000]] = 2.0
    logits[1, [19999, 8192]] = 1.0
    host = _np(logits.float())
    tokens = np.array([[300, 9000], [0, 0]])
    start, uniforms = np.array([0, 3, 4]), np.full((2, 3), 0.5, np.float32)
    _check_verify(start, logits, host, tokens, None, None, uniforms, None)


def test_verify_leaves_drafts_outside_the_vocabulary_out():
    rng = np.random.default_rng(4)
    start, logits, host, tokens, law, law_host, uniforms = _drafted(rng, [2, 2, 2], 2, 500, torch.float32, True)
    tokens[0, 0], tokens[1, 1], tokens[2, 0] = 500, -1, 2 ** 40
    for heat in (None, [1.0, 1.0, 1.0]):
        _check_verify(start, logits, host, tokens, None, None, uniforms, heat)
        _check_verify(start, logits, host, tokens, law, law_host, uniforms, heat)


def test_verify_of_requests_without_rows_and_of_strided_logits():
    rng = np.random.default_rng(5)
    start, logits, host, tokens, law, law_host, uniforms = _drafted(rng, [2, 1], 2, 700, torch.bfloat16, True)
    start = np.array([0, 0, 3, 3, 5])
    tokens, uniforms = np.repeat(tokens, 2, 0), np.repeat(uniforms, 2, 0)
    law, law_host = law.repeat_interleave(2, 0), np.repeat(law_host, 2, 0)
    wide = torch.zeros((7, 901), dtype=torch.bfloat16, device="cuda")     # odd rows, and rows behind the last
    wide[:5, 1:701] = logits
    steps = torch.zeros((2, 4, 701), dtype=torch.bfloat16, device="cuda")  # a draft model's rows, step by step
    steps[..., 1:] = law.transpose(0, 1)
    _check_verify(start, wide[:, 1:701], host, tokens, steps[..., 1:].transpose(0, 1), law_host, uniforms, [1.0, 0.8, 0.0, 1.2])


def test_verify_replays_in_a_graph():
    rng = np.random.default_rng(6)
    ops = _ops()
    start, logits, host, tokens, law, law_host, uniforms = _drafted(rng, [2, 2, 2], 2, 9000, torch.bfloat16, True)
    d = [logits, _i64(tokens), _i32(start), torch.tensor(uniforms, device="cuda")]
    heat = torch.tensor([1.0, 0.0, 0.7], device="cuda")
    out = (torch.empty((3, 3), dtype=torch.int64, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda"))
    ops.verify_draft(*d, draft_logits=law, temperature=heat, tokens=out[0], accepted=out[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.verify_draft(*d, draft_logits=law, temperature=heat, tokens=out[0], accepted=out[1])
    for i in range(5):
        uniforms = rng.random((3, 3)).astype(np.float32)
        d[3].copy_(torch.tensor(uniforms))
        out[0].fill_(-5)
        graph.replay()
        want, count = oracle.verify(host, tokens, start, uniforms, law_host, [1.0, 0.0, 0.7])
        np.testing.assert_array_equal(_np(out[0]), want)
        np.testing.assert_array_equal(_np(out[1]), count)


def test_verify_draws_from_the_target():
    # over many random numbers the drawn tokens follow the target, whatever the draft: counts within 5 deviations
    rng = np.random.default_rng(7)
    vocab, requests = 12, 4000
    z, y = rng.standard_normal(vocab).astype(np.float32), rng.standard_normal(vocab).astype(np.float32)
    p = oracle.law(z, 1.0)
    q = oracle.law(y, 1.0)
    logits = torch.tensor(z, device="cuda").expand(2 * requests, vocab)
    law = torch.tensor(y, device="cuda").expand(requests, 1, vocab)
    tokens = rng.choice(vocab, size=(requests, 1), p=q)
    got, accepted = _ops().verify_draft(
        logits, _i64(tokens), _i32(2 * np.arange(requests + 1)),
        torch.tensor(rng.random((requests, 2)).astype(np.float32), device="cuda"), draft_logits=law,
        temperature=torch.ones(requests, device="cuda"))
    counts = np.bincount(_np(got)[:, 0], minlength=vocab)
    assert (np.abs(counts - requests * p) <= 5 * np.sqrt(requests * p * (1 - p)) + 1).all()
    assert abs(float(accepted.float().mean()) - np.minimum(p, q).sum()) < 5 * 0.5 / np.sqrt(requests)


# ---------------------------------------------------------------- together
def test_serving_steps_over_one_cache():
    """Prompts in chunks, decodes and drafted tokens of four requests through a packed layer: every operator of a
    step takes what the one before it left, requests keep what stood and pages are handed out as they grow."""

    ops = _ops()
    rng = np.random.default_rng(0)
    hq, hkv, dim, hidden, vocab, page, requests = 4, 2, 64, 256, 512, 16, 4
    width = (hq + 2 * hkv) * dim
    weights = {name: ops.w4_quantize(to_gpu_bf16(bf16_normal(rng, shape, 0.06)), 64)
               for name, shape in (("qkv", (width, hidden)), ("out", (hidden, hq * dim)), ("head", (vocab, hidden)))}
    embedding, norm = to_gpu_bf16(bf16_normal(rng, (vocab, hidden))), torch.ones(hidden, dtype=torch.bfloat16, device="cuda")
    angle = np.arange(256)[:, None] / 1e4 ** ((np.arange(dim) % (dim // 2)) * 2 / dim)
    cos, sin = (torch.tensor(f(angle), device="cuda").to(torch.bfloat16) for f in (np.cos, np.sin))
    (keys, values), _ = _cache(rng, 40, hkv, page, dim, "dense")
    tables = _i32(np.full((requests, 12), -1))
    counts, free, start = _i32([0] * requests), _i32(rng.permutation(40)), _i32([0])
    texts = [list(rng.integers(0, vocab, n)) for n in (50, 3, 17, 90)]
    context, seen = [0] * requests, [[[] for _ in range(requests)] for _ in range(2)]
    for number in range(9):
        chunks = []
        for r, text in enumerate(texts):
            left = len(text) - context[r]
            if left > 1:
                chunks.append(text[context[r]: context[r] + 32])
            else:  # the last token and up to three guesses
                chunks.append(text[-1:] + list(rng.integers(0, vocab, 3 if number % 2 else 0)))
        new = [len(c) for c in chunks]
        total = sum(new)
        step = ops.paged_tables(_i32(context), _i32(new), tables, counts, free, start, page_size=page, max_tokens=total + 5)
        counts, start = step.page_counts, step.free_start
        ids = _i64(sum(chunks, []) + [0] * 5)
        x = ops.embedding(embedding, ids)
        qkv = ops.w4_matmul(ops.rms_norm(x, norm, 1e-6), *weights["qkv"], 64)
        q = ops.paged_rope_append(qkv, step.positions, step.slots, cos, sin, keys, values, query_heads=hq)
        mixed = ops.paged_attention(q, keys, values, tables, step.query_start, step.kv_lens, out=torch.zeros_like(x))
        # the rows as they were written, then the attention over every row that stood so far, without pages
        host = from_gpu_bf16(qkv).astype(np.float64).reshape(-1, hq + 2 * hkv, dim)
        at = np.concatenate([np.arange(c, c + n) for c, n in zip(context, new)])
        turned, turns = oracle.rope(host[:total, : hq + hkv],
                                    *(from_gpu_bf16(t).astype(np.float64)[at][:, None] for t in (cos, sin)))
        slots = _np(step.slots)[:total]
        now = [from_gpu_bf16(c)[slots // page, :, slots % page].astype(np.float64) for c in (keys, values)]
        rows = np.concatenate([from_gpu_bf16(q)[:total].astype(np.float64), now[0]], 1)
        assert (np.abs(rows - turned) <= HALF * np.abs(turned) + 2.0 ** -22 * turns).all()
        np.testing.assert_array_equal(now[1], host[:total, hq + hkv:])
        first = 0
        for r, n in enumerate(new):
            for side, fresh in zip(seen, now):
                side[r] = side[r][: context[r]] + list(fresh[first: first + n])
            k, v = (np.array(side[r])[None].transpose(0, 2, 1, 3) for side in seen)  # one page that holds them all
            want, size, _ = oracle.attention(rows[first: first + n, :hq], k, v, np.zeros((1, 1), int), [0, n],
                                             [context[r] + n])
            got = from_gpu_bf16(mixed)[first: first + n].astype(np.float64)
            assert (np.abs(got - want) <= attention_bound(want, size)).all()
            first += n
        assert not bool(mixed[total:].any())
        x = ops.w4_matmul(mixed, *weights["out"], 64, residual=x)
        logits = ops.w4_matmul(ops.rms_norm(x, norm, 1e-6), *weights["head"], 64)
        # a prompt's chunk has no drafts: its last row alone is judged
        drafted = [n - 1 if len(t) - c <= 1 else 0 for n, t, c in zip(new, texts, context)]
        ends = np.cumsum(new)
        rows = np.concatenate([np.arange(e - 1 - d, e) for e, d in zip(ends, drafted)])
        judged = logits[_i64(rows)]
        drafts = np.zeros((requests, 3), np.int64)
        for r, d in enumerate(drafted):
            drafts[r, :d] = chunks[r][1:] if d else []
            if d:  # the first guess is right more often than chance would have it
                best = int(judged[int(np.sum(drafted[:r])) + r].float().argmax())
                drafts[r, 0] = best if number % 4 == 1 else drafts[r, 0]
        uniforms = rng.random((requests, 4)).astype(np.float32)
        heat = [0.0, 1.0, 0.0, 0.5]
        begin = np.concatenate([[0], np.cumsum(np.array(drafted) + 1)])
        tokens, accepted = ops.verify_draft(judged, _i64(drafts), _i32(begin), torch.tensor(uniforms, device="cuda"),
                                            temperature=torch.tensor(heat, device="cuda"))
        expected, count = oracle.verify(_np(judged.float()), drafts, begin, uniforms, None, heat)
        np.testing.assert_array_equal(_np(tokens), expected)
        np.testing.assert_array_equal(_np(accepted), count)
        for r in range(requests):
            left = len(texts[r]) - context[r]
            if left > new[r]:      # the prompt goes on
                context[r] += new[r]
            elif left > 1:         # the prompt is in the cache: its first token follows
                context[r] += new[r]
                texts[r].append(int(expected[r, 0]))
            else:                  # what stood of the guesses that were fed (the first may have been put in later)
                stood = 0
                while stood < count[r] and drafts[r, stood] == chunks[r][1 + stood]:
                    stood += 1
                context[r] += 1 + stood
                texts[r] += [int(t) for t in expected[r, : stood + 1]]
    assert int(counts.sum()) == int(start) and len(set(_np(tables)[_np(tables) >= 0])) == int(start)


def test_a_captured_step_of_every_operator_replays():
    """Decodes and drafted tokens of six requests: the step captured once against the same steps called one by one."""

    ops = _ops()
    hq, hkv, dim, vocab, page, requests, room, drafts = 8, 2, 64, 5000, 16, 6, 24, 3
    device = dict(device="cuda")

    def state():
        rng = np.random.default_rng(19)
        (keys, values), _ = _cache(rng, 400, hkv, page, dim, "dense")
        context = np.array([0, 15, 16, 700, 3, 250])
        counts = -(-context // page)
        tables, order, at = np.full((requests, 64), -1, np.int32), rng.permutation(400), 0
        for r, count in enumerate(counts):
            tables[r, :count], at = order[at: at + count], at + count
        angle = rng.random((1024, dim)) * 6
        cos, sin = (torch.tensor(f(angle), **device).to(torch.bfloat16) for f in (np.cos, np.sin))
        return dict(context=_i32(context), new=_i32([1] * requests), tables=_i32(tables), counts=_i32(counts),
                    free=_i32(order[at:]), start=_i32([0]), keys=keys, values=values, cos=cos, sin=sin,
                    qkv=torch.zeros((room, (hq + 2 * hkv) * dim), dtype=torch.bfloat16, **device),
                    logits=torch.zeros((room, vocab), **device), drafts=_i64(np.zeros((requests, drafts))),
                    uniforms=torch.zeros((requests, drafts + 1), **device),
                    heat=torch.tensor([0.0, 1.0, 0.7, 0.0, 2.0, 1.0], **device),
                    error=torch.zeros(1, dtype=torch.int32, **device),
                    out=torch.zeros((room, hq * dim), dtype=torch.bfloat16, **device),
                    q=torch.zeros((room, hq, dim), dtype=torch.bfloat16, **device))

    def run(d):
        step = d.get("step")
        step = ops.paged_tables(d["context"], d["new"], d["tables"], d["counts"], d["free"], d["start"],
                                page_size=page, max_tokens=room, step=step, error=d["error"])
        ops.paged_rope_append(d["qkv"], step.positions, step.slots, d["cos"], d["sin"], d["keys"], d["values"],
                              query_heads=hq, q_out=d["q"], error=d["error"])
        ops.paged_attention(d["q"], d["keys"], d["values"], d["tables"], step.query_start, step.kv_lens, out=d["out"],
                            max_query_len=drafts + 1)
        tokens, accepted = ops.verify_draft(d["logits"], d["drafts"], step.query_start, d["uniforms"],
                                            temperature=d["heat"])
        return step, tokens, accepted

    one, two = state(), state()
    spare = state()
    spare["step"] = run(spare)[0]._replace(page_counts=spare["counts"], free_start=spare["start"])
    two["step"] = ops.PagedStep(*(torch.zeros_like(t) for t in spare["step"][:4]), two["counts"], two["start"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(two)
    rng = np.random.default_rng(20)
    for _ in range(12):
        new = rng.integers(0, drafts + 2, requests)
        qkv, logits = bf16_normal(rng, tuple(one["qkv"].shape)), rng.standard_normal((room, vocab)) * 3
        guesses, uniforms = rng.integers(0, vocab, (requests, drafts)), rng.random((requests, drafts + 1))
        for d in (one, two):
            d["new"].copy_(_i32(new))
            d["qkv"].copy_(to_gpu_bf16(qkv))
            d["logits"].copy_(torch.tensor(logits, **device))
            d["drafts"].copy_(_i64(guesses))
            d["uniforms"].copy_(torch.tensor(uniforms, **device))
        step, tokens, accepted = run(one)
        one["counts"], one["start"] = step.page_counts, step.free_start
        graph.replay()
        for a, b in zip((*step, tokens, accepted), (*captured[0], *captured[1:])):
            assert bool((a == b).all())
        for name in ("tables", "keys", "values", "q", "out", "error"):
            assert bool((one[name] == two[name]).all()), name
        # what stood of each request is kept
        context = torch.where(one["new"] > 0, step.kv_lens - one["new"] + accepted + 1, step.kv_lens)
        for d in (one, two):
            d["context"].copy_(context)
    assert int(one["error"]) == 0
