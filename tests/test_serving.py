"""The operators over a 4-bit paged cache, on pages and on logits without a GPU: their plain restatements' own cases and
what the entry points refuse on the host."""

from __future__ import annotations

import ctypes
import math
import sys
import warnings

import numpy as np
import pytest
import torch

import aotolith_amd
from aotolith_amd import _lib, ops
from aotolith_amd.csrc import build
from oracle import serving as oracle

GOOD = ctypes.c_void_p(4096)  # an address that no entry point may read: each refuses first


def _refused(status, code, word):
    assert status == code
    assert word in _lib.last_error()


def _cache(**changes):
    a = dict(keys=4096, values=4096, key_scales=4097, value_scales=4099, page_stride=2048, head_stride=1024,
             slot_stride=64, scale_page_stride=7, scale_head_stride=5, scale_slot_stride=3, pages=4) | changes
    return _lib.MX4_CACHE.pack(*(0 if x is None else x for x in a.values()))


CACHE_REFUSALS = [
    (dict(keys=None), 1), (dict(values=None), 1), (dict(key_scales=None), 1), (dict(value_scales=None), 1),
    (dict(pages=0), 1), (dict(keys=4104), 1), (dict(values=4097), 1), (dict(page_stride=2056), 1),
    (dict(head_stride=8), 1), (dict(slot_stride=65), 1)]


def _append(changed=None, **changes):
    a = dict(qkv=GOOD, row=2048, positions=GOOD, slots=GOOD, cos=GOOD, sin=GOOD, rows=100,
             cache=_cache(**(changed or {})), page=16, tokens=3, heads=12, kv_heads=2, dim=128, q=GOOD) | changes
    return _lib.library().aoto_hip_paged_rope_append_mx4(*a.values(), None, None)


@pytest.mark.parametrize("changes,code", [
    (dict(qkv=None), 1), (dict(positions=None), 1), (dict(slots=None), 1), (dict(cos=None), 1), (dict(sin=None), 1),
    (dict(q=None), 1), (dict(rows=0), 1), (dict(page=0), 1), (dict(page=2 ** 20 + 1), 1), (dict(tokens=0), 1),
    (dict(heads=0), 1), (dict(kv_heads=0), 1), (dict(dim=96), 4), (dict(dim=0), 1), (dict(row=2049), 1),
    (dict(qkv=ctypes.c_void_p(4098)), 1), (dict(q=ctypes.c_void_p(4104)), 1), (dict(heads=2 ** 30), 4)])
def test_append_refuses(changes, code):
    _refused(_append(**changes), code, "paged_rope_append_mx4")


@pytest.mark.parametrize("changes,code", CACHE_REFUSALS)
def test_every_entry_point_refuses_a_bad_cache(changes, code):
    _refused(_append(changes), code, "paged_rope_append_mx4")
    _refused(_unpack(changes), code, "paged_unpack_mx4")
    _refused(_attention(changes), code, "paged_attention_mx4")


def _unpack(changed=None, **changes):
    a = dict(cache=_cache(**(changed or {})), page=16, kv_heads=2, dim=128, keys=GOOD, values=GOOD) | changes
    return _lib.library().aoto_hip_paged_unpack_mx4(*a.values(), None)


@pytest.mark.parametrize("changes,code", [
    (dict(keys=None), 1), (dict(values=None), 1), (dict(keys=ctypes.c_void_p(4100)), 1), (dict(dim=32), 4),
    (dict(page=2 ** 20, kv_heads=16), 4), (dict(cache=None), 1)])
def test_unpack_refuses(changes, code):
    _refused(_unpack(**changes), code, "paged_unpack_mx4")


def _attention(changed=None, **changes):
    a = dict(q=GOOD, q_token=1536, q_head=128, cache=_cache(**(changed or {})), page=16, tables=GOOD, stride=8,
             blocks=8, start=GOOD, kv=GOOD, tokens=3, requests=2, heads=12, kv_heads=2, dim=128, causal=1, scale=0.125,
             rows=0, length=0, workspace=GOOD, out=GOOD) | changes
    return _lib.library().aoto_hip_paged_attention_mx4(*a.values(), None)


@pytest.mark.parametrize("changes,code", [
    (dict(q=None), 1), (dict(tables=None), 1), (dict(start=None), 1), (dict(kv=None), 1), (dict(out=None), 1),
    (dict(cache=None), 1), (dict(tokens=0), 1), (dict(requests=0), 1), (dict(blocks=0), 1), (dict(stride=7), 1),
    (dict(heads=13), 1), (dict(kv_heads=0), 1), (dict(dim=192), 4), (dict(q_head=68), 1),
    (dict(q=ctypes.c_void_p(4104)), 1), (dict(out=ctypes.c_void_p(4104)), 1), (dict(rows=-1), 1), (dict(length=-1), 1),
    *[(dict(scale=v), 1) for v in (0.0, -0.125, math.inf, math.nan)],
    (dict(blocks=2 ** 24 + 1, stride=2 ** 25), 4), (dict(heads=129, kv_heads=1), 4)])
def test_attention_refuses(changes, code):
    _refused(_attention(**changes), code, "paged_attention_mx4")


@pytest.mark.parametrize("changes", [
    dict(page_stride=2 ** 32), dict(page_stride=-2048), dict(slot_stride=2 ** 26), dict(slot_stride=-64),
    dict(slot_stride=2 ** 60), dict(slot_stride=2 ** 62), dict(scale_page_stride=2 ** 32), dict(scale_page_stride=-1),
    dict(scale_slot_stride=2 ** 26 + 1), dict(scale_slot_stride=-1), dict(scale_slot_stride=2 ** 62)])
def test_attention_refuses_what_its_addresses_do_not_reach(changes):
    _refused(_attention(changes), 4, "paged_attention_mx4")


def test_workspaces_of_empty_calls_are_empty():
    lib = _lib.library()
    assert lib.aoto_hip_paged_attention_mx4_workspace(0, 1, 8, 16, 14, 2, 64, 0, 0) == 0
    assert lib.aoto_hip_paged_attention_mx4_workspace(1, 1, 8, 16, 15, 2, 64, 0, 0) == 0
    assert lib.aoto_hip_paged_attention_mx4_workspace(1, 1, 800, 16, 14, 2, 64, 1, 0) > 0


def _fork(**changes):
    a = dict(parents=GOOD, lens=GOOD, tables=GOOD, stride=8, counts=GOOD, shares=GOOD, free=GOOD, start=GOOD,
             requests=4, blocks=8, count=100, pages=50, page=16, lens_out=GOOD, counts_out=GOOD, start_out=GOOD,
             source=GOOD, target=GOOD, plan=GOOD) | changes
    return _lib.library().aoto_hip_paged_fork(*a.values(), None, None)


@pytest.mark.parametrize("changes,code", [
    *[({name: None}, 1) for name in ("parents", "lens", "tables", "counts", "shares", "free", "start", "lens_out",
                                     "counts_out", "start_out", "source", "target", "plan")],
    (dict(requests=0), 1), (dict(blocks=0), 1), (dict(count=-1), 1), (dict(pages=0), 1), (dict(page=0), 1),
    (dict(stride=7), 1), (dict(blocks=2 ** 20 + 1, stride=2 ** 21), 4), (dict(page=2 ** 20 + 1), 4)])
def test_fork_refuses(changes, code):
    _refused(_fork(**changes), code, "paged_fork")


def _tables(**changes):
    a = dict(lens=GOOD, new=GOOD, tables=GOOD, stride=8, counts=GOOD, free=GOOD, start=GOOD, shares=GOOD, requests=2,
             blocks=8, count=10, pages=10, page=16, most=4, query=GOOD, kv=GOOD, positions=GOOD, slots=GOOD,
             counts_out=GOOD, start_out=GOOD) | changes
    return _lib.library().aoto_hip_paged_tables_shared(*a.values(), None, None)


@pytest.mark.parametrize("changes,code", [
    *[({name: None}, 1) for name in ("lens", "new", "tables", "counts", "free", "start", "query", "kv", "positions",
                                     "slots", "counts_out", "start_out")],
    (dict(pages=0), 1), (dict(shares=None, pages=-1), 1), (dict(requests=0), 1), (dict(blocks=0), 1),
    (dict(count=-1), 1), (dict(page=0), 1), (dict(most=-1), 1), (dict(stride=7), 1),
    (dict(blocks=2 ** 20 + 1, stride=2 ** 21), 4), (dict(page=2 ** 20 + 1), 4), (dict(most=2 ** 30), 4)])
def test_tables_of_shared_pages_refuse(changes, code):
    _refused(_tables(**changes), code, "paged_tables")


def _release(**changes):
    a = dict(keep=GOOD, tables=GOOD, stride=8, counts=GOOD, shares=GOOD, free=GOOD, start=GOOD, requests=4, blocks=8,
             count=100, pages=50, page=16, counts_out=GOOD, start_out=GOOD, scratch=GOOD) | changes
    return _lib.library().aoto_hip_paged_release(*a.values(), None, None)


@pytest.mark.parametrize("changes,code", [
    *[({name: None}, 1) for name in ("keep", "tables", "counts", "shares", "free", "start", "counts_out", "start_out",
                                     "scratch")],
    (dict(requests=0), 1), (dict(blocks=0), 1), (dict(count=-1), 1), (dict(pages=0), 1), (dict(page=0), 1),
    (dict(stride=7), 1), (dict(blocks=2 ** 20 + 1, stride=2 ** 21), 4), (dict(page=2 ** 20 + 1), 4)])
def test_release_refuses(changes, code):
    _refused(_release(**changes), code, "paged_release")


def _compact(**changes):
    a = dict(tables=GOOD, stride=8, counts=GOOD, shares=GOOD, free=GOOD, start=GOOD, requests=4, blocks=8, count=100,
             pages=50, source=GOOD, target=GOOD, moved=GOOD, state=GOOD) | changes
    return _lib.library().aoto_hip_paged_compact(*a.values(), None, None)


@pytest.mark.parametrize("changes,code", [
    *[({name: None}, 1) for name in ("tables", "counts", "shares", "free", "start", "source", "target", "moved",
                                     "state")],
    (dict(requests=0), 1), (dict(blocks=0), 1), (dict(count=-1), 1), (dict(pages=0), 1), (dict(stride=7), 1),
    (dict(blocks=2 ** 20 + 1, stride=2 ** 21), 4)])
def test_compact_refuses(changes, code):
    _refused(_compact(**changes), code, "paged_compact")


def _apart(call, names, **changes):
    """`call` with arrays of 64 KB each, apart from each other."""

    at = {name: 2 ** 20 + 2 ** 16 * i for i, name in enumerate(names)}
    at |= {name: at[x] if x in at else x for name, x in changes.items()}
    return call(**{name: ctypes.c_void_p(x) if name in names else x for name, x in at.items()})


FORK_IN = ("parents", "lens", "tables", "counts", "shares", "free", "start")
FORK_OUT = ("lens_out", "counts_out", "start_out", "source", "target", "plan")


@pytest.mark.parametrize("out,other", [(a, b) for a in FORK_OUT for b in FORK_IN + FORK_OUT
                                       if a not in (b, b + "_out")])
def test_fork_refuses_outputs_that_overlap_other_arrays(out, other):
    # a parent's number read after a page's was written there would be a row of no table
    _refused(_apart(_fork, FORK_IN + FORK_OUT, **{out: other}), 1, "overlap")


@pytest.mark.parametrize("changes", [
    dict(source=2 ** 20 + 2 * 2 ** 16 + 4 * 31), dict(target=2 ** 20 + 4 * 2 ** 16 + 4 * 49),
    dict(lens_out=2 ** 20 + 2 ** 16 - 12), dict(counts_out=2 ** 20 + 12 * 2 ** 16 + 28),
    dict(stride=20, source=2 ** 20 + 2 * 2 ** 16 + 4 * 17), dict(stride=12, source=2 ** 20 + 2 * 2 ** 16 + 4 * 9),
    dict(stride=20, source=2 ** 20 + 2 * 2 ** 16 - 12), dict(stride=20, source=2 ** 20 + 2 * 2 ** 16 + 4 * 67)])
def test_fork_refuses_outputs_that_overlap_other_arrays_in_part(changes):
    # the last table entry, the last share, all but the first length, the last entry of the plan; of tables with other
    # columns: the first entry of the second row behind those, and with too few, the first entry, the last
    _refused(_apart(_fork, FORK_IN + FORK_OUT, **changes), 1, "overlap")


COMPACT_IN = ("tables", "counts", "shares", "free", "start")
COMPACT_OUT = ("source", "target", "moved", "state")


@pytest.mark.parametrize("out,other", [(a, b) for a in COMPACT_OUT for b in COMPACT_IN + COMPACT_OUT if a != b])
def test_compact_refuses_outputs_that_overlap_other_arrays(out, other):
    _refused(_apart(_compact, COMPACT_IN + COMPACT_OUT, **{out: other}), 1, "overlap")


def _copy(tensor=None, **changes):
    t = dict(data=4096, planes=2, plane_stride=4096, page_stride=64, page_bytes=64) | (tensor or {})
    a = dict(tensors=_lib.PAGE_TENSOR.pack(*(0 if x is None else x for x in t.values())), count=1, pages=4,
             source=GOOD, target=GOOD, pairs=3) | changes
    return _lib.library().aoto_hip_paged_copy(*a.values(), None, None, None)


@pytest.mark.parametrize("tensor,changes,code", [
    ({}, dict(tensors=None), 1), ({}, dict(source=None), 1), ({}, dict(target=None), 1), ({}, dict(count=0), 1),
    ({}, dict(pages=0), 1), ({}, dict(pairs=0), 1), (dict(data=None), {}, 1), (dict(planes=0), {}, 1),
    (dict(page_bytes=0), {}, 1), (dict(planes=2 ** 20 + 1), {}, 4), (dict(page_bytes=2 ** 35), {}, 4),
    (dict(planes=2 ** 19, page_bytes=2 ** 33), {}, 4)])
def test_copy_refuses(tensor, changes, code):
    _refused(_copy(tensor, **changes), code, "paged_copy")


def test_copy_looks_at_all_tensors_before_it_copies():
    # the launch for the first ones would answer that no code object is loaded
    tensor = [4096, 1, 4096, 4096, 1024]
    for bad, code in ((tensor[:4] + [0], 1), (tensor[:1] + [1 << 21] + tensor[2:], 4)):
        tensors = b"".join(_lib.PAGE_TENSOR.pack(*t) for t in [tensor] * 40 + [bad])
        _refused(_lib.library().aoto_hip_paged_copy(tensors, 41, 4, GOOD, GOOD, 2, None, None, None), code,
                 "paged_copy")


def _adjust(fields=None, **changes):
    names = ("query_start", "history", "history_lens", "prompt_lens", "draft_tokens", "repetition", "presence",
             "frequency", "bias_tokens", "bias_values", "allowed", "history_stride", "draft_stride", "bias_stride",
             "value_stride", "allowed_stride", "history_len", "drafts", "biases")
    assert set(fields or {}) <= set(names)
    arg = _lib.ADJUSTMENTS.pack(*((fields or {}).get(name, 0) for name in names))
    a = dict(logits=GOOD, f32=0, row=1000, rows=9, vocab=1000, requests=3, adjust=arg, out=GOOD,
             out_row=1000) | changes
    return _lib.library().aoto_hip_adjust_logits(*a.values(), None)


@pytest.mark.parametrize("adjust,changes,code", [
    ({}, dict(logits=None), 1), ({}, dict(out=None), 1), ({}, dict(out_row=999), 1), ({}, dict(adjust=None), 1),
    ({}, dict(rows=0), 1), ({}, dict(out_row=1008), 1),
    ({}, dict(vocab=0), 1), ({}, dict(requests=0), 1), ({}, dict(vocab=2 ** 30 + 1), 4), ({}, dict(requests=65536), 4),
    ({}, dict(logits=ctypes.c_void_p(4097)), 1), ({}, dict(f32=1, out=ctypes.c_void_p(4098)), 1),
    (dict(history_len=5), {}, 1), (dict(drafts=2), {}, 1), (dict(biases=2), {}, 1),
    (dict(biases=2, bias_tokens=4096), {}, 1), (dict(history_len=-1), {}, 1), (dict(drafts=-1), {}, 1),
    (dict(history_len=2 ** 30, history=4096), {}, 4)])
def test_adjust_refuses(adjust, changes, code):
    _refused(_adjust(adjust, **changes), code, "adjust_logits")


def _host_cache():
    return ops.PagedMx4(*(torch.zeros((1, 1, 1, n), dtype=torch.uint8) for n in (32, 32, 2, 2)))


@pytest.mark.parametrize("call", [
    lambda i, b, l: ops.paged_rope_append_mx4(l, i.long(), i.long(), l, l, _host_cache(), query_heads=1),
    lambda i, b, l: ops.paged_unpack_mx4(_host_cache()),
    lambda i, b, l: ops.paged_attention_mx4(l, _host_cache(), b, i, i),
    lambda i, b, l: ops.paged_fork(i, i, b, i, i, i, i, page_size=16),
    lambda i, b, l: ops.paged_release(i, b, i, i, i, i, page_size=16),
    lambda i, b, l: ops.paged_compact(b, i, i, i, i),
    lambda i, b, l: ops.paged_copy(l, i, i),
    lambda i, b, l: ops.adjust_logits(l)])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="on the GPU"):
        call(torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32),
             torch.zeros((1, 1), dtype=torch.bfloat16))


def test_other_types_are_refused():
    with pytest.raises(TypeError, match="bf16 or f32"):
        ops.adjust_logits(torch.zeros((1, 8), dtype=torch.float16))
    with pytest.raises(TypeError, match="PagedMx4"):
        ops.paged_unpack_mx4(torch.zeros(1))
    with pytest.raises(ValueError, match="multiples of 64"):
        ops.paged_mx4_cache(4, 2, 16, 96, device="cpu")


def test_a_new_cache_is_zero():
    cache = ops.paged_mx4_cache(3, 2, 5, 128, device="cpu")
    assert [tuple(t.shape) for t in cache] == [(3, 2, 5, 64)] * 2 + [(3, 2, 5, 4)] * 2
    assert all(t.dtype == torch.uint8 and not t.any() for t in cache)
    assert all(t.data_ptr() % 16 == 0 for t in cache[:2]) and cache.keys.stride() == cache.values.stride()


# ---------------------------------------------------------------- the restatements
def test_codes_of_the_restatement():
    x = np.zeros((1, 32))
    x[0, :16] = [7.0, 6.0, 5.0, 5.01, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, 0.26, -0.25, -0.75, -7.0, -3.49, 2.0]
    codes, scales = oracle.mx4_pack(x)
    assert scales.tolist() == [[127]]
    np.testing.assert_array_equal(oracle.mx4_unpack(codes, scales)[0, :16],
                                  [6, 6, 4, 6, 4, 2, 2, 1, 1, 0, 0.5, -0.0, -1, -6, -3, 2])
    x[0, 0] = 7.001  # the next power of two
    assert oracle.mx4_pack(x)[1].tolist() == [[128]]
    for value, byte in ((0.0, 1), (1e-44, 1), (3e38, 252), (np.inf, 255), (np.nan, 255)):
        x[:] = 0
        x[0, 5] = value
        codes, scales = oracle.mx4_pack(x)
        assert scales.tolist() == [[byte]]
        assert np.isnan(oracle.mx4_unpack(codes, scales)).all() == (byte == 255)


def test_pages_of_the_restatement():
    tables = np.array([[4, 7, 2], [-1, -1, -1], [-1, -1, -1], [5, -1, -1]], np.int32)
    shares, free = np.zeros(8, np.int32), np.array([9, 0, 6, 1, 3], np.int32)
    lens, counts, start, source, target, tables, shares, error = oracle.fork(
        [-1, 0, 0, -1], [40, 0, 0, 16], tables, [3, 0, 0, 1], shares, free, 1, 16)
    assert (lens.tolist(), counts.tolist(), int(start[0]), error) == ([40, 40, 40, 16], [3, 3, 3, 1], 3, 0)
    assert (source.tolist(), target.tolist()) == ([-1, 2, 2, -1], [-1, 0, 6, -1])
    assert tables[1].tolist() == [4, 7, 0] and tables[2].tolist() == [4, 7, 6]
    assert shares.tolist() == [0, 0, 0, 0, 2, 0, 0, 2]
    counts, start, free, shares, error = oracle.release([0, 17, -1, 0], tables, counts, shares, free, start[0], 16)
    assert (counts.tolist(), int(start[0]), error) == ([0, 2, 3, 0], 0, 0)
    assert free.tolist() == [5, 2, 0, 1, 3] and shares.tolist() == [0, 0, 0, 0, 1, 0, 0, 1]
    # held: 4, 7, 6; free: 0, 1, 2, 3, 5
    source, target, count, tables, shares, free, error = oracle.compact(tables, counts, shares, free, 0)
    assert (source[:3].tolist(), target[:3].tolist(), int(count[0]), error) == ([4, 6, 7], [0, 1, 2], 3, 0)
    assert tables[1, :2].tolist() == [0, 2] and tables[2].tolist() == [0, 2, 1]
    assert shares.tolist() == [1, 0, 1, 0, 0, 0, 0, 0] and free.tolist() == [3, 4, 5, 6, 7]


def test_pages_of_the_restatement_are_given_back_once():
    tables, shares = np.array([[4, 2], [4, 1]], np.int32), np.array([0, 0, 0, 0, 1], np.int32)
    free = np.array([0, 0, 0, 3], np.int32)
    first = oracle.release([0, 0], tables, [2, 2], shares, free, 3, 16)
    assert first[2].tolist() == [4, 2, 1, 3] and first[1].tolist() == [0] and first[4] == 0
    again = oracle.release([0, -1], tables, [2, 2], first[3], first[2], 0, 16)   # the counts of before
    assert again[2].tolist() == [4, 2, 1, 3] and again[1].tolist() == [0] and again[4] == 128
    assert again[3].tolist() == [0] * 5


def test_rows_of_the_restatement_that_end_inside_a_page_of_others():
    # rows 0, 1, 2 hold pages 4 and 7, row 0 also 2; 1 and 2 are cut inside 7
    tables, shares = np.array([[4, 7, 2], [4, 7, -1], [4, 7, -1]], np.int32), np.array([0] * 8, np.int32)
    shares[[4, 7]] = 2
    free = np.array([1, 3, 5])
    counts, start, free, shares, error = oracle.release([-1, 20, 18], tables, [3, 2, 2], shares, free, 0, 16)
    assert counts.tolist() == [3, 2, 2] and error == 0
    lens, counts, start, source, target, one, left, error = oracle.fork(
        [-1] * 3, [40, 20, 18], tables, counts, shares, free, 0, 16)
    assert (source.tolist(), target.tolist(), start.tolist(), error) == ([-1, 7, 7], [-1, 1, 3], [2], 0)
    assert one.tolist() == [[4, 7, 2], [4, 1, -1], [4, 3, -1]] and left[[4, 7]].tolist() == [2, 0]
    # row 0 ends there too: the last of the three keeps the page; without free pages all stay as they are
    *_, source, target, one, left, error = oracle.fork([-1] * 3, [20, 20, 18], tables, counts, shares, free, 0, 16)
    assert (source.tolist(), one[:, 1].tolist(), left[7], error) == ([7, 7, -1], [1, 3, 7], 0, 0)
    lens, _, start, source, _, one, left, error = oracle.fork(
        [-1] * 3, [20, 20, 18], tables, counts, shares, free, 2, 16)
    assert (source.tolist(), one[:, 1].tolist(), left[7], error) == ([7, -1, -1], [5, 7, 7], 1, 512 + 2)
    assert lens.tolist() == [20, 20, 18] and start.tolist() == [3]


def test_adjustments_of_the_restatement():
    z = np.array([[2.0, -2.0, 1.0, 0.5, 0.0, 3.0]] * 2)
    out, _, written = oracle.adjust(
        z, [0, 2], np.array([[0, 1, 1, 5]]), [3], [1], np.array([[2]]), [2.0], [0.5], [0.25], np.array([[3, 3, -1, 9]]),
        np.array([[7.0, 1.0, 5.0, 5.0]]), np.array([[0b101111], [-1]], np.int32))
    np.testing.assert_array_equal(out[0], [1.0, -5.0, 1.0, 1.5, -np.inf, 3.0])
    np.testing.assert_array_equal(out[1], [1.0, -5.0, -0.25, 1.5, 0.0, 3.0])
    assert written.all()


def test_structs_are_the_headers():
    # pointers, 64-bit strides, 32-bit counts and the room behind them, as the C ABI lays them out
    assert [x.size for x in (_lib.MX4_CACHE, _lib.PAGE_TENSOR, _lib.ADJUSTMENTS)] == [88, 40, 144]


# ---------------------------------------------------------------- the compiled calls
@pytest.mark.parametrize("failure", [RuntimeError("no Python.h"), FileNotFoundError("g++"), ImportError("torch"), None])
def test_a_build_without_the_calls_keeps_the_rest(monkeypatch, tmp_path, failure):
    paths = {name: tmp_path / name for name in ("CODE_OBJECT", "LIBRARY", "CALLS")}
    for name, path in paths.items():
        monkeypatch.setattr(build, name, str(path))
        path.write_text("old")

    def run(command, verbose):
        if failure is not None and any("calls.cpp" in word for word in command):
            raise failure
        with open(command[command.index("-o") + 1], "w") as made:
            made.write("new")

    monkeypatch.setattr(build, "_run", run)
    if failure is None:
        build.build()
    else:
        with pytest.warns(UserWarning, match="_calls.so is not built"):
            build.build()
    assert {name: path.read_text() for name, path in paths.items() if path.exists()} == (
        {name: "new" for name in paths if failure is None or name != "CALLS"})


def test_a_build_that_fails_changes_nothing(monkeypatch, tmp_path):
    paths = [tmp_path / name for name in ("CODE_OBJECT", "LIBRARY", "CALLS")]
    for path in paths:
        monkeypatch.setattr(build, path.name, str(path))
        path.write_text("old")

    def run(command, verbose):
        if any("kernels.hip" in word for word in command):
            raise RuntimeError("build step failed")

    monkeypatch.setattr(build, "_run", run)
    with pytest.raises(RuntimeError, match="build step failed"):
        build.build()
    assert [path.read_text() for path in paths] == ["old"] * 3


class _Calls:
    def __init__(self, built_for):
        if built_for is not None:
            self.built_for = built_for

    def bind(self, *args):
        raise AssertionError("bound")


@pytest.mark.parametrize("built_for", [None, "", "torch 2.9.1 0123456, cpython-310"])
def test_calls_that_were_built_for_another_torch_are_not_bound(monkeypatch, built_for):
    monkeypatch.setattr(aotolith_amd, "_calls", _Calls(built_for), raising=False)
    monkeypatch.setitem(sys.modules, "aotolith_amd._calls", aotolith_amd._calls)
    monkeypatch.setattr(ops, "_calls", ops._Unbound())
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    with pytest.warns(UserWarning, match="another build of torch"):
        ops._bind_calls()
    assert ops._calls.paged_unpack_mx4(None) is None
    with warnings.catch_warnings():
        warnings.simplefilter("error")   # once
        ops._bind_calls()


def test_calls_that_were_built_for_this_torch_are_bound(monkeypatch):
    monkeypatch.setattr(aotolith_amd, "_calls", _Calls(build.calls_built_for()), raising=False)
    monkeypatch.setitem(sys.modules, "aotolith_amd._calls", aotolith_amd._calls)
    monkeypatch.setattr(ops, "_calls", ops._Unbound())
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    with pytest.raises(AssertionError, match="bound"):
        ops._bind_calls()


def test_the_built_calls_say_what_they_were_built_for():
    calls = pytest.importorskip("aotolith_amd._calls")
    assert calls.built_for == build.calls_built_for()
