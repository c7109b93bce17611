"""The paged-cache operators without a GPU: their plain restatements' own cases, what the entry points refuse on the
host and the exactness of the verification's exponential."""

from __future__ import annotations

import ctypes
import math
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

from aotolith_amd import _lib, ops
from oracle import paged as oracle

GOOD = ctypes.c_void_p(4096)  # an address that no entry point may read: each refuses first


def _refused(status, code, word):
    assert status == code
    assert word in _lib.last_error()


def _tables(**changes):
    a = dict(context=GOOD, new=GOOD, tables=GOOD, stride=8, counts=GOOD, free=GOOD, start=GOOD, requests=4, blocks=8,
             count=100, page=16, tokens=32, query_start=GOOD, kv=GOOD, positions=GOOD, slots=GOOD, counts_out=GOOD,
             start_out=GOOD) | changes
    return _lib.library().aoto_hip_paged_tables(*a.values(), None, None)


@pytest.mark.parametrize("name", ["context", "new", "tables", "counts", "free", "start", "query_start", "kv",
                                  "positions", "slots", "counts_out", "start_out"])
def test_tables_refuse_null_pointers(name):
    _refused(_tables(**{name: None}), _lib.AOTO_ERR_ARGUMENT, "null pointer")


@pytest.mark.parametrize("changes,code", [
    (dict(requests=0), 1), (dict(blocks=0), 1), (dict(count=-1), 1), (dict(page=0), 1), (dict(tokens=-1), 1),
    (dict(stride=7), 1), (dict(blocks=2 ** 20 + 1, stride=2 ** 21), 4), (dict(page=2 ** 20 + 1), 4),
    (dict(tokens=2 ** 30), 4)])
def test_tables_refuse_shapes(changes, code):
    _refused(_tables(**changes), code, "paged_tables")


def _append(**changes):
    a = dict(qkv=GOOD, row=1152, positions=GOOD, slots=GOOD, cos=GOOD, sin=GOOD, rows=100, keys=GOOD, values=GOOD,
             page_stride=2048, head_stride=1024, slot_stride=64, pages=4, page=16, tokens=3, heads=14, kv_heads=2,
             dim=64, q=GOOD) | changes
    return _lib.library().aoto_hip_paged_rope_append(*a.values(), None, None)


@pytest.mark.parametrize("changes,code", [
    (dict(qkv=None), 1), (dict(positions=None), 1), (dict(slots=None), 1), (dict(cos=None), 1), (dict(sin=None), 1),
    (dict(keys=None), 1), (dict(values=None), 1), (dict(q=None), 1), (dict(rows=0), 1), (dict(pages=0), 1),
    (dict(page=0), 1), (dict(page=2 ** 20 + 1), 1), (dict(tokens=0), 1), (dict(heads=0), 1), (dict(kv_heads=0), 1),
    (dict(dim=24), 4), (dict(row=1153), 1), (dict(slot_stride=65), 1), (dict(page_stride=4), 1),
    (dict(keys=ctypes.c_void_p(4104)), 1), (dict(qkv=ctypes.c_void_p(4098)), 1), (dict(q=ctypes.c_void_p(4104)), 1)])
def test_append_refuses(changes, code):
    _refused(_append(**changes), code, "paged_rope_append")


def _attention(**changes):
    a = dict(q=GOOD, q_token=896, q_head=64, keys=GOOD, values=GOOD, page_stride=2048, head_stride=1024,
             slot_stride=64, pages=4, page=16, tables=GOOD, stride=8, blocks=8, start=GOOD, kv=GOOD, tokens=3,
             requests=2, heads=14, kv_heads=2, dim=64, causal=1, scale=0.125, rows=0, length=0, workspace=GOOD,
             out=GOOD) | changes
    return _lib.library().aoto_hip_paged_attention(*a.values(), None)


@pytest.mark.parametrize("changes,code", [
    (dict(q=None), 1), (dict(keys=None), 1), (dict(values=None), 1), (dict(tables=None), 1), (dict(start=None), 1),
    (dict(kv=None), 1), (dict(out=None), 1), (dict(tokens=0), 1), (dict(requests=0), 1), (dict(blocks=0), 1),
    (dict(stride=7), 1), (dict(heads=13), 1), (dict(kv_heads=0), 1), (dict(dim=96), 4), (dict(q_head=68), 1),
    (dict(q=ctypes.c_void_p(4104)), 1), (dict(out=ctypes.c_void_p(4104)), 1), (dict(values=ctypes.c_void_p(4112 + 8)), 1),
    (dict(head_stride=1028), 1), (dict(rows=-1), 1), (dict(length=-1), 1)])
def test_attention_refuses(changes, code):
    _refused(_attention(**changes), code, "paged_attention")


@pytest.mark.parametrize("changes,code", [
    *[(dict(scale=v), 1) for v in (0.0, -0.125, math.inf, math.nan)],
    (dict(page_stride=2 ** 32), 4), (dict(page_stride=-2048), 4), (dict(slot_stride=2 ** 26), 4),
    (dict(slot_stride=-64), 4), (dict(slot_stride=2 ** 60), 4), (dict(slot_stride=2 ** 62), 4),  # page times it wraps
    (dict(blocks=2 ** 24 + 1, stride=2 ** 25), 4), (dict(heads=129, kv_heads=1), 4)])
def test_attention_refuses_what_its_addresses_do_not_reach(changes, code):
    _refused(_attention(**changes), code, "paged_attention")


@pytest.mark.parametrize("changes", [
    dict(requests=21846), dict(requests=13108, law=GOOD), dict(requests=65536, drafts=0)])
def test_verify_refuses_more_rows_than_a_launch_has(changes):
    # requests * (drafts + 1), with a draft model's logits requests * (2 drafts + 1): 65536 and more
    _refused(_verify(**changes), _lib.AOTO_ERR_UNSUPPORTED, "requests of")


def _verify(**changes):
    a = dict(logits=GOOD, f32=0, row=1000, rows=9, vocab=1000, drafts_in=GOOD, law=None, law_request=0, law_row=0,
             start=GOOD, uniforms=GOOD, temperature=GOOD, requests=3, drafts=2, workspace=GOOD, out=GOOD,
             accepted=GOOD) | changes
    return _lib.library().aoto_hip_verify_draft(*a.values(), None)


@pytest.mark.parametrize("changes,code", [
    (dict(logits=None), 1), (dict(drafts_in=None), 1), (dict(start=None), 1), (dict(uniforms=None), 1),
    (dict(workspace=None), 1), (dict(out=None), 1), (dict(accepted=None), 1), (dict(rows=0), 1), (dict(vocab=0), 1),
    (dict(requests=0), 1), (dict(drafts=-1), 1), (dict(drafts=63), 4), (dict(vocab=2 ** 30 + 1), 4), (dict(logits=ctypes.c_void_p(4097)), 1),
    (dict(f32=1, logits=ctypes.c_void_p(4098)), 1), (dict(law=ctypes.c_void_p(4097)), 1)])
def test_verify_refuses(changes, code):
    _refused(_verify(**changes), code, "verify_draft")


def test_workspaces_of_empty_calls_are_empty():
    lib = _lib.library()
    assert lib.aoto_hip_verify_draft_workspace(0, 3, 100) == 0
    assert lib.aoto_hip_verify_draft_workspace(2, -1, 100) == 0
    assert lib.aoto_hip_verify_draft_workspace(2, 3, 100) > 0
    assert lib.aoto_hip_paged_attention_workspace(0, 1, 8, 16, 14, 2, 64, 0, 0) == 0


@pytest.mark.parametrize("call", [
    lambda i, b, l: ops.paged_tables(i, i, b, i, i, i, page_size=16, max_tokens=4),
    lambda i, b, l: ops.paged_rope_append(l, i.long(), i.long(), l, l, l, l, query_heads=1),
    lambda i, b, l: ops.paged_attention(l, l, l, b, i, i),
    lambda i, b, l: ops.verify_draft(l, b.long(), i, i.float())])
def test_host_tensors_are_refused(call):
    with pytest.raises(ValueError, match="on the GPU"):
        call(torch.zeros(1, dtype=torch.int32), torch.zeros((1, 1), dtype=torch.int32),
             torch.zeros((1, 1), dtype=torch.bfloat16))


# ---------------------------------------------------------------- the restatements
def test_tables_of_the_restatement():
    # 16-token pages: 20 tokens grow by 13 into a third page, 16 by one into a second
    got = oracle.tables([20, 16], [13, 1], np.array([[7, 8, -1], [5, -1, -1]]), [2, 1], np.array([9, 4, 6]), 0, 16, 16)
    np.testing.assert_array_equal(got[0], [0, 13, 14])
    np.testing.assert_array_equal(got[1], [33, 17])
    np.testing.assert_array_equal(got[2][:14], list(range(20, 33)) + [16])
    np.testing.assert_array_equal(got[3], [8 * 16 + 4 + i for i in range(12)] + [9 * 16, 4 * 16, -1, -1])
    np.testing.assert_array_equal(got[4], [[7, 8, 9], [5, 4, -1]])
    np.testing.assert_array_equal(got[5], [3, 2])
    assert got[6] == 2 and got[7] == 0


def test_verification_of_the_restatement_keeps_the_target():
    # summed over the draft's law and the random numbers, the first token has the target's law: p = q-part + rest-part
    p, q = np.array([0.5, 0.3, 0.2, 0.0]), np.array([0.1, 0.6, 0.1, 0.2])
    with np.errstate(divide="ignore"):
        logits, law = np.log(p)[None].repeat(2, 0), np.log(q)[None, None]
    total = np.zeros(4)
    steps = (np.arange(400) + 0.5) / 400
    for x in range(4):
        for u in steps:
            token, count = oracle.verify(logits, np.array([[x]]), [0, 2], np.array([[u, 0.5]]), law, [1.0])
            if count[0]:
                total[x] += q[x] / 400
            else:
                rest = np.maximum(p - q, 0)
                total += q[x] / 400 * rest / rest.sum()
    np.testing.assert_allclose(total, p, atol=2e-3)  # a step of 1/400 on each of the drafts that may fall


def test_attention_of_the_restatement_by_hand():
    # two keys of equal score: the mean of their values; the row before sees the first alone
    keys, values = np.zeros((1, 1, 4, 2)), np.arange(8.0).reshape(1, 1, 4, 2)
    out, _, written = oracle.attention(np.ones((3, 1, 2)), keys, values, np.array([[0]]), [0, 2], [2])
    np.testing.assert_allclose(out, [[0, 1], [1, 2], [0, 0]])
    assert written.tolist() == [True, True, False]


def test_exponential_series_is_exact_to_the_last_bits():
    # the series that the verification takes 2^x with, its rounding of x by a sum with 1.5 * 2^52 included: below
    # 4 steps of 2^-53 (a remainder of 1.7e-16 over 2^f >= 0.7, and the last products' roundings)
    x = -np.concatenate([np.linspace(0, 60, 20001), np.linspace(0, 1, 5001), [1000.0, 1999.5]])
    whole = (x + 6755399441055744.0) - 6755399441055744.0
    f = x - whole
    assert np.abs(f).max() <= 0.5
    s = np.zeros_like(f)
    for k in range(12, -1, -1):
        s = s * f + np.float64(np.log(np.longdouble(2)) ** k / np.longdouble(math.factorial(k)))
    got = np.ldexp(s, whole.astype(int))
    exact = np.exp2(x.astype(np.longdouble)).astype(np.float64)
    assert np.all(np.abs(got - exact) <= 4 * 2.0 ** -53 * exact)
    assert got[-1] == 0.0  # what weighs less than any number weighs nothing


# ---------------------------------------------------------------- the verification's exponential, as the kernels have it
_EXP2 = r"""
#include <cmath>
#include <cstdint>
#include <cstring>
using std::fma; using std::ldexp;
#define AOTO_DEVICE static inline
static inline uint64_t bits(double v) { uint64_t b; std::memcpy(&b, &v, 8); return b; }
static inline int __double2loint(double v) { return (int)(uint32_t)bits(v); }
static inline int __double2hiint(double v) { return (int)(uint32_t)(bits(v) >> 32); }
static inline double __hiloint2double(int hi, int lo) {
  const uint64_t b = (uint64_t)(uint32_t)hi << 32 | (uint32_t)lo;
  double v;
  std::memcpy(&v, &b, 8);
  return v;
}
#include "exp2.h"
extern "C" void powers(const double* d, double heat32, int n, double* of, double* added, double* table) {
  for (int j = 0; j < 32; ++j) table[j] = aoto::exp2_32nds(j);
  for (int i = 0; i < n; ++i) of[i] = aoto::exp2_of(d[i], heat32, table);
  for (int i = 0; i < n; ++i) added[i] = aoto::exp2_added(d[i], heat32, table, 0.0);
}
"""


@pytest.mark.parametrize("heat32", [32.0, 32 * math.log2(math.e), 32 * math.log2(math.e) / 0.7, 1e-3, 3e5])
def test_exponentials_of_the_verification(tmp_path, heat32):
    """``csrc/exp2.h`` compiled for the host: 2^(d heat32 / 32) within 27 steps of 2^-53.

    The series' remainder is (ln 2 / 64)^6 / 6! = 2.24e-15 = 20.2 steps, over e^f >= 0.989 20.4. A table entry is off by
    3: its y by 2 roundings of up to 0.69, its last two products and sums by 1 + 0.4, the others by less than 0.2. The
    series' last sum and the product of the two are a rounding each; its other terms, of a factor of 0.011, 0.1; f, once
    rounded at 1/2, 0.02. The exact value's own rounding here adds half a step: 20.4 + 3 + 2 + 0.12 + 0.5 < 27.
    """

    compiler = shutil.which("g++") or shutil.which("c++")
    if compiler is None:
        pytest.skip("no host compiler")
    (tmp_path / "powers.cpp").write_text(_EXP2)
    include = os.path.join(os.path.dirname(ops.__file__), "csrc")
    subprocess.run([compiler, "-O1", "-std=c++17", "-ffp-contract=off", "-fPIC", "-shared", "-I" + include,
                    str(tmp_path / "powers.cpp"), "-o", str(tmp_path / "powers.so")], check=True)
    rng = np.random.default_rng(0)
    x = -np.concatenate([np.linspace(0, 60, 40001), np.linspace(0, 2, 20001), rng.random(40000) * 999, [0.0, 1.0, 999.9]])
    d = x * 32 / heat32
    of, added, table = np.empty_like(d), np.empty_like(d), np.empty(32)
    pointer = ctypes.POINTER(ctypes.c_double)
    powers = ctypes.CDLL(str(tmp_path / "powers.so")).powers
    powers.argtypes = [pointer, ctypes.c_double, ctypes.c_int, pointer, pointer, pointer]
    powers(*(v.ctypes.data_as(pointer) if isinstance(v, np.ndarray) else v for v in (d, heat32, len(d), of, added, table)))
    exact = np.exp2(d.astype(np.longdouble) * np.longdouble(heat32) / 32).astype(np.float64)
    step = 2.0 ** -53
    assert (np.abs(of - exact) <= 27 * step * exact).all()
    assert (np.abs(added - exact) <= 27 * step * exact).all()
    entries = np.exp2(np.arange(32, dtype=np.longdouble) / 32).astype(np.float64)
    assert (np.abs(table - entries) <= 3.5 * step * entries).all()
    low = np.array([-1100.0, -2000.0]) * 32 / heat32      # where the floors of the weights lie: nothing
    powers(*(v.ctypes.data_as(pointer) if isinstance(v, np.ndarray) else v for v in (low, heat32, 2, of, added, table)))
    assert (of[:2] == 0.0).all()
