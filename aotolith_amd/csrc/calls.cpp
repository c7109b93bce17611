// The serving operators' calls from Python without Python's share of the time: arguments checked, outputs allocated and
// the C ABI called in one step. A decode step's kernels run 2 to 10 us each, and the same checks in Python take 5 to 8
// us a call.
//
// Every function gives None where it does not make the call, for an argument that is not what the kernels assume or a
// call that the C ABI refuses: ops.py goes through its own checks then, which give the reason, and makes or refuses the
// call. So nothing is refused here, and nothing is accepted that ops.py would refuse. A call that fails on its way to
// the GPU is an exception and not made a second time: some of its kernels may run.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <utility>
#include <vector>

#include "aoto_hip.h"

namespace {

using at::kBFloat16;
using at::kByte;
using at::kFloat;
using at::kInt;
using at::kLong;
using at::Tensor;

// The entry points of the library that ctypes loaded, by address, and what the call needs from Python.
struct Library {
  decltype(&aoto_hip_code_object_loaded) loaded = nullptr;
  decltype(&aoto_hip_paged_rope_append_mx4) append = nullptr;
  decltype(&aoto_hip_paged_unpack_mx4) unpack = nullptr;
  decltype(&aoto_hip_paged_attention_mx4) attention = nullptr;
  decltype(&aoto_hip_paged_attention_mx4_workspace) attention_workspace = nullptr;
  decltype(&aoto_hip_paged_fork) fork = nullptr;
  decltype(&aoto_hip_paged_release) release = nullptr;
  decltype(&aoto_hip_paged_compact) compact = nullptr;
  decltype(&aoto_hip_paged_copy) copy = nullptr;
  decltype(&aoto_hip_adjust_logits) adjust = nullptr;
  PyObject* raw_stream = nullptr;   // device -> address of its current stream
  PyObject* mx4 = nullptr;          // ops.PagedMx4
  PyObject* check = nullptr;        // status -> its exception
} lib;

// An argument that is not as it should be.
struct Unfit {};
// A Python exception is set.
struct Raised {};

void need(bool fits) {
  if (!fits) throw Unfit();
}

// A call's tensors, all on the device of the first, which is the current one.
struct Call {
  int device = -1;
  const Tensor& tensor(PyObject* object, at::ScalarType type, int dims) {
    need(THPVariable_CheckExact(object));
    const Tensor& t = THPVariable_Unpack(object);
    need(t.is_cuda() && t.scalar_type() == type && t.dim() == dims && t.layout() == at::kStrided);
    if (device < 0) {
      device = t.get_device();
      need(c10::impl::getDeviceGuardImpl(at::kCUDA)->getDevice().index() == device && lib.loaded());
    }
    need(t.get_device() == device);
    return t;
  }
  const Tensor& whole(PyObject* object, at::ScalarType type, int dims) {
    const Tensor& t = tensor(object, type, dims);
    need(t.is_contiguous());
    return t;
  }
  const Tensor& list(PyObject* object, at::ScalarType type, int64_t count) {
    const Tensor& t = whole(object, type, 1);
    need(t.size(0) == count);
    return t;
  }
  // rows of contiguous elements at any strides
  const Tensor& rows(PyObject* object, at::ScalarType type, int dims) {
    const Tensor& t = tensor(object, type, dims);
    need(t.stride(dims - 1) == 1);
    return t;
  }
  template <typename T>
  T* one(PyObject* object) {
    return object == Py_None ? nullptr : static_cast<T*>(list(object, kInt, 1).data_ptr());
  }
  Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    return at::empty(shape, at::TensorOptions().dtype(type).device(at::kCUDA, device));
  }
  // A part of an allocation as a tensor of its own, no view: a tenth of a view's time.
  static Tensor part(const Tensor& all, int64_t from, at::IntArrayRef shape) {
    Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_storage_offset(from);
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    return t;
  }
  // int32 lists of these lengths in one allocation
  std::vector<Tensor> lists(std::initializer_list<int64_t> counts) const {
    int64_t at = 0;
    for (int64_t n : counts) at += n;
    const Tensor all = empty({at}, kInt);
    std::vector<Tensor> parts;
    parts.reserve(counts.size());
    at = 0;
    for (int64_t n : counts) parts.push_back(part(all, at, {n})), at += n;
    return parts;
  }
  void* stream() const {
    PyObject* number = PyLong_FromLong(device);
    need(number);
    PyObject* address = PyObject_CallOneArg(lib.raw_stream, number);
    Py_DECREF(number);
    need(address);
    void* at = PyLong_AsVoidPtr(address);
    Py_DECREF(address);
    need(!PyErr_Occurred());
    return at;
  }
};

template <typename T>
T* data(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }

int number(PyObject* object) {
  int overflow = 0;
  need(PyLong_Check(object));
  const long long v = PyLong_AsLongLongAndOverflow(object, &overflow);
  need(!overflow && v >= INT32_MIN && v <= INT32_MAX);
  return (int)v;
}
int small(int64_t n) {
  need(n <= INT32_MAX);
  return (int)n;
}

struct Cache {
  aoto_mx4_cache c;
  int64_t kv_heads, page, dim;
};
Cache cache_of(Call& call, PyObject* object) {
  need(PyObject_TypeCheck(object, reinterpret_cast<PyTypeObject*>(lib.mx4)) && PyTuple_GET_SIZE(object) == 4);
  const Tensor& k = call.rows(PyTuple_GET_ITEM(object, 0), kByte, 4);
  const Tensor& v = call.rows(PyTuple_GET_ITEM(object, 1), kByte, 4);
  const Tensor& ks = call.rows(PyTuple_GET_ITEM(object, 2), kByte, 4);
  const Tensor& vs = call.rows(PyTuple_GET_ITEM(object, 3), kByte, 4);
  need(k.sizes() == v.sizes() && k.strides() == v.strides() && ks.sizes() == vs.sizes() &&
       ks.strides() == vs.strides() && k.size(3) % 32 == 0 && ks.size(0) == k.size(0) && ks.size(1) == k.size(1) &&
       ks.size(2) == k.size(2) && ks.size(3) == k.size(3) / 16);
  Cache to;
  to.kv_heads = k.size(1), to.page = k.size(2), to.dim = 2 * k.size(3);
  to.c = {k.data_ptr(), v.data_ptr(), ks.data_ptr(), vs.data_ptr(), k.stride(0), k.stride(1), k.stride(2),
          ks.stride(0), ks.stride(1), ks.stride(2), small(k.size(0))};
  return to;
}

PyObject* wrapped(const Tensor& t) { return THPVariable_Wrap(t); }
PyObject* wrapped(std::initializer_list<Tensor> tensors) {
  PyObject* all = PyTuple_New((Py_ssize_t)tensors.size());
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* one = all ? wrapped(t) : nullptr;
    if (!one) {
      Py_XDECREF(all);
      return nullptr;
    }
    PyTuple_SET_ITEM(all, i++, one);
  }
  return all;
}

void ok(int status) {
  if (status == AOTO_OK) return;
  need(status != AOTO_ERR_ARGUMENT && status != AOTO_ERR_UNSUPPORTED);
  if (PyObject* number = PyLong_FromLong(status)) {
    Py_XDECREF(PyObject_CallOneArg(lib.check, number));
    Py_DECREF(number);
  }
  need(PyErr_Occurred());
  throw Raised();
}

// The C ABI's call without the interpreter's lock: a launch may wait for room in its queue.
template <typename F>
int unlocked(F call) {
  struct Unlocked {
    PyThreadState* state = PyEval_SaveThread();
    ~Unlocked() { PyEval_RestoreThread(state); }
  } here;
  return call();
}

PyObject* append(PyObject* const* a) {
  Call call;
  const Tensor& qkv = call.rows(a[0], kBFloat16, 2);
  const int64_t tokens = qkv.size(0);
  const Cache cache = cache_of(call, a[5]);
  const int64_t heads = number(a[6]);
  need(heads > 0 && qkv.size(1) == (heads + 2 * cache.kv_heads) * cache.dim);
  const Tensor& positions = call.list(a[1], kLong, tokens);
  const Tensor& slots = call.list(a[2], kLong, tokens);
  const Tensor& cos = call.whole(a[3], kBFloat16, 2);
  const Tensor& sin = call.whole(a[4], kBFloat16, 2);
  need(cos.size(1) == cache.dim && sin.sizes() == cos.sizes());
  Tensor q;
  if (a[7] != Py_None) {
    q = call.whole(a[7], kBFloat16, 3);
    need(q.size(0) == tokens && q.size(1) == heads && q.size(2) == cache.dim);
  }
  int32_t* error = call.one<int32_t>(a[8]);
  if (!q.defined()) q = call.empty({tokens, heads, cache.dim}, kBFloat16);
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.append(qkv.data_ptr(), qkv.stride(0), data<int64_t>(positions), data<int64_t>(slots), cos.data_ptr(),
                      sin.data_ptr(), small(cos.size(0)), &cache.c, small(cache.page), small(tokens), (int)heads,
                      small(cache.kv_heads), small(cache.dim), q.data_ptr(), error, stream);
  }));
  return wrapped(q);
}

PyObject* unpack(PyObject* const* a) {
  Call call;
  const Cache cache = cache_of(call, a[0]);
  const std::array<int64_t, 4> shape = {cache.c.pages, cache.kv_heads, cache.page, cache.dim};
  const int64_t size = shape[0] * shape[1] * shape[2] * shape[3];
  const Tensor all = call.empty({2 * size}, kBFloat16);
  const Tensor keys = call.part(all, 0, shape), values = call.part(all, size, shape);
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.unpack(&cache.c, small(cache.page), small(cache.kv_heads), small(cache.dim), keys.data_ptr(),
                      values.data_ptr(), stream);
  }));
  return wrapped({keys, values});
}

PyObject* attention(PyObject* const* a) {
  Call call;
  const Tensor& q = call.rows(a[0], kBFloat16, 3);
  const int64_t tokens = q.size(0), heads = q.size(1), dim = q.size(2);
  const Cache cache = cache_of(call, a[1]);
  need(cache.dim == dim);
  const Tensor& tables = call.rows(a[2], kInt, 2);
  const int64_t requests = tables.size(0), blocks = tables.size(1);
  const Tensor& start = call.list(a[3], kInt, requests + 1);
  const Tensor& kv = call.list(a[4], kInt, requests);
  const int causal = PyObject_IsTrue(a[5]);
  need(causal >= 0);
  double scale;
  if (a[6] == Py_None) {
    scale = 1.0 / std::sqrt((double)dim);
  } else {
    need(PyFloat_CheckExact(a[6]));
    scale = PyFloat_AS_DOUBLE(a[6]);
  }
  const int rows = number(a[7]), keys = number(a[8]);
  Tensor out;
  if (a[10] != Py_None) {
    out = call.whole(a[10], kBFloat16, 2);
    need(out.size(0) == tokens && out.size(1) == heads * dim);
  }
  const size_t size =
      lib.attention_workspace(small(tokens), small(requests), small(blocks), small(cache.page), small(heads),
                              small(cache.kv_heads), small(dim), rows, keys);
  Tensor workspace;
  if (a[9] != Py_None) {
    need(THPVariable_CheckExact(a[9]));
    workspace = THPVariable_Unpack(a[9]);
    need(workspace.is_cuda() && workspace.get_device() == call.device);
    if (!workspace.is_contiguous() || workspace.nbytes() < size) workspace = Tensor();
  }
  if (size && !workspace.defined()) workspace = call.empty({(int64_t)size}, kByte);
  if (!out.defined()) out = call.empty({tokens, heads * dim}, kBFloat16);
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.attention(q.data_ptr(), q.stride(0), q.stride(1), &cache.c, small(cache.page), data<int32_t>(tables),
                         tables.stride(0), small(blocks), data<int32_t>(start), data<int32_t>(kv), small(tokens),
                         small(requests), small(heads), small(cache.kv_heads), small(dim), causal, (float)scale, rows,
                         keys, size ? workspace.data_ptr() : nullptr, out.data_ptr(), stream);
  }));
  return wrapped(out);
}

// block_tables, page_counts, shares, free_pages, free_start and the error, as the functions on pages take them.
struct Pool {
  const Tensor &shares, &tables, &counts, &free, &start;
  int32_t* error;
  int64_t requests;
  Pool(Call& call, PyObject* const* a, PyObject* e)
      : shares(call.whole(a[2], kInt, 1)), tables(call.rows(a[0], kInt, 2)),
        counts(call.list(a[1], kInt, tables.size(0))), free(call.whole(a[3], kInt, 1)), start(call.list(a[4], kInt, 1)),
        error(call.one<int32_t>(e)), requests(tables.size(0)) {
    need(shares.size(0) > 0);
  }
};

PyObject* fork(PyObject* const* a) {
  Call call;
  const Pool p(call, a + 2, a[8]);
  const Tensor& parents = call.list(a[0], kInt, p.requests);
  const Tensor& lens = call.list(a[1], kInt, p.requests);
  const int page = number(a[7]);
  const int64_t n = p.requests;
  const std::vector<Tensor> out = call.lists({n, n, 1, n, n, 2 * n});
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.fork(data<int32_t>(parents), data<int32_t>(lens), data<int32_t>(p.tables), p.tables.stride(0),
                    data<int32_t>(p.counts), data<int32_t>(p.shares), data<int32_t>(p.free), data<int32_t>(p.start),
                    small(n), small(p.tables.size(1)), small(p.free.size(0)), small(p.shares.size(0)), page,
                    data<int32_t>(out[0]), data<int32_t>(out[1]), data<int32_t>(out[2]), data<int32_t>(out[3]),
                    data<int32_t>(out[4]), data<int32_t>(out[5]), p.error, stream);
  }));
  return wrapped({out[0], out[1], out[2], out[3], out[4]});
}

PyObject* release(PyObject* const* a) {
  Call call;
  const Pool p(call, a + 1, a[7]);
  const Tensor& keep = call.list(a[0], kInt, p.requests);
  const int page = number(a[6]);
  const std::vector<Tensor> out = call.lists({p.requests, 1, p.shares.size(0) / 1024 + 2});
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.release(data<int32_t>(keep), data<int32_t>(p.tables), p.tables.stride(0), data<int32_t>(p.counts),
                       data<int32_t>(p.shares), data<int32_t>(p.free), data<int32_t>(p.start), small(p.requests),
                       small(p.tables.size(1)), small(p.free.size(0)), small(p.shares.size(0)), page,
                       data<int32_t>(out[0]), data<int32_t>(out[1]), data<int32_t>(out[2]), p.error, stream);
  }));
  return wrapped({out[0], out[1]});
}

PyObject* compact(PyObject* const* a) {
  Call call;
  const Pool p(call, a, a[5]);
  const int64_t n = p.shares.size(0);
  const std::vector<Tensor> out = call.lists({n, n, 1, n});
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.compact(data<int32_t>(p.tables), p.tables.stride(0), data<int32_t>(p.counts), data<int32_t>(p.shares),
                       data<int32_t>(p.free), data<int32_t>(p.start), small(p.requests), small(p.tables.size(1)),
                       small(p.free.size(0)), small(n), data<int32_t>(out[0]), data<int32_t>(out[1]),
                       data<int32_t>(out[2]), data<int32_t>(out[3]), p.error, stream);
  }));
  return wrapped({out[0], out[1], out[2]});
}

// A tensor's pages, as ops.py's _page_tensor reads them.
aoto_page_tensor pages_of(const Tensor& t, int64_t dim, int64_t pages) {
  need(t.is_cuda() && t.layout() == at::kStrided && dim >= 0 && dim < t.dim() && t.dim() <= 16 && t.numel() > 0 &&
       t.size(dim) == pages);
  std::array<std::pair<int64_t, int64_t>, 16> inner;
  int count = 0;
  for (int64_t i = dim + 1; i < t.dim(); ++i)
    if (t.size(i) > 1) inner[count++] = {t.stride(i), t.size(i)};
  std::sort(inner.begin(), inner.begin() + count);
  int64_t dense = 1;
  for (int i = 0; i < count; ++i) {
    need(inner[i].first == dense);
    dense *= inner[i].second;
  }
  int64_t planes = 1, plane_stride = 0;
  for (int64_t i = dim - 1; i >= 0; --i) {
    if (t.size(i) == 1) continue;
    if (planes > 1) need(t.stride(i) == planes * plane_stride);
    else plane_stride = t.stride(i);
    planes *= t.size(i);
  }
  const int64_t page_stride = pages > 1 ? t.stride(dim) : dense;
  std::pair<int64_t, int64_t> low = {page_stride, pages};
  std::pair<int64_t, int64_t> high = {planes > 1 ? plane_stride : page_stride * pages, planes};
  if (high < low) std::swap(low, high);
  need(low.first >= dense && high.first >= low.first * (low.second - 1) + dense);
  const int64_t size = t.element_size();
  return {t.data_ptr(), planes, plane_stride * size, page_stride * size, dense * size};
}

PyObject* copy(PyObject* const* a) {
  Call call;
  const Tensor& source = call.whole(a[1], kInt, 1);
  const Tensor& target = call.list(a[2], kInt, source.size(0));
  const int32_t* count = call.one<int32_t>(a[3]);
  const int dim = number(a[4]);
  int32_t* error = call.one<int32_t>(a[5]);
  const bool single = THPVariable_CheckExact(a[0]);
  need(single || PyList_CheckExact(a[0]) || PyTuple_Check(a[0]));
  const Py_ssize_t n = single ? 1 : PySequence_Fast_GET_SIZE(a[0]);
  need(n > 0 && source.size(0) > 0);
  std::vector<aoto_page_tensor> tensors;
  tensors.reserve((size_t)n);
  int64_t pages = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* object = single ? a[0] : PySequence_Fast_GET_ITEM(a[0], i);
    need(THPVariable_CheckExact(object));
    const Tensor& t = THPVariable_Unpack(object);
    need(t.is_cuda() && t.get_device() == call.device && dim >= 0 && dim < t.dim());
    if (pages < 0) pages = t.size(dim);
    tensors.push_back(pages_of(t, dim, pages));
  }
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.copy(tensors.data(), small(n), small(pages), data<int32_t>(source), data<int32_t>(target),
                    small(source.size(0)), count, error, stream);
  }));
  Py_RETURN_TRUE;
}

PyObject* adjust(PyObject* const* a) {
  Call call;
  need(THPVariable_CheckExact(a[0]));
  const at::ScalarType type = THPVariable_Unpack(a[0]).scalar_type();
  need(type == kBFloat16 || type == kFloat);
  const Tensor& logits = call.rows(a[0], type, 2);
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  int64_t requests = rows;
  aoto_adjustments j{};
  if (a[1] != Py_None) {
    const Tensor& start = call.whole(a[1], kInt, 1);
    requests = start.size(0) - 1;
    need(requests >= 1);
    j.query_start = data<int32_t>(start);
  }
  auto lists = [&](PyObject* object, at::ScalarType of, int64_t count, int64_t columns,
                   int64_t& stride) -> const Tensor& {
    const Tensor& t = call.rows(object, of, 2);
    need(t.size(0) == count && (columns < 0 || t.size(1) == columns));
    stride = t.stride(0);
    return t;
  };
  auto each = [&](PyObject* object, at::ScalarType of) -> void* {
    return object == Py_None ? nullptr : call.list(object, of, requests).data_ptr();
  };
  // from 2 on: history, history_lens, prompt_lens, draft_tokens, repetition, presence, frequency, bias_tokens,
  // bias_values, allowed, out
  if (a[2] != Py_None) {
    const Tensor& t = lists(a[2], kLong, requests, -1, j.history_stride);
    j.history = data<int64_t>(t), j.history_len = small(t.size(1));
  } else {
    need(a[3] == Py_None && a[4] == Py_None);
  }
  j.history_lens = static_cast<int32_t*>(each(a[3], kInt)), j.prompt_lens = static_cast<int32_t*>(each(a[4], kInt));
  if (a[5] != Py_None) {
    const Tensor& t = lists(a[5], kLong, requests, -1, j.draft_stride);
    j.draft_tokens = data<int64_t>(t), j.drafts = small(t.size(1));
  }
  j.repetition = static_cast<float*>(each(a[6], kFloat)), j.presence = static_cast<float*>(each(a[7], kFloat));
  j.frequency = static_cast<float*>(each(a[8], kFloat));
  need((a[9] == Py_None) == (a[10] == Py_None));
  if (a[9] != Py_None) {
    const Tensor& t = lists(a[9], kLong, requests, -1, j.bias_stride);
    j.bias_tokens = data<int64_t>(t), j.biases = small(t.size(1));
    j.bias_values = data<float>(lists(a[10], kFloat, requests, j.biases, j.value_stride));
  }
  if (a[11] != Py_None) j.allowed = data<int32_t>(lists(a[11], kInt, rows, (vocab + 31) / 32, j.allowed_stride));
  Tensor out;
  if (a[12] != Py_None) {
    out = call.rows(a[12], type, 2);
    need(out.sizes() == logits.sizes());
    need(out.storage().data() != logits.storage().data() ||
         (out.data_ptr() == logits.data_ptr() && out.strides() == logits.strides()));
  } else {
    out = call.empty({rows, vocab}, type);
  }
  void* const stream = call.stream();
  ok(unlocked([&] {
    return lib.adjust(logits.data_ptr(), type == kFloat, logits.stride(0), small(rows), small(vocab), small(requests),
                      &j, out.data_ptr(), out.stride(0), stream);
  }));
  return wrapped(out);
}

// None, with no Python error left behind, where the call was not made.
template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  try {
    if (count == N) return F(args);
  } catch (const Raised&) {
    return nullptr;
  } catch (...) {
  }
  PyErr_Clear();
  Py_RETURN_NONE;
}

// bind(addresses of the entry points in the order of Library, raw_stream, PagedMx4, check)
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != 13) {
    PyErr_SetString(PyExc_TypeError, "bind takes ten addresses, a function, a type and a function");
    return nullptr;
  }
  void* at[10];
  for (int i = 0; i < 10; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  auto set = [&](auto& to, int i) { to = reinterpret_cast<std::decay_t<decltype(to)>>(at[i]); };
  set(lib.loaded, 0), set(lib.append, 1), set(lib.unpack, 2), set(lib.attention, 3), set(lib.attention_workspace, 4);
  set(lib.fork, 5), set(lib.release, 6), set(lib.compact, 7), set(lib.copy, 8), set(lib.adjust, 9);
  for (int i = 10; i < 13; ++i) Py_INCREF(args[i]);
  Py_XDECREF(lib.raw_stream), Py_XDECREF(lib.mx4), Py_XDECREF(lib.check);
  lib.raw_stream = args[10], lib.mx4 = args[11], lib.check = args[12];
  Py_RETURN_NONE;
}

#define AOTO_CALL(NAME, F, N) \
  {NAME, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&bind)), METH_FASTCALL, nullptr},
    AOTO_CALL("paged_rope_append_mx4", append, 9),
    AOTO_CALL("paged_unpack_mx4", unpack, 1),
    AOTO_CALL("paged_attention_mx4", attention, 11),
    AOTO_CALL("paged_fork", fork, 9),
    AOTO_CALL("paged_release", release, 8),
    AOTO_CALL("paged_compact", compact, 6),
    AOTO_CALL("paged_copy", copy, 6),
    AOTO_CALL("adjust_logits", adjust, 13),
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// built_for: the torch and Python of the headers; with others nothing here but this may be called.
PyMODINIT_FUNC PyInit__calls() {
  PyObject* calls = PyModule_Create(&module);
  if (calls && PyModule_AddStringConstant(calls, "built_for", AOTO_BUILT_FOR) < 0) Py_CLEAR(calls);
  return calls;
}
