/*
 * Binding of the kv4 entry points that takes torch tensors as they are: the
 * checks, the outputs and the call in one step from Python.  With the checks in
 * Python and the outputs made there, a call cost 7 us (kv4_append) to 15 us
 * (kv4_schedule, six outputs) of host time for 5 us of GPU time.
 *
 * A function answers None for arguments that it does not know to be right; the
 * caller (csed499ii_b200/kv4.py) then takes its own way, whose checks say what
 * is wrong.  Otherwise kv4_append answers the status of the C ABI, and the
 * others a status and their outputs.
 */
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>

#include "../../include/sm100_marlin.h"

namespace {

// The tensor behind a Python object, or null.
const at::Tensor* tensor_of(PyObject* o) {
  return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr;
}

bool ints_on(const at::Tensor* t, int dev) {
  return t && t->scalar_type() == at::kInt && t->is_cuda() && t->get_device() == dev && t->is_contiguous();
}

struct Cache {
  const at::Tensor* t;
  int pages, heads, page_size, dim, dtype, dev;

  bool from(PyObject* o) {
    t = tensor_of(o);
    if (!t || !t->is_cuda() || t->dim() != 4 || !t->is_contiguous()) return false;
    if (t->scalar_type() != at::kHalf && t->scalar_type() != at::kBFloat16) return false;
    const auto s = t->sizes();
    if (s[3] != 8 * 64 + 64 && s[3] != 8 * 128 + 64) return false;
    if (s[0] > INT_MAX || s[1] > INT_MAX || s[2] > INT_MAX / 16) return false;
    pages = static_cast<int>(s[0]);
    heads = static_cast<int>(s[1]);
    page_size = static_cast<int>(s[2]) * 16;
    dim = s[3] == 8 * 64 + 64 ? 64 : 128;
    dtype = t->scalar_type() == at::kHalf ? SM100_MARLIN_FP16 : SM100_MARLIN_BF16;
    dev = t->get_device();
    return true;
  }
  // (tokens, heads, dim) of the cache's type with contiguous channels
  bool takes(const at::Tensor* x) const {
    return x && x->is_cuda() && x->get_device() == dev && x->scalar_type() == t->scalar_type() &&
           x->dim() == 3 && x->size(2) == dim && x->stride(2) == 1 && x->size(0) <= INT_MAX;
  }
};

// Entries from `from` on of a tensor in one dimension, as a tensor of these sizes.
at::Tensor part_of(const at::Tensor& t, int64_t from, at::IntArrayRef sizes) {
  at::Tensor x = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  x.unsafeGetTensorImpl()->set_storage_offset(from);
  x.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return x;
}

void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream(dev).stream(); }

PyObject* none() { Py_RETURN_NONE; }

/* kv4_append(k, v, cache, slots) */
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Cache c;
  if (n != 4 || !c.from(args[2])) return none();
  const at::Tensor *k = tensor_of(args[0]), *v = tensor_of(args[1]), *slots = tensor_of(args[3]);
  if (!c.takes(k) || !c.takes(v) || k->size(1) != c.heads || v->size(1) != c.heads ||
      v->size(0) != k->size(0) || !ints_on(slots, c.dev) || slots->numel() != k->size(0))
    return none();
  const int rc = sm100_marlin_kv4_append(
      k->const_data_ptr(), k->stride(0), k->stride(1), v->const_data_ptr(), v->stride(0), v->stride(1),
      c.t->mutable_data_ptr(), c.pages, c.heads, c.page_size, c.dim, c.dtype,
      static_cast<const int*>(slots->const_data_ptr()), static_cast<int>(k->size(0)), c.dev, stream_of(c.dev));
  return PyLong_FromLong(rc);
}

/* kv4_read(cache, slots) -> (status, k, v) */
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Cache c;
  if (n != 2 || !c.from(args[0])) return none();
  const at::Tensor* slots = tensor_of(args[1]);
  if (!ints_on(slots, c.dev) || slots->numel() > INT_MAX) return none();
  const int64_t sizes[] = {slots->numel(), c.heads, c.dim}, of_k = sizes[0] * sizes[1] * sizes[2];
  const at::Tensor both = at::empty({2 * of_k}, c.t->options()), k = part_of(both, 0, sizes), v = part_of(both, of_k, sizes);
  const int rc = sm100_marlin_kv4_read(c.t->const_data_ptr(), c.pages, c.heads, c.page_size, c.dim, c.dtype,
                                       static_cast<const int*>(slots->const_data_ptr()),
                                       static_cast<int>(slots->numel()), k.mutable_data_ptr(),
                                       v.mutable_data_ptr(), c.dev, stream_of(c.dev));
  return Py_BuildValue("iNN", rc, THPVariable_Wrap(k), THPVariable_Wrap(v));
}

/* kv4_attention(q, cache, block_tables, lens, starts, max_new, window, scale, workspace)
 * -> (status, out); starts None: one row for each request; max_new None: all rows;
 * scale None: 1 / sqrt(head_dim). */
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  Cache c;
  if (n != 9 || !c.from(args[1])) return none();
  const at::Tensor *q = tensor_of(args[0]), *tables = tensor_of(args[2]), *lens = tensor_of(args[3]);
  const at::Tensor *starts = args[4] == Py_None ? nullptr : tensor_of(args[4]), *space = tensor_of(args[8]);
  if (!c.takes(q) || !ints_on(tables, c.dev) || tables->dim() != 2 || !ints_on(lens, c.dev) ||
      !ints_on(space, c.dev) || tables->size(0) != lens->numel() || q->size(1) == 0 || c.heads == 0 ||
      q->size(1) % c.heads != 0 || tables->size(1) > INT_MAX || lens->numel() > INT_MAX - 1)
    return none();
  long long max_new = q->size(0);
  if (args[4] == Py_None) {
    if (q->size(0) != lens->numel()) return none();
    max_new = 1;
  } else {
    if (!ints_on(starts, c.dev) || starts->numel() != lens->numel() + 1) return none();
    if (args[5] != Py_None) max_new = PyLong_AsLongLong(args[5]);
  }
  const long long window = PyLong_AsLongLong(args[6]);
  const double scale = args[7] == Py_None ? 1.0 / std::sqrt(static_cast<double>(c.dim)) : PyFloat_AsDouble(args[7]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  if (window < 0 || window > INT_MAX || max_new < 0 || max_new > INT_MAX) return none();
  const at::Tensor out = at::empty(q->sizes(), q->options());
  const int rc = sm100_marlin_kv4_attention(
      q->const_data_ptr(), q->stride(0), q->stride(1), c.t->const_data_ptr(), c.pages, c.heads, c.page_size,
      c.dim, c.dtype, static_cast<const int*>(tables->const_data_ptr()), tables->stride(0),
      static_cast<int>(tables->size(1)), static_cast<const int*>(lens->const_data_ptr()),
      starts ? static_cast<const int*>(starts->const_data_ptr()) : nullptr, static_cast<int>(lens->numel()),
      static_cast<int>(q->size(0)), static_cast<int>(q->size(1)), static_cast<int>(max_new),
      static_cast<int>(window), static_cast<float>(scale), out.mutable_data_ptr(), space->mutable_data_ptr(),
      static_cast<size_t>(space->numel()) * 4, c.dev, stream_of(c.dev));
  return Py_BuildValue("iN", rc, THPVariable_Wrap(out));
}

/* kv4_schedule(new_lens, lens, block_tables, free_pages, free_count, rows, page_size, lens_out, free_count_out)
 * -> (status, lens_out, free_count_out, starts, slots, positions, fate) */
PyObject* schedule(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) return none();
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i) t[i] = tensor_of(args[i]);
  if (!t[0] || !t[0]->is_cuda()) return none();
  const int dev = t[0]->get_device();
  const int64_t batch = t[0]->numel();
  for (int i = 0; i < 5; ++i)
    if (!ints_on(t[i], dev)) return none();
  const long long rows = PyLong_AsLongLong(args[5]), page = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return none();
  }
  const at::Tensor *lens_out = args[7] == Py_None ? nullptr : tensor_of(args[7]);
  const at::Tensor *count_out = args[8] == Py_None ? nullptr : tensor_of(args[8]);
  if (t[1]->numel() != batch || batch > 8192 || t[2]->dim() != 2 || t[2]->size(0) != batch ||
      t[2]->size(1) > INT_MAX || t[3]->numel() > INT_MAX || t[4]->numel() != 1 || rows < 0 ||
      rows > INT_MAX || page <= 0 || page > INT_MAX ||
      (args[7] != Py_None && (!ints_on(lens_out, dev) || lens_out->numel() != batch)) ||
      (args[8] != Py_None && (!ints_on(count_out, dev) || count_out->numel() != 1)))
    return none();
  // What only this step needs shares one allocation; lengths and count, which
  // stay, have their own.
  const auto options = t[0]->options();
  const int64_t at_slots = (batch + 64) / 64 * 64, at_positions = at_slots + (rows + 63) / 64 * 64,
                at_fate = at_positions + (rows + 63) / 64 * 64;
  const at::Tensor step = at::empty({at_fate + batch}, options);
  const at::Tensor out[6] = {lens_out ? *lens_out : at::empty({batch}, options),
                             count_out ? *count_out : at::empty({1}, options),
                             part_of(step, 0, {batch + 1}),
                             part_of(step, at_slots, {rows}),
                             part_of(step, at_positions, {rows}),
                             part_of(step, at_fate, {batch})};
  int* to[6];
  for (int i = 0; i < 6; ++i) to[i] = static_cast<int*>(out[i].mutable_data_ptr());
  const int rc = sm100_marlin_kv4_schedule(
      static_cast<const int*>(t[0]->const_data_ptr()), static_cast<const int*>(t[1]->const_data_ptr()),
      static_cast<int*>(t[2]->mutable_data_ptr()), t[2]->stride(0), static_cast<int>(t[2]->size(1)),
      static_cast<int>(batch), static_cast<int*>(t[3]->mutable_data_ptr()), static_cast<int>(t[3]->numel()),
      static_cast<const int*>(t[4]->const_data_ptr()), static_cast<int>(rows), static_cast<int>(page), to[0],
      to[1], to[2], to[3], to[4], to[5], dev, stream_of(dev));
  PyObject* answer = PyTuple_New(7);
  if (!answer) return nullptr;
  PyTuple_SET_ITEM(answer, 0, PyLong_FromLong(rc));
  for (int i = 0; i < 6; ++i) PyTuple_SET_ITEM(answer, i + 1, THPVariable_Wrap(out[i]));
  return answer;
}

// C++ exceptions (an allocation that failed) become Python's.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* type = nullptr;
    if (PyObject* torch = PyImport_ImportModule("torch")) {
      type = PyObject_GetAttrString(torch, "OutOfMemoryError");
      Py_DECREF(torch);
    }
    PyErr_SetString(type ? type : PyExc_RuntimeError, e.what_without_backtrace());
    Py_XDECREF(type);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define ENTRY(name, f) {name, (PyCFunction)(void (*)(void))guarded<f>, METH_FASTCALL, nullptr}

PyMethodDef methods[] = {ENTRY("kv4_append", append), ENTRY("kv4_read", read), ENTRY("kv4_attention", attention),
                         ENTRY("kv4_schedule", schedule), {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torchfast", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torchfast(void) { return PyModule_Create(&module); }
