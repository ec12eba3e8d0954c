// The two calls of a decode step as Python makes them, in C++: ri_append_kv, and ri_decode_step or ri_host_step by a prepared
// call; and the operators that assembled execution buffers are attended with.  Made by Python a short context's step takes the
// host longer than the GPU (15.3 us against 13.8 captured, 8 groups of 8192 tokens; here 8.7), and beside the launches that is an
// attribute, a method call and a comparison for each of the buffers whose address a prepared call holds, an output tensor, a call
// through ctypes.  Everything is looked at in every call; what is not the usual case (tensors that are not plain ones on one
// device, rows of another shape or type, a buffer that has moved or is too short) is answered with None, and the caller goes its
// general way.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <vector>

#include "../../include/retro_mi355.h"

namespace {

// the tensor behind a Python object, null unless it is a plain one with memory of its own
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.has_storage() ? &t : nullptr;
}

// hipStream_t of the current device's current stream
ri_stream_t current_stream() {
  return (ri_stream_t)c10::hip::getCurrentHIPStream(c10::hip::current_device()).stream();
}

bool shape_is(const at::Tensor& t, PyObject* shape) {
  if (!PyTuple_Check(shape) || PyTuple_GET_SIZE(shape) != t.dim()) return false;
  for (int64_t i = 0; i < t.dim(); ++i) {
    const long long n = PyLong_AsLongLong(PyTuple_GET_ITEM(shape, i));
    if (n == -1 && PyErr_Occurred()) throw python_error();
    if (n != t.size(i)) return false;
  }
  return true;
}

// append(key_row, value_row, steady_k, steady_v, pos, pos_dev or None, row_shape): status, or None where it has to be the general way
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "append: seven arguments");
    return nullptr;
  }
  const at::Tensor* t[4];
  for (int i = 0; i < 4; ++i)
    if (!(t[i] = plain(args[i]))) Py_RETURN_NONE;
  const at::Tensor &k = *t[2], &v = *t[3];
  const int device = k.get_device();
  const long long pos = PyLong_AsLongLong(args[4]);
  if (pos == -1 && PyErr_Occurred()) return nullptr;
  if (device < 0 || !k.is_cuda() || v.get_device() != device || k.dim() != 4 || v.sizes() != k.sizes() || k.size(3) != 128 ||
      !k.is_contiguous() || !v.is_contiguous() || pos >= k.size(2))
    Py_RETURN_NONE;
  for (int i = 0; i < 2; ++i) {
    const at::Tensor &row = *t[i], &zone = *t[i + 2];
    if (row.get_device() != device || row.scalar_type() != zone.scalar_type() || !row.is_contiguous() ||
        !shape_is(row, args[6]) || row.numel() != k.size(0) * k.size(1) * 128 || (uintptr_t)row.data_ptr() % 16 != 0)
      Py_RETURN_NONE;
  }
  const int64_t* pos_dev = nullptr;
  if (args[5] != Py_None) {
    const at::Tensor* p = plain(args[5]);
    if (!p || p->get_device() != device || p->scalar_type() != at::kLong) Py_RETURN_NONE;
    pos_dev = (const int64_t*)p->data_ptr();
  }
  const void *kr = t[0]->data_ptr(), *vr = t[1]->data_ptr();
  void *kz = k.data_ptr(), *vz = v.data_ptr();
  const int64_t stride = k.size(2);
  const int groups = (int)(k.size(0) * k.size(1));
  const ri_stream_t stream = current_stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = ri_append_kv(kr, vr, kz, vz, stride, pos, pos_dev, groups, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
  END_HANDLE_TH_ERRORS
}

// A prepared call: the struct's address, the addresses it was made of and the numbers beside them.  The owner keeps the struct
// and the tensors alive.
struct Step {
  PyObject_HEAD
  const ri_decode_step_t* step;
  const ri_lru_t* lru;
  std::vector<const void*>* held;
  std::vector<long long>* numbers;
  at::ScalarType dtype;
  int device;
  int64_t queries;
};

bool addresses(PyObject* tensors, std::vector<const void*>& out) {
  const Py_ssize_t n = PyTuple_GET_SIZE(tensors);
  out.resize(n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    PyObject* o = PyTuple_GET_ITEM(tensors, i);
    const at::Tensor* t = o == Py_None ? nullptr : plain(o);
    if (o != Py_None && !t) return false;
    out[i] = t ? t->data_ptr() : nullptr;
  }
  return true;
}

// Step(step address, lru address or 0, centroids, tensors, numbers); tensors and numbers as `run` is given them
PyObject* step_new(PyTypeObject* type, PyObject* args, PyObject*) {
  HANDLE_TH_ERRORS
  unsigned long long step, lru;
  PyObject *centroids, *tensors, *numbers;
  if (!PyArg_ParseTuple(args, "KKOO!O!", &step, &lru, &centroids, &PyTuple_Type, &tensors, &PyTuple_Type, &numbers)) return nullptr;
  const at::Tensor* c = plain(centroids);
  if (!c) {
    PyErr_SetString(PyExc_TypeError, "Step: centroids are not a plain tensor");
    return nullptr;
  }
  std::vector<const void*> held;
  if (!addresses(tensors, held)) {
    PyErr_SetString(PyExc_TypeError, "Step: a buffer is not a plain tensor");
    return nullptr;
  }
  std::vector<long long> values;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(numbers); ++i) {
    values.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(numbers, i)));
    if (PyErr_Occurred()) return nullptr;
  }
  Step* self = (Step*)type->tp_alloc(type, 0);
  if (!self) return nullptr;
  self->step = (const ri_decode_step_t*)(uintptr_t)step;
  self->lru = (const ri_lru_t*)(uintptr_t)lru;
  self->held = new std::vector<const void*>(std::move(held));
  self->numbers = new std::vector<long long>(std::move(values));
  self->dtype = c->scalar_type();
  self->device = c->get_device();
  self->queries = (int64_t)self->step->BG * self->step->gs * 128;
  return (PyObject*)self;
  END_HANDLE_TH_ERRORS
}

void step_dealloc(PyObject* o) {
  Step* self = (Step*)o;
  delete self->held;
  delete self->numbers;
  PyTypeObject* type = Py_TYPE(o);
  type->tp_free(o);
  Py_DECREF(type);
}

// run(queries, static_len, out_shape, tensors, numbers): the output, None where the call is not this one's, or the status
PyObject* step_run(PyObject* o, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const Step* self = (const Step*)o;
  if (n != 5 || !PyTuple_Check(args[2]) || !PyTuple_Check(args[3]) || !PyTuple_Check(args[4])) {
    PyErr_SetString(PyExc_TypeError, "run: queries, static_len, out_shape, tensors, numbers");
    return nullptr;
  }
  const at::Tensor* q = plain(args[0]);
  if (!q || at::impl::torch_function_mode_enabled() || q->get_device() != self->device || q->scalar_type() != self->dtype ||
      !q->is_contiguous() || q->numel() != self->queries)
    Py_RETURN_NONE;
  if ((size_t)PyTuple_GET_SIZE(args[3]) != self->held->size() || (size_t)PyTuple_GET_SIZE(args[4]) != self->numbers->size())
    Py_RETURN_NONE;
  for (size_t i = 0; i < self->held->size(); ++i) {
    PyObject* x = PyTuple_GET_ITEM(args[3], i);
    const at::Tensor* t = x == Py_None ? nullptr : plain(x);
    if ((x != Py_None && !t) || (t ? t->data_ptr() : nullptr) != (*self->held)[i]) Py_RETURN_NONE;
  }
  for (size_t i = 0; i < self->numbers->size(); ++i) {
    const long long x = PyLong_AsLongLong(PyTuple_GET_ITEM(args[4], i));
    if (x == -1 && PyErr_Occurred()) return nullptr;
    if (x != (*self->numbers)[i]) Py_RETURN_NONE;
  }
  const long static_len = PyLong_AsLong(args[1]);
  if (static_len == -1 && PyErr_Occurred()) return nullptr;
  int64_t shape[4], elements = 1;
  if (PyTuple_GET_SIZE(args[2]) != 4) Py_RETURN_NONE;
  for (int i = 0; i < 4; ++i) {
    shape[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(args[2], i));
    elements *= shape[i];
  }
  if (PyErr_Occurred()) return nullptr;
  if (elements != self->queries) Py_RETURN_NONE;
  at::Tensor out = at::empty(at::IntArrayRef(shape, 4), q->options().requires_grad(false));
  const void* qp = q->data_ptr();
  void* op = out.data_ptr();
  const ri_stream_t stream = current_stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = self->lru ? ri_host_step(self->step, self->lru, qp, (int)static_len, op, stream)
                     : ri_decode_step(self->step, qp, (int)static_len, op, stream);
  Py_END_ALLOW_THREADS
  if (status) return PyLong_FromLong(status);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// plain contiguous device tensors of one type (null: not given); null where one is not
bool device_tensors(PyObject* const* args, int n, at::ScalarType dtype, const at::Tensor** out, bool optional = false) {
  for (int i = 0; i < n; ++i) {
    out[i] = nullptr;
    if (optional && args[i] == Py_None) continue;
    const at::Tensor* t = plain(args[i]);
    if (!t || !t->is_cuda() || t->scalar_type() != dtype || !t->is_contiguous()) return false;
    out[i] = t;
  }
  return true;
}
void* address(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

bool integers(PyObject* const* args, int n, int64_t* out) {
  for (int i = 0; i < n; ++i) {
    if (!PyLong_Check(args[i])) return false;
    int over;
    out[i] = PyLong_AsLongLongAndOverflow(args[i], &over);
    if (over || out[i] < 0 || out[i] > INT32_MAX) return false;
  }
  return true;
}
// at least a b c elements (each within 32 bits)
bool holds(const at::Tensor* t, int64_t a, int64_t b, int64_t c) { return (__int128)t->numel() >= (__int128)a * b * c; }
bool half_type(const at::Tensor* t, at::ScalarType& dtype) {
  dtype = t ? t->scalar_type() : at::kFloat;
  return dtype == at::kHalf || dtype == at::kBFloat16;
}

// gemm_softmax(A, B, D, Softmax, Norm, Sum, batch_count, m, n, k, alpha, beta): status, or None where the wrapper has to look
PyObject* gemm_softmax(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* t[6];
  at::ScalarType dtype;
  int64_t x[4];
  if (n != 12 || !half_type(plain(args[0]), dtype) || !device_tensors(args, 4, dtype, t) ||
      !device_tensors(args + 4, 2, at::kFloat, t + 4) || !integers(args + 6, 4, x))
    Py_RETURN_NONE;
  const int64_t bc = x[0], m = x[1], cols = x[2], k = x[3], tiles = (cols + 255) / 256;
  if (!holds(t[0], bc, m, k) || !holds(t[1], bc, cols, k) || !holds(t[2], bc, m, cols) || !holds(t[3], bc, m, cols) ||
      !holds(t[4], bc, tiles, m) || !holds(t[5], bc, tiles, m))
    Py_RETURN_NONE;
  const double alpha = PyFloat_AsDouble(args[10]), beta = PyFloat_AsDouble(args[11]);
  if (PyErr_Occurred()) {   // (float() takes more)
    PyErr_Clear();
    Py_RETURN_NONE;
  }
  void* p[6];
  for (int i = 0; i < 6; ++i) p[i] = address(t[i]);
  const ri_stream_t stream = current_stream();
  auto* call = dtype == at::kHalf ? ri_batch_gemm_softmax_f16 : ri_batch_gemm_softmax;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = call(p[0], p[1], p[2], (float*)p[4], (float*)p[5], p[3], (int)bc, (int)m, (int)cols, (int)k, (float)alpha, (float)beta,
                stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
  END_HANDLE_TH_ERRORS
}

// gather_vectors(key_data, key_buffer, value_data, value_buffer, src_metadata, dst_metadata, data_offsets, groups, data_length,
// buffer_length, index_size, copy_start, copy_num): as above
PyObject* gather_vectors(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor* t[7];
  at::ScalarType dtype;
  int64_t x[6];
  if (n != 13 || !half_type(plain(args[0]), dtype) || !device_tensors(args, 6, dtype, t) ||
      !device_tensors(args + 6, 1, at::kLong, t + 6) || !integers(args + 7, 6, x))
    Py_RETURN_NONE;
  const int64_t groups = x[0], data = x[1], buffer = x[2];
  if (!holds(t[0], groups, data, 128) || !holds(t[1], groups, buffer, 128) || !holds(t[2], groups, data, 128) ||
      !holds(t[3], groups, buffer, 128) || !holds(t[4], groups, data, 1) || !holds(t[5], groups, buffer, 1) ||
      !holds(t[6], groups, x[3], 1))
    Py_RETURN_NONE;
  void* p[7];
  for (int i = 0; i < 7; ++i) p[i] = address(t[i]);
  const ri_stream_t stream = current_stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = ri_gather_copy_vectors(p[0], p[1], p[2], p[3], p[4], p[5], (const int64_t*)p[6], (int)groups, (int)data, (int)buffer,
                                  (int)x[3], (int)x[4], (int)x[5], stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
  END_HANDLE_TH_ERRORS
}

PyObject* pair_of(at::Tensor&& out, at::Tensor&& lse) {
  PyObject *a = THPVariable_Wrap(std::move(out)), *b = THPVariable_Wrap(std::move(lse));
  PyObject* both = a && b ? PyTuple_Pack(2, a, b) : nullptr;
  Py_XDECREF(a);
  Py_XDECREF(b);
  return both;
}

// flash(q, k, v, weight, previous_out, previous_lse, cache_seqlens, workspace, scale, return_lse): the output, or (output, lse);
// a status that is not zero; None as above.  q [BG, 1, gs, 128], k [BG, S, 1, 128]; the others by their elements.
PyObject* flash(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *t[7], *ws;
  at::ScalarType dtype;
  if (n != 10 || at::impl::torch_function_mode_enabled() || !half_type(plain(args[0]), dtype) ||
      !device_tensors(args, 3, dtype, t) || !device_tensors(args + 3, 2, dtype, t + 3, true) ||
      !device_tensors(args + 5, 1, at::kFloat, t + 5, true) || !device_tensors(args + 6, 1, at::kInt, t + 6, true) ||
      !device_tensors(args + 7, 1, at::kByte, &ws) || (t[4] && !t[5]))
    Py_RETURN_NONE;
  const at::Tensor &q = *t[0], &k = *t[1];
  if (q.dim() != 4 || k.dim() != 4 || q.size(1) != 1 || q.size(3) != 128 || k.size(2) != 1) Py_RETURN_NONE;
  const int64_t BG = q.size(0), gs = q.size(2), S = k.size(1);
  if (!holds(t[1], BG, S, 128) || !holds(t[2], BG, S, 128) || (t[3] && !holds(t[3], BG, S, 1)) ||
      (t[4] && (!holds(t[4], BG, gs, 128) || !holds(t[5], BG, gs, 1))) || (t[6] && !holds(t[6], BG, 1, 1)))
    Py_RETURN_NONE;
  const double scale = PyFloat_AsDouble(args[8]);
  const int with_lse = PyObject_IsTrue(args[9]);
  if (PyErr_Occurred()) return nullptr;
  at::Tensor out = at::empty_like(q), lse;
  if (with_lse) lse = at::empty({BG, gs}, q.options().dtype(at::kFloat).requires_grad(false));
  void* p[7];
  for (int i = 0; i < 7; ++i) p[i] = address(t[i]);
  void *op = out.data_ptr(), *lp = with_lse ? lse.data_ptr() : nullptr, *wp = ws->data_ptr();
  const size_t bytes = (size_t)ws->numel();
  const ri_stream_t stream = current_stream();
  auto* call = dtype == at::kHalf ? ri_weighted_flash_decoding_f16 : ri_weighted_flash_decoding;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = call(p[0], p[1], p[2], p[3], (const int32_t*)p[6], p[4], (const float*)p[5], op, (float*)lp, (int)BG, (int)gs, (int)S,
                (int)S, (float)scale, wp, bytes, stream);
  Py_END_ALLOW_THREADS
  if (status) return PyLong_FromLong(status);
  if (!with_lse) return THPVariable_Wrap(std::move(out));
  return pair_of(std::move(out), std::move(lse));
  END_HANDLE_TH_ERRORS
}

// ---- the paged cache's calls: arguments as the wrappers in kernels.py take them, checked as they check them (there the errors
// are worded); anything that is not in order, and calls on another device than the current one, are left to them.

// a plain tensor on `device` (null and true for None where it may be), of `dims` dimensions and `dtype`
bool paged_tensor(PyObject* o, int dims, at::ScalarType dtype, int device, const at::Tensor** out, bool optional = false) {
  *out = nullptr;
  if (o == Py_None) return optional;
  const at::Tensor* t = plain(o);
  if (!t || !t->is_cuda() || t->get_device() != device || t->dim() != dims || t->scalar_type() != dtype) return false;
  *out = t;
  return true;
}
// strides of the dimensions in front of rows that are moved 16 bytes at a time (0 for one element)
bool paged_rows(const at::Tensor& t, bool writes, int64_t* strides) {
  const int64_t last = t.dim() - 1;
  if (t.stride(last) != 1 || (uintptr_t)t.data_ptr() % 16) return false;
  for (int64_t i = 0; i < last; ++i) {
    strides[i] = t.size(i) > 1 ? t.stride(i) : 0;
    if (strides[i] < 0 || strides[i] % 8 || (writes && t.size(i) > 1 && strides[i] == 0)) return false;
  }
  return true;
}
bool paged_pages(PyObject* const* args, int64_t B, bool writes, ri_paged_t* c, at::ScalarType* dtype, int* device) {
  const at::Tensor *k = plain(args[0]), *v, *table;
  if (!k || !k->is_cuda() || k->dim() != 4 || !half_type(k, *dtype)) return false;
  *device = k->get_device();
  if (*device != c10::hip::current_device() || !paged_tensor(args[1], 4, *dtype, *device, &v) ||
      !paged_tensor(args[2], 2, at::kInt, *device, &table) || v->sizes() != k->sizes() || table->size(0) != B)
    return false;
  int64_t ks[3], vs[3];
  const int64_t pages = k->size(0), heads = k->size(1), rows = k->size(2), dim = k->size(3), n = table->size(1);
  if (pages < 1 || pages > INT32_MAX || heads < 1 || heads > 65535 || rows < 1 || rows & (rows - 1) || (dim != 64 && dim != 128) ||
      !paged_rows(*k, writes, ks) || !paged_rows(*v, writes, vs) || n < 1 || n > (1 << 24) / rows || (n > 1 && table->stride(1) != 1) ||
      table->stride(0) < 0)
    return false;
  *c = {k->data_ptr(), v->data_ptr(), (const int32_t*)table->data_ptr(), ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], table->stride(0),
        (int)pages, (int)heads, (int)rows, (int)dim, (int)n, *dtype == at::kHalf};
  return true;
}
// one int32 to a sequence
bool paged_each(PyObject* o, int64_t B, int device, const at::Tensor** out, bool optional = true) {
  if (!paged_tensor(o, 1, at::kInt, device, out, optional)) return false;
  return !*out || ((*out)->size(0) == B && (B == 1 || (*out)->stride(0) == 1));
}
bool paged_meet(const at::Tensor* a, const at::Tensor* b, int64_t B) {
  if (!a || !b) return false;
  const auto x = (uintptr_t)a->data_ptr(), y = (uintptr_t)b->data_ptr();
  return x < y + 4 * B && y < x + 4 * B;
}
// a value to each row, [B, heads, rows or more]; strides by sequence and head
bool paged_values(PyObject* o, at::ScalarType dtype, int64_t B, int64_t heads, int64_t rows, int device, bool writes,
                  const at::Tensor** out, int64_t* strides) {
  strides[0] = strides[1] = 0;
  if (!paged_tensor(o, 3, dtype, device, out, true)) return false;
  const at::Tensor* t = *out;
  if (!t) return true;
  if (t->size(0) != B || t->size(1) != heads || t->size(2) < rows || (t->size(2) > 1 && t->stride(2) != 1)) return false;
  const int64_t sb = B > 1 ? t->stride(0) : 0, sh = heads > 1 ? t->stride(1) : t->size(2);
  if (sh < rows || (B > 1 && sb < rows) || (writes && B > 1 && heads > 1 && !(sb >= (heads - 1) * sh + rows || sh >= (B - 1) * sb + rows)))
    return false;
  strides[0] = sb;
  strides[1] = sh;
  return true;
}
// the scratch tensor, null where it is missing, elsewhere or too small
void* paged_scratch(PyObject* o, size_t bytes, int device) {
  const at::Tensor* t = plain(o);
  return t && t->is_cuda() && t->get_device() == device && t->scalar_type() == at::kByte && t->is_contiguous() &&
                 (size_t)t->numel() >= bytes ? t->data_ptr() : nullptr;
}
bool paged_scale(PyObject* o, int64_t dim, float* scale) {
  if (o == Py_None) *scale = (float)(1.0 / sqrt((double)dim));
  else if (PyFloat_CheckExact(o)) *scale = (float)PyFloat_AS_DOUBLE(o);
  else return false;
  return true;
}
// an int or, for None, `none`
bool paged_int(PyObject* o, int64_t none, int64_t* out) {
  if (o == Py_None) {
    *out = none;
    return true;
  }
  return PyLong_CheckExact(o) && integers(&o, 1, out);
}

// paged_attention(q, k_pages, v_pages, block_table, cache_seqlens, starts, scores, scale, return_lse, max_len, workspace)
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *q, *lens, *starts, *scores;
  ri_paged_t cache;
  at::ScalarType dtype;
  int device;
  int64_t strides[2], max_len;
  float scale;
  if (n != 11 || at::impl::torch_function_mode_enabled()) Py_RETURN_NONE;
  const at::Tensor* first = plain(args[0]);
  if (!first || first->dim() != 4 || first->size(0) < 1 || first->size(0) > 65535 || first->size(1) != 1) Py_RETURN_NONE;
  const int64_t B = first->size(0);
  if (!paged_pages(args + 1, B, false, &cache, &dtype, &device) || !paged_tensor(args[0], 4, dtype, device, &q) ||
      !q->is_contiguous() || (uintptr_t)q->data_ptr() % 16 || q->size(3) != cache.dim || q->size(2) % cache.heads)
    Py_RETURN_NONE;
  const int64_t hq = q->size(2), gs = hq / cache.heads, room = (int64_t)cache.table_pages * cache.page_rows;
  if (gs < 1 || gs > 16 || !paged_each(args[4], B, device, &lens, false) || !paged_each(args[5], B, device, &starts) ||
      !paged_int(args[9], room, &max_len) || max_len < 1 || max_len > room ||
      (max_len / 16 + 34) * (B > cache.heads ? B : cache.heads) > INT32_MAX || !paged_scale(args[7], cache.dim, &scale) ||
      !paged_values(args[6], at::kFloat, B, cache.heads, max_len, device, true, &scores, strides))
    Py_RETURN_NONE;
  const size_t bytes = ri_paged_attention_workspace_bytes((int)B, cache.heads, (int)gs, cache.dim, (int)max_len, scores != nullptr);
  void* const ws = paged_scratch(args[10], bytes, device);
  if (!ws || (args[8] != Py_True && args[8] != Py_False)) Py_RETURN_NONE;
  const bool with_lse = args[8] == Py_True;
  at::Tensor out = at::empty_like(*q), lse;
  if (with_lse) lse = at::empty({B, hq}, q->options().dtype(at::kFloat).requires_grad(false));
  void *qp = q->data_ptr(), *op = out.data_ptr(), *lp = with_lse ? lse.data_ptr() : nullptr;
  void *np = address(lens), *sp = address(starts), *cp = address(scores);
  const ri_stream_t stream = current_stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = ri_paged_attention(&cache, qp, (const int32_t*)np, (const int32_t*)sp, (float*)cp, strides[0], strides[1], op, (float*)lp,
                              (int)B, (int)gs, (int)max_len, scale, ws, bytes, stream);
  Py_END_ALLOW_THREADS
  if (status) return PyLong_FromLong(status);
  return with_lse ? pair_of(std::move(out), std::move(lse)) : THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// paged_append(key, value, k_pages, v_pages, block_table, cache_seqlens, new_seqlens, scores, positions, token_positions, budget,
// sinks, recent): status
PyObject* paged_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *key, *value, *lens, *held, *scores, *positions, *token;
  ri_paged_t cache;
  at::ScalarType dtype;
  int device;
  int64_t ks[3], vs[3], ss[2], ps[2], budget, sinks, recent;
  if (n != 13 || !(key = plain(args[0])) || key->dim() != 4 || key->size(0) < 1 || key->size(0) > 65535 || key->size(1) != 1) Py_RETURN_NONE;
  const int64_t B = key->size(0);
  if (!paged_pages(args + 2, B, true, &cache, &dtype, &device) || !paged_tensor(args[0], 4, dtype, device, &key) ||
      !paged_tensor(args[1], 4, dtype, device, &value) || key->size(2) != cache.heads || key->size(3) != cache.dim ||
      value->sizes() != key->sizes() || !paged_rows(*key, false, ks) || !paged_rows(*value, false, vs))
    Py_RETURN_NONE;
  const int64_t room = (int64_t)cache.table_pages * cache.page_rows;
  if (!paged_int(args[10], room, &budget) || !integers(args + 11, 1, &sinks) || !integers(args + 12, 1, &recent) || budget < 1 ||
      budget > room || sinks + recent >= budget || !paged_each(args[5], B, device, &lens, false) ||
      !paged_each(args[6], B, device, &held) || paged_meet(held, lens, B) || cache.k_pages == cache.v_pages ||
      !paged_values(args[7], at::kFloat, B, cache.heads, budget, device, true, &scores, ss) ||
      !paged_values(args[8], at::kInt, B, cache.heads, budget, device, true, &positions, ps) ||
      !paged_each(args[9], B, device, &token) || paged_meet(held, token, B) || (scores && !positions) || (positions && !token))
    Py_RETURN_NONE;
  void *kp = key->data_ptr(), *vp = value->data_ptr(), *np = lens->data_ptr(), *hp = address(held), *sp = address(scores),
       *pp = address(positions), *tp = address(token);
  const ri_stream_t stream = current_stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = ri_paged_append(&cache, kp, vp, ks[0], ks[2], vs[0], vs[2], (const int32_t*)np, (int32_t*)hp, (float*)sp, ss[0], ss[1],
                           (int32_t*)pp, ps[0], ps[1], (const int32_t*)tp, (int)B, (int)budget, (int)sinks, (int)recent, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
  END_HANDLE_TH_ERRORS
}

// paged_fill(key, value, k_pages, v_pages, block_table, new_seqlens, seqlens, weights, scores, positions, budget, sinks, recent,
// workspace): status
PyObject* paged_fill(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *key, *value, *held, *lens, *weights, *scores, *positions;
  ri_paged_t cache;
  at::ScalarType dtype;
  int device;
  int64_t ks[3], vs[3], ws[2], ss[2], ps[2], budget, sinks, recent;
  if (n != 14 || !(key = plain(args[0])) || key->dim() != 4 || key->size(0) < 1 || key->size(0) > 65535 || key->size(1) < 1 ||
      key->size(1) > 1 << 24)
    Py_RETURN_NONE;
  const int64_t B = key->size(0), T = key->size(1);
  if (!paged_pages(args + 2, B, true, &cache, &dtype, &device) || !paged_tensor(args[0], 4, dtype, device, &key) ||
      !paged_tensor(args[1], 4, dtype, device, &value) || key->size(2) != cache.heads || key->size(3) != cache.dim ||
      value->sizes() != key->sizes() || !paged_rows(*key, false, ks) || !paged_rows(*value, false, vs))
    Py_RETURN_NONE;
  const int64_t room = (int64_t)cache.table_pages * cache.page_rows;
  if (!paged_int(args[10], room, &budget) || !integers(args + 11, 1, &sinks) || !integers(args + 12, 1, &recent) || budget < 1 ||
      budget > room || sinks + recent > budget)
    Py_RETURN_NONE;
  const int64_t rows = T < budget ? T : budget;
  if (!paged_each(args[5], B, device, &held) || !paged_each(args[6], B, device, &lens) ||
      paged_meet(held, lens, B) || cache.k_pages == cache.v_pages ||
      !paged_values(args[7], at::kFloat, B, cache.heads, T, device, false, &weights, ws) ||
      !paged_values(args[8], at::kFloat, B, cache.heads, rows, device, true, &scores, ss) ||
      !paged_values(args[9], at::kInt, B, cache.heads, rows, device, true, &positions, ps) || (!weights && (T > budget || scores)) ||
      (scores && scores->data_ptr() == weights->data_ptr()))
    Py_RETURN_NONE;
  const size_t bytes = ri_paged_fill_workspace_bytes((int)B, cache.heads, (int)T, (int)budget);
  void* const work = bytes ? paged_scratch(args[13], bytes, device) : nullptr;
  if (bytes && !work) Py_RETURN_NONE;
  void *kp = key->data_ptr(), *vp = value->data_ptr(), *np = address(lens), *hp = address(held), *wp = address(weights),
       *sp = address(scores), *pp = address(positions);
  const ri_stream_t stream = current_stream();
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = ri_paged_fill(&cache, kp, vp, ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], (const int32_t*)np, (const float*)wp, ws[0], ws[1],
                         (int32_t*)hp, (float*)sp, ss[0], ss[1], (int32_t*)pp, ps[0], ps[1], (int)B, (int)T, (int)budget, (int)sinks,
                         (int)recent, work, bytes, stream);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(status);
  END_HANDLE_TH_ERRORS
}

// attention_weights(q, key, seqlens, scale, workspace): the weights, or a status that is not zero
PyObject* attention_weights(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *q, *key, *lens;
  at::ScalarType dtype;
  int64_t qs[3], ks[3];
  float scale;
  if (n != 5 || at::impl::torch_function_mode_enabled() || !(key = plain(args[1])) || !key->is_cuda() || key->dim() != 4 ||
      !half_type(key, dtype))
    Py_RETURN_NONE;
  const int device = key->get_device();
  if (device != c10::hip::current_device() || !paged_tensor(args[0], 4, dtype, device, &q)) Py_RETURN_NONE;
  const int64_t B = q->size(0), W = q->size(1), hq = q->size(2), dim = q->size(3), T = key->size(1), heads = key->size(2);
  if (B < 1 || heads < 1 || B > 65535 / heads || key->size(0) != B || key->size(3) != dim || (dim != 64 && dim != 128) || W < 1 ||
      W > T || T > 1 << 24 || hq % heads || hq / heads < 1 || hq / heads > 16 || !paged_rows(*q, false, qs) ||
      !paged_rows(*key, false, ks) || ks[1] > 1 << 23 || !paged_each(args[2], B, device, &lens) || !paged_scale(args[3], dim, &scale))
    Py_RETURN_NONE;
  const int gs = (int)(hq / heads);
  const size_t bytes = ri_attention_weights_workspace_bytes((int)B, (int)heads, gs, (int)W, (int)T);
  void* const ws = bytes ? paged_scratch(args[4], bytes, device) : nullptr;
  if (!ws) Py_RETURN_NONE;
  at::Tensor out = at::empty({B, heads, T}, key->options().dtype(at::kFloat).requires_grad(false));
  void *qp = q->data_ptr(), *kp = key->data_ptr(), *np = address(lens), *op = out.data_ptr();
  const ri_stream_t stream = current_stream();
  auto* call = dtype == at::kHalf ? ri_attention_weights_f16 : ri_attention_weights;
  int status;
  Py_BEGIN_ALLOW_THREADS
  status = call(qp, kp, (const int32_t*)np, (float*)op, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], (int)B, (int)W, (int)T, (int)heads,
                gs, (int)dim, scale, ws, bytes, stream);
  Py_END_ALLOW_THREADS
  if (status) return PyLong_FromLong(status);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

PyMethodDef step_methods[] = {{"run", (PyCFunction)(void (*)(void))step_run, METH_FASTCALL, nullptr},
                              {nullptr, nullptr, 0, nullptr}};
PyType_Slot step_slots[] = {{Py_tp_new, (void*)step_new},
                            {Py_tp_dealloc, (void*)step_dealloc},
                            {Py_tp_methods, (void*)step_methods},
                            {0, nullptr}};
PyType_Spec step_spec = {"_step_calls.Step", sizeof(Step), 0, Py_TPFLAGS_DEFAULT, step_slots};

PyMethodDef methods[] = {{"append", (PyCFunction)(void (*)(void))append, METH_FASTCALL, nullptr},
                         {"gemm_softmax", (PyCFunction)(void (*)(void))gemm_softmax, METH_FASTCALL, nullptr},
                         {"gather_vectors", (PyCFunction)(void (*)(void))gather_vectors, METH_FASTCALL, nullptr},
                         {"flash", (PyCFunction)(void (*)(void))flash, METH_FASTCALL, nullptr},
                         {"paged_attention", (PyCFunction)(void (*)(void))paged_attention, METH_FASTCALL, nullptr},
                         {"paged_append", (PyCFunction)(void (*)(void))paged_append, METH_FASTCALL, nullptr},
                         {"paged_fill", (PyCFunction)(void (*)(void))paged_fill, METH_FASTCALL, nullptr},
                         {"attention_weights", (PyCFunction)(void (*)(void))attention_weights, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_step_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__step_calls() {
  PyObject* m = PyModule_Create(&module);
  PyObject* type = m ? PyType_FromSpec(&step_spec) : nullptr;
  if (!type || PyModule_AddObject(m, "Step", type) < 0) return nullptr;
  return m;
}
