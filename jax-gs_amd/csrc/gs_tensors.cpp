// The host's look at lists of torch tensors for the many-tensor operators: pointers, types and
// sizes as the C entry points take them, with the checks of the arguments, in one call per
// list.  (From Python every attribute of every tensor is a call of 55 to 130 ns; a step of 148
// tensors has fourteen such sweeps.)
//
//   gather(tensors, device, what)                  -> (pointers, types, counts, kept)
//   pair(params, grads, shapes, device)            -> (to, to_types, of, of_types, counts, kept)
//   written(tensors, grads, others)                -> None: marks as modified in place what a call wrote
//   dense(tensors, device, what, rows)             -> (pointers, types, counts): what is written in place
//   take(tensors, fills, count, device, what)      -> (pointers, row_bytes, strides, rows, fills, out pointers,
//                                                      outputs, kept)
//   move(tensors, fills, index, device, what)      -> (pointers, row_bytes, strides, rows, fills, kept)
//
// The first three (five) of gather and pair are bytes objects holding int64 pointers, int32 types and int64 element
// counts.  A None among the tensors (gradients) has pointer 0 and count 0.  A tensor that is not
// contiguous (or a lazily negated view) is copied; `kept` holds the copies until the caller lets go of it.
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <exception>
#include <string>
#include <vector>

namespace {

struct Refused {
  PyObject* type;
  std::string text;
};

[[noreturn]] void refuse(PyObject* type, std::string text) { throw Refused{type, std::move(text)}; }

std::string dtype_of(PyObject* tensor) {
  std::string name = "another type";
  if (PyObject* dtype = PyObject_GetAttrString(tensor, "dtype")) {
    if (PyObject* s = PyObject_Str(dtype)) {
      if (const char* c = PyUnicode_AsUTF8(s)) name = c;
      Py_DECREF(s);
    }
    Py_DECREF(dtype);
  }
  PyErr_Clear();
  return name;
}

int type_of(const at::Tensor& t, PyObject* tensor, const char* what) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default:
      refuse(PyExc_TypeError, std::string(what) + ": tensors must be float32, bfloat16 or float16, not " + dtype_of(tensor));
  }
}

const at::Tensor& tensor_at(PyObject* list, Py_ssize_t i, const char* what) {
  PyObject* o = PyList_GET_ITEM(list, i);
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(what) + ": entry " + std::to_string(i) + " is not a tensor");
  return THPVariable_Unpack(o);
}

// Device -1 is the host, for tests of these checks: the operators refuse it before.
void on_device(const at::Tensor& t, int64_t device, const char* what, Py_ssize_t i) {
  if ((device >= 0 ? !t.is_cuda() : !t.is_cpu()) || t.get_device() != device)
    refuse(PyExc_ValueError, std::string(what) + ": tensor " + std::to_string(i) + " is on " + t.device().str() +
                                 ", not on cuda:" + std::to_string(device));
}

// Columns of a table, filled in place in bytes objects.
template <class T>
struct Column {
  PyObject* bytes;
  T* at;
  explicit Column(Py_ssize_t n) : bytes(PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(T))) {
    if (!bytes) refuse(PyExc_MemoryError, "out of memory");
    at = reinterpret_cast<T*>(PyBytes_AS_STRING(bytes));
  }
  ~Column() { Py_XDECREF(bytes); }
  Column(const Column&) = delete;
  PyObject* release() {
    PyObject* b = bytes;
    bytes = nullptr;
    return b;
  }
};

// A list that owns the contiguous copies; made when the first is.
struct Kept {
  PyObject* list = nullptr;
  ~Kept() { Py_XDECREF(list); }
  const at::Tensor& add(const at::Tensor& t) {
    if (!list && !(list = PyList_New(0))) refuse(PyExc_MemoryError, "out of memory");
    PyObject* o = THPVariable_Wrap(t.resolve_neg().contiguous());
    if (!o || PyList_Append(list, o) != 0) {
      Py_XDECREF(o);
      refuse(PyExc_MemoryError, "out of memory");
    }
    Py_DECREF(o);  // the list holds it
    return THPVariable_Unpack(o);
  }
  PyObject* release() {
    PyObject* l = list ? list : (Py_INCREF(Py_None), Py_None);
    list = nullptr;
    return l;
  }
};

// Whether the memory at data_ptr() is the tensor's values one after another.
bool plain(const at::Tensor& t) { return t.is_contiguous() && !t.is_neg(); }

bool same_shape(const at::Tensor& t, PyObject* shape) {
  const auto sizes = t.sizes();
  if (PyTuple_GET_SIZE(shape) != (Py_ssize_t)sizes.size()) return false;
  for (size_t d = 0; d < sizes.size(); ++d)
    if (PyLong_AsLongLong(PyTuple_GET_ITEM(shape, (Py_ssize_t)d)) != sizes[d]) return false;
  return true;
}

PyObject* do_gather(PyObject* list, int64_t device, const char* what) {
  const Py_ssize_t n = PyList_GET_SIZE(list);
  Column<int64_t> pointers(n), counts(n);
  Column<int32_t> types(n);
  Kept kept;
  for (Py_ssize_t i = 0; i < n; ++i) {
    pointers.at[i] = counts.at[i] = types.at[i] = 0;
    if (PyList_GET_ITEM(list, i) == Py_None) continue;
    const at::Tensor* t = &tensor_at(list, i, what);
    on_device(*t, device, what, i);
    types.at[i] = type_of(*t, PyList_GET_ITEM(list, i), what);
    if (!plain(*t)) t = &kept.add(*t);
    pointers.at[i] = (int64_t)(uintptr_t)t->data_ptr();
    counts.at[i] = t->numel();
  }
  return Py_BuildValue("NNNN", pointers.release(), types.release(), counts.release(), kept.release());
}

PyObject* do_pair(PyObject* params, PyObject* grads, PyObject* shapes, int64_t device) {
  const char* what = "AdamW";
  const Py_ssize_t n = PyList_GET_SIZE(params);
  if (n != PyList_GET_SIZE(shapes)) refuse(PyExc_ValueError, "AdamW: the parameters are not those of the state");
  if (n != PyList_GET_SIZE(grads))
    refuse(PyExc_ValueError, "AdamW: " + std::to_string(PyList_GET_SIZE(grads)) + " gradients for " +
                                 std::to_string(n) + " tensors");
  Column<int64_t> to(n), of(n), counts(n);
  Column<int32_t> to_types(n), of_types(n);
  Kept kept;
  std::vector<std::pair<uintptr_t, uintptr_t>> spans;
  spans.reserve((size_t)n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor& p = tensor_at(params, i, what);
    PyObject* shape = PyList_GET_ITEM(shapes, i);
    if (!PyTuple_Check(shape) || !same_shape(p, shape))
      refuse(PyExc_ValueError, "AdamW: the parameters are not those of the state");
    on_device(p, device, what, i);
    if (!plain(p))
      refuse(PyExc_ValueError, "AdamW: parameter " + std::to_string(i) + " must be contiguous");
    to_types.at[i] = type_of(p, PyList_GET_ITEM(params, i), what);
    to.at[i] = (int64_t)(uintptr_t)p.data_ptr();
    counts.at[i] = of.at[i] = of_types.at[i] = 0;
    if (p.numel()) spans.emplace_back((uintptr_t)p.data_ptr(), (uintptr_t)p.data_ptr() + p.nbytes());
    if (PyList_GET_ITEM(grads, i) == Py_None) continue;
    const at::Tensor* g = &tensor_at(grads, i, what);
    if (g->sizes() != p.sizes() || g->device() != p.device())
      refuse(PyExc_ValueError, "AdamW: gradient " + std::to_string(i) + " must be shaped like its parameter, on " +
                                   p.device().str());
    of_types.at[i] = type_of(*g, PyList_GET_ITEM(grads, i), what);
    if (!plain(*g)) g = &kept.add(*g);
    of.at[i] = (int64_t)(uintptr_t)g->data_ptr();
    counts.at[i] = p.numel();
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second)
      refuse(PyExc_ValueError, "AdamW: parameters overlap, or one is given twice");
  return Py_BuildValue("NNNNNN", to.release(), to_types.release(), of.release(), of_types.release(),
                       counts.release(), kept.release());
}

// Nothing here makes a graph: what autograd would have to follow is refused.
void no_graph(const at::Tensor& t, const char* what) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(PyExc_RuntimeError, std::string(what) + " is not differentiated: call it under torch.no_grad()");
  // torch.no_grad() does not stop the forward mode: a tangent would stay as it was, or be lost
  if (t._fw_grad(0).defined())
    refuse(PyExc_RuntimeError, std::string(what) + " is not differentiated: a tensor carries a tangent");
}

// The memory of a tensor's rows: rows * row bytes, `stride` from one to the next.
struct Rows {
  uintptr_t at;
  int64_t bytes, stride, rows;
  uintptr_t end() const { return rows && bytes ? at + (uintptr_t)((rows - 1) * stride + bytes) : at; }
};

bool overlap(const Rows& a, const Rows& b) {  // a.at <= b.at < a.end()
  // rows side by side in one array: one stride, and b's row between a's and a's next
  if (a.rows > 1 && b.rows > 1 && a.stride == b.stride) {
    const int64_t d = (int64_t)((b.at - a.at) % (uintptr_t)a.stride);
    return d < a.bytes || d + b.bytes > a.stride;
  }
  return true;
}

void check_overlap(std::vector<Rows>& all, const char* what) {
  std::sort(all.begin(), all.end(), [](const Rows& a, const Rows& b) { return a.at < b.at; });
  for (size_t i = 0; i < all.size(); ++i)
    for (size_t j = i + 1; j < all.size() && all[j].at < all[i].end(); ++j)
      if (overlap(all[i], all[j]))
        refuse(PyExc_ValueError, std::string(what) + ": tensors overlap, or one is given twice");
}

PyObject* do_dense(PyObject* list, int64_t device, const char* what, bool rows) {
  const Py_ssize_t n = PyList_GET_SIZE(list);
  Column<int64_t> pointers(n), counts(n);
  Column<int32_t> types(n);
  std::vector<Rows> spans;
  spans.reserve((size_t)n);
  for (Py_ssize_t i = 0; i < n; ++i) {
    pointers.at[i] = counts.at[i] = types.at[i] = 0;
    if (PyList_GET_ITEM(list, i) == Py_None) continue;
    const at::Tensor& t = tensor_at(list, i, what);
    on_device(t, device, what, i);
    types.at[i] = type_of(t, PyList_GET_ITEM(list, i), what);
    no_graph(t, what);
    // any order of the elements does, unless rows are told apart
    if (t.layout() != at::kStrided || t.is_neg() || !(rows ? t.is_contiguous() : t.is_non_overlapping_and_dense()))
      refuse(PyExc_ValueError, std::string(what) + ": tensor " + std::to_string(i) +
                                   (rows ? " must be contiguous" : " must be dense, without gaps between its elements"));
    pointers.at[i] = (int64_t)(uintptr_t)t.data_ptr();
    counts.at[i] = t.numel();
    if (t.numel()) spans.push_back(Rows{(uintptr_t)t.data_ptr(), (int64_t)t.nbytes(), (int64_t)t.nbytes(), 1});
  }
  check_overlap(spans, what);
  return Py_BuildValue("NNN", pointers.release(), types.release(), counts.release());
}

// Tensor i's rows, all with the same number of them; `own`: in place, nothing is copied.
Rows rows_of(const at::Tensor*& t, PyObject* list, Py_ssize_t i, int64_t device, const char* what, int64_t& rows,
             Kept* kept) {
  t = &tensor_at(list, i, what);
  if (t->layout() != at::kStrided || t->is_quantized())
    refuse(PyExc_TypeError, std::string(what) + ": tensor " + std::to_string(i) + " must be a plain strided one");
  on_device(*t, device, what, i);
  if (t->dim() == 0) refuse(PyExc_ValueError, std::string(what) + ": tensor " + std::to_string(i) + " has no rows");
  if (rows < 0) rows = t->size(0);
  if (t->size(0) != rows)
    refuse(PyExc_ValueError, std::string(what) + ": tensor " + std::to_string(i) + " has " + std::to_string(t->size(0)) +
                                 " rows, not " + std::to_string(rows));
  no_graph(*t, what);
  int64_t row = 1;
  bool inner = !t->is_neg() && !t->is_conj();
  for (int64_t d = t->dim() - 1; d > 0; --d) {
    if (t->size(d) != 1 && t->stride(d) != row) inner = false;
    row *= t->size(d);
  }
  if (!kept && row > 0 && rows > 1 && t->stride(0) < row) inner = false;
  if (row > 0 && rows > 0 && !inner) {
    if (!kept) refuse(PyExc_ValueError, std::string(what) + ": the rows of tensor " + std::to_string(i) + " must be contiguous and apart");
    t = &kept->add(t->resolve_conj());
  }
  const int64_t size = (int64_t)t->element_size();
  return Rows{(uintptr_t)t->data_ptr(), row * size, (t->dim() && rows > 1 ? t->stride(0) : row) * size, rows};
}

// The row that tensor i's fill gives, NULL without one.
int64_t fill_of(PyObject* fills, Py_ssize_t i, const at::Tensor& t, int64_t device, const char* what, Kept& kept) {
  if (fills == Py_None || PyList_GET_ITEM(fills, i) == Py_None) return 0;
  const at::Tensor* f = &tensor_at(fills, i, what);
  on_device(*f, device, what, i);
  if (f->scalar_type() != t.scalar_type() || f->sizes() != t.sizes().slice(1))
    refuse(PyExc_ValueError, std::string(what) + ": fill " + std::to_string(i) + " must be one row of its tensor");
  no_graph(*f, what);
  if (!plain(*f) || f->is_conj()) f = &kept.add(f->resolve_conj());
  return (int64_t)(uintptr_t)f->data_ptr();
}

PyObject* do_take(PyObject* list, PyObject* fills, int64_t count, int64_t device, const char* what) {
  const Py_ssize_t n = PyList_GET_SIZE(list);
  if (fills != Py_None && (!PyList_Check(fills) || PyList_GET_SIZE(fills) != n))
    refuse(PyExc_ValueError, std::string(what) + ": one fill for each tensor, or none");
  Column<int64_t> pointers(n), bytes(n), strides(n), fill(n), out(n);
  Kept kept, outputs;
  if (!(outputs.list = PyList_New(0))) refuse(PyExc_MemoryError, "out of memory");
  int64_t rows = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t;
    const Rows r = rows_of(t, list, i, device, what, rows, &kept);
    pointers.at[i] = (int64_t)r.at;
    bytes.at[i] = r.bytes;
    strides.at[i] = r.stride;
    fill.at[i] = fill_of(fills, i, *t, device, what, kept);
    auto shape = t->sizes().vec();
    shape[0] = count;
    const at::Tensor made = at::empty(shape, t->options().memory_format(at::MemoryFormat::Contiguous));
    out.at[i] = (int64_t)(uintptr_t)made.data_ptr();
    PyObject* o = THPVariable_Wrap(made);
    if (!o || PyList_Append(outputs.list, o) != 0) {
      Py_XDECREF(o);
      refuse(PyExc_MemoryError, "out of memory");
    }
    Py_DECREF(o);
  }
  return Py_BuildValue("NNNLNNNN", pointers.release(), bytes.release(), strides.release(), (long long)(rows < 0 ? 0 : rows),
                       fill.release(), out.release(), outputs.release(), kept.release());
}

PyObject* do_move(PyObject* list, PyObject* fills, const at::Tensor& index, int64_t device, const char* what) {
  const Py_ssize_t n = PyList_GET_SIZE(list);
  if (fills != Py_None && (!PyList_Check(fills) || PyList_GET_SIZE(fills) != n))
    refuse(PyExc_ValueError, std::string(what) + ": one fill for each tensor, or none");
  Column<int64_t> pointers(n), bytes(n), strides(n), fill(n);
  Kept kept;
  std::vector<Rows> spans, own;
  spans.reserve((size_t)n);
  int64_t rows = -1;
  for (Py_ssize_t i = 0; i < n; ++i) {
    const at::Tensor* t;
    const Rows r = rows_of(t, list, i, device, what, rows, nullptr);
    pointers.at[i] = (int64_t)r.at;
    bytes.at[i] = r.bytes;
    strides.at[i] = r.stride;
    fill.at[i] = fill_of(fills, i, *t, device, what, kept);
    if (r.rows && r.bytes) spans.push_back(r);
    if (fill.at[i] && r.bytes) own.push_back(Rows{(uintptr_t)fill.at[i], r.bytes, r.bytes, 1});
  }
  // what is read besides must not be written either
  if (index.numel()) own.push_back(Rows{(uintptr_t)index.data_ptr(), (int64_t)index.nbytes(), (int64_t)index.nbytes(), 1});
  for (const Rows& x : own)
    for (const Rows& r : spans)
      if (x.at < r.end() && r.at < x.end())
        refuse(PyExc_ValueError, std::string(what) + ": the index and the fills must not lie in the tensors that are moved");
  check_overlap(spans, what);
  return Py_BuildValue("NNNLNN", pointers.release(), bytes.release(), strides.release(), (long long)(rows < 0 ? 0 : rows),
                       fill.release(), kept.release());
}

// The kernels write through addresses: autograd, which has to refuse a backward pass over values that
// it saved and that are no longer there, is told of it.  Tensors without a gradient take no part, nor
// does a None among the others; tensors of inference mode count no versions.
void mark(PyObject* list, Py_ssize_t i) {
  const at::Tensor& t = tensor_at(list, i, "written");
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

PyObject* do_written(PyObject* tensors, PyObject* grads, PyObject* others) {
  if (PyList_GET_SIZE(tensors) != PyList_GET_SIZE(grads)) refuse(PyExc_ValueError, "written: lists of different lengths");
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(tensors); ++i)
    if (PyList_GET_ITEM(grads, i) != Py_None) mark(tensors, i);
  for (Py_ssize_t i = 0; i < PyList_GET_SIZE(others); ++i)
    if (PyList_GET_ITEM(others, i) != Py_None) mark(others, i);
  Py_RETURN_NONE;
}

template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& r) {
    PyErr_SetString(r.type, r.text.c_str());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject* gather(PyObject*, PyObject* args) {
  PyObject* list;
  long long device;
  const char* what;
  if (!PyArg_ParseTuple(args, "O!Ls", &PyList_Type, &list, &device, &what)) return nullptr;
  return guarded([&] { return do_gather(list, device, what); });
}

PyObject* pair(PyObject*, PyObject* args) {
  PyObject *params, *grads, *shapes;
  long long device;
  if (!PyArg_ParseTuple(args, "O!O!O!L", &PyList_Type, &params, &PyList_Type, &grads, &PyList_Type, &shapes, &device))
    return nullptr;
  return guarded([&] { return do_pair(params, grads, shapes, device); });
}

PyObject* written(PyObject*, PyObject* args) {
  PyObject *tensors, *grads, *others;
  if (!PyArg_ParseTuple(args, "O!O!O!", &PyList_Type, &tensors, &PyList_Type, &grads, &PyList_Type, &others)) return nullptr;
  return guarded([&] { return do_written(tensors, grads, others); });
}

PyObject* dense(PyObject*, PyObject* args) {
  PyObject* list;
  long long device;
  const char* what;
  int rows;
  if (!PyArg_ParseTuple(args, "O!Lsp", &PyList_Type, &list, &device, &what, &rows)) return nullptr;
  return guarded([&] { return do_dense(list, device, what, rows != 0); });
}

PyObject* take(PyObject*, PyObject* args) {
  PyObject *list, *fills;
  long long count, device;
  const char* what;
  if (!PyArg_ParseTuple(args, "O!OLLs", &PyList_Type, &list, &fills, &count, &device, &what)) return nullptr;
  return guarded([&] { return do_take(list, fills, count, device, what); });
}

PyObject* move(PyObject*, PyObject* args) {
  PyObject *list, *fills, *index;
  long long device;
  const char* what;
  if (!PyArg_ParseTuple(args, "O!OOLs", &PyList_Type, &list, &fills, &index, &device, &what)) return nullptr;
  return guarded([&] {
    if (!THPVariable_Check(index)) refuse(PyExc_TypeError, std::string(what) + ": the index is not a tensor");
    return do_move(list, fills, THPVariable_Unpack(index), device, what);
  });
}

PyMethodDef methods[] = {{"dense", dense, METH_VARARGS, "Pointers, types and counts of tensors written in place."},
                         {"take", take, METH_VARARGS, "Pointers and rows of tensors, and new tensors for rows taken."},
                         {"move", move, METH_VARARGS, "Pointers and rows of tensors that are moved in place."},
                         {"gather", gather, METH_VARARGS, "Pointers, types and counts of a list of tensors."},
                         {"pair", pair, METH_VARARGS, "The same of parameters and their gradients."},
                         {"written", written, METH_VARARGS, "Marks tensors as modified in place."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
