// The host's look at lists of torch tensors for the many-tensor operators: pointers, types and
// sizes as the C entry points take them, with the checks of the arguments, in one call per
// list.  (From Python every attribute of every tensor is a call of 55 to 130 ns; a step of 148
// tensors has fourteen such sweeps.)
//
//   gather(tensors, device, what)                  -> (pointers, types, counts, kept)
//   pair(params, grads, shapes, device)            -> (to, to_types, of, of_types, counts, kept)
//   written(tensors, grads, others)                -> None: marks as modified in place what a call wrote
//
// The first three (five) are bytes objects holding int64 pointers, int32 types and int64 element
// counts.  A None among the tensors (gradients) has pointer 0 and count 0.  A tensor that is not
// contiguous (or a lazily negated view) is copied; `kept` holds the copies until the caller lets go of it.
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

void on_device(const at::Tensor& t, int64_t device, const char* what, Py_ssize_t i) {
  if (!t.is_cuda() || t.get_device() != device)
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

PyMethodDef methods[] = {{"gather", gather, METH_VARARGS, "Pointers, types and counts of a list of tensors."},
                         {"pair", pair, METH_VARARGS, "The same of parameters and their gradients."},
                         {"written", written, METH_VARARGS, "Marks tensors as modified in place."},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
