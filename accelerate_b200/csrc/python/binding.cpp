// The calls that every run of a program makes from Python, without ctypes: wrap, execute, free.  A call through
// ctypes costs about a microsecond and a half, and a run makes a dozen of them; a small kernel takes two.  Everything
// else of the C ABI goes through ctypes (backend.py), which also hands over the entry points' addresses.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <cstdint>
#include <cstring>
#include <memory>
#include <new>
#include <string>
#include <vector>

namespace {

int (*f_wrap)(void*, const char*, int, const int64_t*, void* const*, uint64_t*);
int (*f_run)(void*, const uint64_t*, int, uint64_t*, int);
int (*f_info)(void*, uint64_t, int, int*, int64_t*, int, int*, int32_t*);
int (*f_devptr)(void*, uint64_t, int, void**);
int (*f_free)(void*, uint64_t);
const char* (*f_error)();
PyObject* error_class;      // B200Error(code, message)
PyObject* type_names;       // scalar types in the library's order

PyObject* fail(int rc, const char* message) {
  // (a message may quote what the caller passed: any bytes)
  PyObject* text = PyUnicode_DecodeUTF8(message, (Py_ssize_t)strlen(message), "replace");
  PyObject* args = text ? Py_BuildValue("(iN)", rc, text) : nullptr;
  if (args) {
    PyErr_SetObject(error_class, args);
    Py_DECREF(args);
  }
  return nullptr;
}
bool to_u64(PyObject* o, uint64_t* v) {
  *v = PyLong_AsUnsignedLongLong(o);
  return !(*v == (uint64_t)-1 && PyErr_Occurred());
}
// One result of a run, as the library describes it; arrays of more dimensions or leaves than `few` take memory of their own
struct Result {
  Result() = default;
  Result(const Result&) = delete;
  uint64_t id = 0;
  int rank = 0, leaves = 0;
  struct { int64_t shape[8]; int32_t types[32]; void* ptrs[32]; } few;
  std::vector<int64_t> more_shape;
  std::vector<int32_t> more_types;
  std::vector<void*> more_ptrs;
  int64_t* shape = few.shape;
  int32_t* types = few.types;
  void** ptrs = few.ptrs;
};
constexpr int kRank = 1024, kLeaves = 1 << 16;
int describe(void* ctx, Result& r) {
  int rc = f_info(ctx, r.id, 8, &r.rank, r.shape, 32, &r.leaves, r.types);
  if (rc) {
    r.more_shape.resize(kRank);
    r.more_types.resize(kLeaves);
    r.more_ptrs.resize(kLeaves);
    r.shape = r.more_shape.data();
    r.types = r.more_types.data();
    r.ptrs = r.more_ptrs.data();
    rc = f_info(ctx, r.id, kRank, &r.rank, r.shape, kLeaves, &r.leaves, r.types);
  }
  for (int l = 0; !rc && l < r.leaves; ++l) rc = f_devptr(ctx, r.id, l, &r.ptrs[l]);
  return rc;
}

// setup(wrap, run, info, devptr, free, last_error, error class, type names)
PyObject* setup(PyObject*, PyObject* args) {
  unsigned long long a[6];
  PyObject *e, *t;
  if (!PyArg_ParseTuple(args, "KKKKKKOO!", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &e, &PyTuple_Type, &t)) return nullptr;
  f_wrap = (decltype(f_wrap))a[0];
  f_run = (decltype(f_run))a[1];
  f_info = (decltype(f_info))a[2];
  f_devptr = (decltype(f_devptr))a[3];
  f_free = (decltype(f_free))a[4];
  f_error = (decltype(f_error))a[5];
  Py_INCREF(e);
  Py_INCREF(t);
  error_class = e;
  type_names = t;
  Py_RETURN_NONE;
}

// wrap(ctx, element type, shape, pointers) -> id
PyObject* wrap(PyObject*, PyObject* const* args, Py_ssize_t n) {
  uint64_t ctx;
  if (n != 4 || !f_wrap) return PyErr_Format(PyExc_TypeError, "wrap(ctx, elt, shape, ptrs)");
  if (!to_u64(args[0], &ctx)) return nullptr;
  const char* elt = PyBytes_AsString(args[1]);
  if (!elt) return nullptr;
  PyObject *shape = PySequence_Fast(args[2], "a shape is a sequence"), *ptrs = nullptr;
  if (shape) ptrs = PySequence_Fast(args[3], "one pointer per leaf");
  PyObject* r = nullptr;
  if (ptrs) {
    std::vector<int64_t> sh;
    std::vector<void*> p;
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(shape); ++i) sh.push_back(PyLong_AsLongLong(PySequence_Fast_GET_ITEM(shape, i)));
    for (Py_ssize_t i = 0; i < PySequence_Fast_GET_SIZE(ptrs) && !PyErr_Occurred(); ++i) {
      PyObject* q = PySequence_Fast_GET_ITEM(ptrs, i);
      p.push_back(nullptr);
      if (q == Py_None) continue;
      // a number, or an object that holds one (ctypes.c_void_p, whose null is None)
      PyObject* number = PyIndex_Check(q) ? PyNumber_Index(q) : PyObject_GetAttrString(q, "value");
      if (!number) PyErr_Format(PyExc_TypeError, "a pointer is a number, a ctypes.c_void_p or None, not %R", q);
      if (number && number != Py_None) p.back() = PyLong_AsVoidPtr(number);
      Py_XDECREF(number);
    }
    if (!PyErr_Occurred()) {
      uint64_t id = 0;
      int rc;
      p.push_back(nullptr);
      sh.push_back(0);
      Py_BEGIN_ALLOW_THREADS
      rc = f_wrap((void*)ctx, elt, (int)sh.size() - 1, sh.data(), p.data(), &id);
      Py_END_ALLOW_THREADS
      r = rc ? fail(rc, f_error()) : PyLong_FromUnsignedLongLong(id);
    }
  }
  Py_XDECREF(shape);
  Py_XDECREF(ptrs);
  return r;
}

// execute(ctx, program, input ids, number of results) -> [(id, shape, leaf types, pointers)]
PyObject* execute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  uint64_t ctx, prog;
  if (n != 4 || !f_run) return PyErr_Format(PyExc_TypeError, "execute(ctx, program, ids, results)");
  if (!to_u64(args[0], &ctx) || !to_u64(args[1], &prog)) return nullptr;
  const long n_out = PyLong_AsLong(args[3]);
  if (n_out == -1 && PyErr_Occurred()) return nullptr;
  if (n_out < 0 || n_out > 1 << 20) return PyErr_Format(PyExc_ValueError, "bad number of results");
  PyObject* seq = PySequence_Fast(args[2], "ids are a sequence");
  if (!seq) return nullptr;
  std::vector<uint64_t> ins((size_t)PySequence_Fast_GET_SIZE(seq) + 1), outs((size_t)n_out + 1);
  std::unique_ptr<Result[]> results;     // (described once the library has accepted their number)
  const int n_in = (int)ins.size() - 1;
  bool ok = true;
  for (int i = 0; ok && i < n_in; ++i) ok = to_u64(PySequence_Fast_GET_ITEM(seq, i), &ins[i]);
  Py_DECREF(seq);
  if (!ok) return nullptr;
  // Everything that takes the context's lock, in one stretch without the interpreter's: another thread may hold the
  // former for as long as a download takes, and wait for the latter.
  int rc;
  std::string error;
  auto release = [&] { for (long k = 0; k < n_out; ++k) f_free((void*)ctx, outs[k]); };
  Py_BEGIN_ALLOW_THREADS
  rc = f_run((void*)prog, ins.data(), n_in, outs.data(), (int)n_out);
  if (rc) {
    error = f_error();
  } else {
    results.reset(new (std::nothrow) Result[(size_t)n_out]);
    for (long k = 0; results && !rc && k < n_out; ++k) {
      results[k].id = outs[k];
      rc = describe((void*)ctx, results[k]);
    }
    if (rc) error = f_error();
    if (rc || !results) release();       // (nobody else knows the results' ids)
  }
  Py_END_ALLOW_THREADS
  if (rc) return fail(rc, error.c_str());
  if (!results) return PyErr_NoMemory();
  PyObject* list = PyList_New(n_out);
  for (long k = 0; list && k < n_out; ++k) {
    const Result& r = results[k];
    PyObject *item = nullptr, *sh = PyTuple_New(r.rank), *ty = PyList_New(r.leaves), *pt = PyTuple_New(r.leaves);
    for (int d = 0; sh && d < r.rank; ++d) PyTuple_SET_ITEM(sh, d, PyLong_FromLongLong(r.shape[d]));
    for (int l = 0; ty && pt && l < r.leaves; ++l) {
      PyObject* name = PyTuple_GetItem(type_names, r.types[l]);
      Py_XINCREF(name);
      PyList_SET_ITEM(ty, l, name);
      PyTuple_SET_ITEM(pt, l, PyLong_FromVoidPtr(r.ptrs[l]));
    }
    if (sh && ty && pt && !PyErr_Occurred()) item = Py_BuildValue("(KOOO)", (unsigned long long)r.id, sh, ty, pt);
    Py_XDECREF(sh);
    Py_XDECREF(ty);
    Py_XDECREF(pt);
    if (!item) {
      Py_CLEAR(list);
      break;
    }
    PyList_SET_ITEM(list, k, item);
  }
  if (!list) {
    Py_BEGIN_ALLOW_THREADS
    release();
    Py_END_ALLOW_THREADS
  }
  return list;
}

// free(ctx, id): as b200_array_free; the result is its status
PyObject* free_(PyObject*, PyObject* const* args, Py_ssize_t n) {
  uint64_t ctx, id;
  if (n != 2 || !f_free) return PyErr_Format(PyExc_TypeError, "free(ctx, id)");
  if (!to_u64(args[0], &ctx) || !to_u64(args[1], &id)) return nullptr;
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f_free((void*)ctx, id);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

PyMethodDef methods[] = {{"setup", setup, METH_VARARGS, nullptr},
                         {"wrap", (PyCFunction)(void (*)(void))wrap, METH_FASTCALL, nullptr},
                         {"execute", (PyCFunction)(void (*)(void))execute, METH_FASTCALL, nullptr},
                         {"free", (PyCFunction)(void (*)(void))free_, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
