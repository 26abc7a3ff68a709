// Usual calls of the serving operators made natively: a CPython module (no GPU code) that reads torch's tensors, makes the results, and calls
// the C ABI.  A small call costs as much as its checks, attribute by attribute in Python, as its launch (12 us a call; 3 to 6 with this module), and nothing
// may be remembered between calls, since a tensor's storage, shape and strides can be changed at any time.
//
// It only ever ACCEPTS: calls without `out` and `stream` whose tensors are plain ones (torch.Tensor itself) of the types, shapes and strides that
// drafts.py, pages.py, adapters.py and cache.py's cache_write take.  Anything else, whether it is wrong or merely unusual, gives None, and the Python
// functions decide and word the error.  An error of the C ABI comes back as its number.  No exception leaves this file.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>

#include "../../include/frisk_b200.h"

namespace {

constexpr size_t kBeside = 1 << 16;  // bytes
// execute's contexts by device, looked up anew by each call: one may have been closed, or given place to another; and the attributes that hold its address
PyObject *contexts = nullptr, *name_h = nullptr, *name_value = nullptr;

// the C ABI, as the library that Python has loaded offers it
struct Abi {
  decltype(&frisk_b200_draft_verify) verify;
  decltype(&frisk_b200_cache_fork) fork;
  decltype(&frisk_b200_cache_grow) grow;
  decltype(&frisk_b200_cache_compact) compact;
  decltype(&frisk_b200_cache_pages_workspace_bytes) pages_workspace;
  decltype(&frisk_b200_cache_copy) copy;
  decltype(&frisk_b200_cache_keep) keep;
  decltype(&frisk_b200_adapter_gemm) adapters;
  decltype(&frisk_b200_adapter_workspace_bytes) adapters_workspace;
  decltype(&frisk_b200_cache_write) write;
} abi = {};

struct Unusual {};  // left to Python

void require(bool usual) {
  if (!usual) throw Unusual();
}

const at::Tensor& tensor(PyObject* o) {
  require(THPVariable_CheckExact(o));
  const at::Tensor& t = THPVariable_Unpack(o);
  require(t.defined() && t.layout() == at::kStrided && t.is_cuda());
  return t;
}
int64_t whole(PyObject* o) {
  require(PyLong_CheckExact(o));
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw Unusual();
  }
  return x;
}
void* address(const at::Tensor& t) { return t.data_ptr(); }

int index_of(const at::Tensor& t) {
  const int dev = t.get_device();
  require(dev >= 0);
  return dev;
}
struct Owned {  // a reference, given back with the interpreter's lock held
  PyObject* object;
  explicit Owned(PyObject* o) : object(o) { require(o); }
  Owned(const Owned&) = delete;
  ~Owned() { Py_DECREF(object); }
};
PyObject* found(int dev) {  // the device's context, whose reference is new
  const Owned key(PyLong_FromLong(dev));
  PyObject* o = contexts ? PyDict_GetItemWithError(contexts, key.object) : nullptr;
  Py_XINCREF(o);
  return o;
}
// The library's context of a device, which stays while this does
struct Context {
  Owned owner;
  frisk_b200_ctx* handle;
  explicit Context(int dev) : owner(found(dev)) {
    const Owned held(PyObject_GetAttr(owner.object, name_h));  // None if it is closed
    require(held.object != Py_None);
    const Owned value(PyObject_GetAttr(held.object, name_value));
    handle = static_cast<frisk_b200_ctx*>(PyLong_AsVoidPtr(value.object));
    require(handle && !PyErr_Occurred());
  }
};
// a dense list of n elements
void* list(const at::Tensor& t, at::ScalarType type, int64_t n, int dev) {
  require(t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.get_device() == dev && t.is_contiguous());
  return address(t);
}
void* list(PyObject* o, at::ScalarType type, int64_t n, int dev) { return list(tensor(o), type, n, dev); }
// rows whose elements are neighbours
void rows_of(const at::Tensor& t, int dim, int dev) { require(t.dim() == dim && t.get_device() == dev && (t.stride(dim - 1) == 1 || t.size(dim - 1) <= 1)); }

at::Tensor made(at::IntArrayRef shape, at::ScalarType type, int dev) {
  return at::Tensor(at::detail::empty_cuda(shape, type, c10::Device(c10::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}
// The new tables of a call in one allocation (each costs 0.8 us; a fork and a grow 13.1 us, with allocations of their own 15.8): tensors of their own on one storage, on 64
// bytes.  What keeps one of them keeps all, as the functions' documentation says.
struct Results {
  at::Tensor held;
  int64_t bytes = 0;
  int64_t place(int64_t n) {  // of n more bytes
    const int64_t at = bytes;
    bytes += (n + 63) / 64 * 64;
    return at;
  }
  void allocate(int dev) { held = made({bytes}, at::kByte, dev); }
  at::Tensor at_place(int64_t place, at::IntArrayRef shape, at::ScalarType type) const {
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(held.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_storage_offset(place / (int64_t)c10::elementSize(type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    return t;
  }
};
void* stream_of(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return FRISK_B200_F32;
    case at::kHalf: return FRISK_B200_F16;
    case at::kBFloat16: return FRISK_B200_BF16;
    case at::kFloat8_e4m3fn: return FRISK_B200_E4M3;
    default: throw Unusual();
  }
}

// a call of the C ABI, without the interpreter's lock
template <typename F>
int call(F&& f) {
  PyThreadState* state = PyEval_SaveThread();
  const int rc = f();
  PyEval_RestoreThread(state);
  return rc;
}
PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* out = PyTuple_New((Py_ssize_t)tensors.size());
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) {
    PyObject* one = out ? THPVariable_Wrap(t) : nullptr;
    if (!one) {
      Py_XDECREF(out);
      return nullptr;
    }
    PyTuple_SET_ITEM(out, i++, one);
  }
  return out;
}

// Runs a function; what it does not take gives None.
template <typename F>
PyObject* usually(F&& f) {
  try {
    return f();
  } catch (...) {
    // (also what torch throws, as where memory runs out: Python meets it again, and reports it)
    if (PyErr_Occurred()) PyErr_Clear();
    Py_RETURN_NONE;
  }
}

// The sizes, type and tensors of a cache, a tuple of two or four tensors
frisk_b200_cache_desc cache_of(PyObject* cache, int* dev) {
  require(PyTuple_CheckExact(cache) && (PyTuple_GET_SIZE(cache) == 2 || PyTuple_GET_SIZE(cache) == 4));
  const bool four = PyTuple_GET_SIZE(cache) == 4;
  const at::Tensor &k = tensor(PyTuple_GET_ITEM(cache, 0)), &v = tensor(PyTuple_GET_ITEM(cache, 1));
  const int code = code_of(k.scalar_type());
  require(code != FRISK_B200_F32 && (code == FRISK_B200_E4M3) == four && v.scalar_type() == k.scalar_type());
  require(k.dim() == 4 && v.sizes() == k.sizes() && k.is_contiguous() && v.is_contiguous());
  *dev = index_of(k);
  require(v.get_device() == *dev);
  for (int i = 0; i < 4; ++i) require(k.size(i) <= INT32_MAX);
  frisk_b200_cache_desc d = {};
  d.pages = k.size(0);
  d.heads = (int32_t)k.size(1);
  d.page = (int32_t)k.size(2);
  d.D = (int32_t)k.size(3);
  d.dtype = code;
  d.rows = INT32_MAX;  // (calls that see no packed rows, only their counts)
  d.k = address(k);
  d.v = address(v);
  if (four) {
    uint8_t** parts[2] = {&d.k_exponent, &d.v_exponent};
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& e = tensor(PyTuple_GET_ITEM(cache, 2 + i));
      require(e.scalar_type() == at::kByte && e.sizes() == k.sizes().slice(0, 3) && e.is_contiguous() && e.get_device() == *dev);
      *parts[i] = static_cast<uint8_t*>(address(e));
    }
  }
  return d;
}
// an int32 table [batch, width]
const at::Tensor& table_of(PyObject* o, int dev) {
  const at::Tensor& t = tensor(o);
  require(t.scalar_type() == at::kInt);
  rows_of(t, 2, dev);
  require(t.size(0) < INT32_MAX && t.size(1) <= INT32_MAX);
  return t;
}

// verify(tokens, parents, starts, target, draft, accept, sample, max_new)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return usually([&]() -> PyObject* {
    require(n == 8);
    const at::Tensor &target = tensor(a[3]), &tokens = tensor(a[0]), &starts = tensor(a[2]);
    const int dev = index_of(target), code = code_of(target.scalar_type());
    require(code != FRISK_B200_E4M3);
    rows_of(target, 2, dev);
    const int64_t rows = target.size(0), vocab = target.size(1), batch = starts.dim() == 1 ? starts.size(0) - 1 : -1, max_new = whole(a[7]);
    require(batch >= 0 && batch < INT32_MAX && vocab <= INT32_MAX && max_new >= 1 && max_new <= 1024);
    frisk_b200_verify_desc d = {rows, target.stride(0), 0, (int32_t)batch, (int32_t)max_new, (int32_t)vocab, code, tokens.scalar_type() == at::kLong};
    void* draft = nullptr;
    if (a[4] != Py_None) {
      const at::Tensor& t = tensor(a[4]);
      require(t.scalar_type() == target.scalar_type() && t.sizes() == target.sizes());
      rows_of(t, 2, dev);
      d.draft_stride = t.stride(0);
      draft = address(t);
    }
    const void* p_tokens = list(tokens, d.tokens64 ? at::kLong : at::kInt, rows, dev);
    const int32_t* parents = a[1] == Py_None ? nullptr : static_cast<const int32_t*>(list(a[1], at::kInt, rows, dev));
    const int32_t* p_starts = static_cast<const int32_t*>(list(starts, at::kInt, batch + 1, dev));
    const float *accept = static_cast<const float*>(list(a[5], at::kFloat, rows, dev)), *sample = static_cast<const float*>(list(a[6], at::kFloat, batch, dev));
    // (one allocation for all would take 1 us off the host's 5.3, not off the call, which waits for the kernel)
    const at::Tensor kept = made({batch, max_new}, at::kInt, dev), counts = made({batch}, at::kInt, dev), next = made({batch}, tokens.scalar_type(), dev);
    void* stream = stream_of(dev);
    const Context context(dev);
    const int rc = call([&] {
      return abi.verify(context.handle, &d, p_tokens, parents, p_starts, address(target), draft, accept, sample, static_cast<int32_t*>(address(kept)),
                        static_cast<int32_t*>(address(counts)), address(next), stream);
    });
    return rc ? PyLong_FromLong(rc) : tuple_of({kept, counts, next});
  });
}

// change(which, cache, users, table, starts, lengths, parents): fork, grow and compact
PyObject* change(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return usually([&]() -> PyObject* {
    require(n == 7);
    const int which = (int)whole(a[0]);
    int dev;
    frisk_b200_cache_desc d = cache_of(a[1], &dev);
    const at::Tensor& table = table_of(a[3], dev);
    const int64_t batch = table.size(0), width = table.size(1);
    frisk_b200_page_tables t = {};
    t.users = static_cast<const int32_t*>(list(a[2], at::kInt, d.pages, dev));
    t.table_out_stride = width;
    d.table = static_cast<const int32_t*>(address(table));
    d.batch = (int32_t)batch;
    d.table_width = (int32_t)width;
    d.table_stride = table.stride(0);
    if (a[4] != Py_None) d.starts = static_cast<const int32_t*>(list(a[4], at::kInt, batch + 1, dev));
    if (a[5] != Py_None) d.lengths = static_cast<const int32_t*>(list(a[5], at::kInt, batch, dev));
    const int32_t* parents = a[6] == Py_None ? nullptr : static_cast<const int32_t*>(list(a[6], at::kInt, batch, dev));
    const size_t bytes = abi.pages_workspace(&d, which);
    const int64_t n_third = which == FRISK_B200_PAGES_COMPACT ? 1 : batch;
    Results r;
    const int64_t at_users = r.place(d.pages * 4), at_table = r.place(batch * width * 4), at_third = r.place(n_third * 4);
    // (a small workspace beside the results; a larger one would be held with them)
    const bool beside = bytes <= kBeside;
    const int64_t at_workspace = beside ? r.place((int64_t)bytes) : 0;
    r.allocate(dev);
    at::Tensor workspace;
    if (!beside) workspace = made({(int64_t)bytes}, at::kByte, dev);
    const at::Tensor users = r.at_place(at_users, {d.pages}, at::kInt), to = r.at_place(at_table, {batch, width}, at::kInt), third = r.at_place(at_third, {n_third}, at::kInt);
    t.users_out = static_cast<int32_t*>(address(users));
    t.table_out = static_cast<int32_t*>(address(to));
    t.lengths_out = static_cast<int32_t*>(address(third));
    void *ws = !bytes ? nullptr : beside ? static_cast<char*>(address(r.held)) + at_workspace : address(workspace), *stream = stream_of(dev);
    const Context context(dev);
    const int rc = call([&] {
      return which == FRISK_B200_PAGES_FORK   ? abi.fork(context.handle, &d, &t, parents, ws, bytes, stream)
             : which == FRISK_B200_PAGES_GROW ? abi.grow(context.handle, &d, &t, ws, bytes, stream)
                                              : abi.compact(context.handle, &d, &t, ws, bytes, stream);
    });
    return rc ? PyLong_FromLong(rc) : tuple_of({users, to, third});
  });
}

// the tables of packed rows: of a cache's descriptor
void tables_of(frisk_b200_cache_desc& d, PyObject* table, PyObject* starts, PyObject* lengths, int dev) {
  const at::Tensor& t = table_of(table, dev);
  const int64_t batch = t.size(0);
  d.table = static_cast<const int32_t*>(address(t));
  d.batch = (int32_t)batch;
  d.table_width = (int32_t)t.size(1);
  d.table_stride = t.stride(0);
  d.starts = static_cast<const int32_t*>(list(starts, at::kInt, batch + 1, dev));
  d.lengths = static_cast<const int32_t*>(list(lengths, at::kInt, batch, dev));
}

// write(cache, k, v, table, starts, lengths): True where it is done
PyObject* write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return usually([&]() -> PyObject* {
    require(n == 6);
    int dev;
    frisk_b200_cache_desc d = cache_of(a[0], &dev);
    const at::Tensor &k = tensor(a[1]), &v = tensor(a[2]);
    const int code = code_of(k.scalar_type());
    require((code == FRISK_B200_F16 || code == FRISK_B200_BF16) && (d.dtype == FRISK_B200_E4M3 || d.dtype == code));
    require(v.scalar_type() == k.scalar_type() && k.dim() == 3 && v.sizes() == k.sizes() && k.size(1) == d.heads && k.size(2) == d.D);
    frisk_b200_packed packed[2];
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& t = i ? v : k;
      require(t.stride(2) == 1 && t.get_device() == dev);
      packed[i] = {address(t), t.stride(0), t.stride(1)};
    }
    d.rows = k.size(0);
    tables_of(d, a[3], a[4], a[5], dev);
    void* stream = stream_of(dev);
    const Context context(dev);
    const int rc = call([&] { return abi.write(context.handle, &d, code, &packed[0], &packed[1], stream); });
    if (rc) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
  });
}

// keep(cache, table, starts, lengths, kept, counts)
PyObject* keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return usually([&]() -> PyObject* {
    require(n == 6);
    int dev;
    frisk_b200_cache_desc d = cache_of(a[0], &dev);
    tables_of(d, a[1], a[2], a[3], dev);
    const at::Tensor& kept = table_of(a[4], dev);
    const int64_t batch = d.batch;
    require(kept.size(0) == batch);
    const int32_t* counts = static_cast<const int32_t*>(list(a[5], at::kInt, batch, dev));
    const at::Tensor out = made({batch}, at::kInt, dev);
    void* stream = stream_of(dev);
    const Context context(dev);
    const int rc = call([&] {
      return abi.keep(context.handle, &d, static_cast<const int32_t*>(address(kept)), kept.stride(0), (int32_t)kept.size(1), counts,
                      static_cast<int32_t*>(address(out)), stream);
    });
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  });
}

// copy(cache, source, target, into): True where it is done
PyObject* copy(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return usually([&]() -> PyObject* {
    require(n == 4);
    int dev, other;
    const frisk_b200_cache_desc from = cache_of(a[0], &dev), into = cache_of(a[3], &other);
    const at::Tensor& source = tensor(a[1]);
    require(other == dev && source.dim() == 1);
    const int64_t count = source.size(0);
    const int32_t *s = static_cast<const int32_t*>(list(source, at::kInt, count, dev)), *t = static_cast<const int32_t*>(list(a[2], at::kInt, count, dev));
    void* stream = stream_of(dev);
    const Context context(dev);
    const int rc = call([&] { return abi.copy(context.handle, &from, &into, s, t, count, stream); });
    if (rc) return PyLong_FromLong(rc);
    Py_RETURN_TRUE;
  });
}

// adapters(x, a, b, c, starts, adapters, scales)
PyObject* adapters(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return usually([&]() -> PyObject* {
    require(n == 7);
    const at::Tensor &x = tensor(o[0]), &a = tensor(o[1]), &b = tensor(o[2]), &c = tensor(o[3]), &which = tensor(o[5]);
    const int dev = index_of(x), code = code_of(x.scalar_type()), code_c = code_of(c.scalar_type());
    require((code == FRISK_B200_F16 || code == FRISK_B200_BF16) && a.scalar_type() == x.scalar_type() && b.scalar_type() == x.scalar_type() &&
            (code_c == code || code_c == FRISK_B200_F32));
    rows_of(x, 2, dev);
    rows_of(a, 3, dev);
    rows_of(b, 3, dev);
    rows_of(c, 2, dev);
    frisk_b200_adapter_desc d = {};
    d.rows = x.size(0);
    d.K = x.size(1);
    d.N = b.size(1);
    require(a.size(2) == d.K && b.size(0) == a.size(0) && b.size(2) == a.size(1) && c.size(0) == d.rows && c.size(1) == d.N);
    require(a.size(0) <= INT32_MAX && a.size(1) >= 8 && a.size(1) <= 128 && which.dim() == 1 && which.size(0) < INT32_MAX);
    d.ldx = x.stride(0);
    d.lda = a.stride(1);
    d.a_step = a.stride(0);
    d.ldb = b.stride(1);
    d.b_step = b.stride(0);
    d.ldc = c.stride(0);
    d.ldo = d.N;
    d.rank = (int32_t)a.size(1);
    d.count = (int32_t)a.size(0);
    d.batch = (int32_t)which.size(0);
    d.dtype = code;
    d.dtype_c = code_c;
    const int32_t *starts = static_cast<const int32_t*>(list(o[4], at::kInt, d.batch + (int64_t)1, dev)),
                  *p_which = static_cast<const int32_t*>(list(which, at::kInt, d.batch, dev));
    const float* scales = o[6] == Py_None ? nullptr : static_cast<const float*>(list(o[6], at::kFloat, d.count, dev));
    const size_t bytes = abi.adapters_workspace(&d);
    at::Tensor workspace;
    if (bytes) workspace = made({(int64_t)bytes}, at::kByte, dev);
    const at::Tensor out = made({d.rows, d.N}, c.scalar_type(), dev);
    void *ws = bytes ? address(workspace) : nullptr, *stream = stream_of(dev);
    const Context context(dev);
    const int rc = call([&] {
      return abi.adapters(context.handle, &d, address(x), address(a), address(b), address(c), scales, starts, p_which, address(out), ws, bytes, stream);
    });
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  });
}

// library(contexts, ten addresses): where contexts are, and the C ABI's functions in the order of Abi
PyObject* library(PyObject*, PyObject* const* a, Py_ssize_t n) {
  void* at[10];
  if (n != 11 || !PyDict_Check(a[0])) {
    PyErr_SetString(PyExc_ValueError, "a dictionary and ten addresses");
    return nullptr;
  }
  for (int i = 0; i < 10; ++i) {
    at[i] = PyLong_AsVoidPtr(a[1 + i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address of 0");
      return nullptr;
    }
  }
  static_assert(sizeof(Abi) == sizeof(at), "one address each");
  memcpy(&abi, at, sizeof(at));
  if (!name_h) name_h = PyUnicode_InternFromString("_h");
  if (!name_value) name_value = PyUnicode_InternFromString("value");
  if (!name_h || !name_value) return nullptr;
  Py_INCREF(a[0]);
  Py_XSETREF(contexts, a[0]);
  Py_RETURN_NONE;
}
// context(device): the address that calls on that device would be given, or None
PyObject* context(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return usually([&]() -> PyObject* {
    require(n == 1);
    return PyLong_FromVoidPtr(Context((int)whole(a[0])).handle);
  });
}

template <typename F>
PyCFunction fast(F f) {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}
PyMethodDef methods[] = {{"verify", fast(verify), METH_FASTCALL, nullptr},     {"change", fast(change), METH_FASTCALL, nullptr},
                         {"write", fast(write), METH_FASTCALL, nullptr},       {"keep", fast(keep), METH_FASTCALL, nullptr},         {"copy", fast(copy), METH_FASTCALL, nullptr},
                         {"adapters", fast(adapters), METH_FASTCALL, nullptr}, {"library", fast(library), METH_FASTCALL, nullptr},
                         {"context", fast(context), METH_FASTCALL, nullptr},   {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }
