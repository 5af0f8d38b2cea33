// Python module _native: the paged K/V cache's entry points on torch tensors.
//
// One step of a live stream is a few kernels of 3-5 us each.  Reading and checking eight tensors from Python and
// handing their addresses to ctypes takes 5 us of the host a call, here under one; the launch itself takes 3.
// Host code only: it checks tensors (type, shape, device, contiguity) and calls the C ABI, whose own checks follow, through
// the addresses that bind() is given, so that there is one copy of the library and of its error message.  Each function
// returns the C ABI's status.  ValueError: a tensor does not fit; TypeError: something is no tensor.
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <initializer_list>
#include <stdexcept>

#include "trf_hip.h"

namespace {

decltype(&trf_page_plan_limited) page_plan_fn;
decltype(&trf_page_release) page_release_fn;
decltype(&trf_paged_append) paged_append_fn;
decltype(&trf_paged_attention) paged_attention_fn;

struct NoTensor : std::exception {};

struct Args {
  PyObject* const* a;
  int next = 0;
  long device;

  long number() {
    const long x = PyLong_AsLong(a[next++]);
    if (x == -1 && PyErr_Occurred()) throw NoTensor();
    return x;
  }
  int32_t number32(const char* name) {
    const long x = number();
    if (x != int32_t(x)) throw std::invalid_argument(c10::str(name, " must be a 32-bit number, got ", x));
    return int32_t(x);
  }
  double real() {
    const double x = PyFloat_AsDouble(a[next++]);
    if (x == -1.0 && PyErr_Occurred()) throw NoTensor();
    return x;
  }
  // A tensor on the current device; null for None where that is allowed.
  const at::Tensor* tensor(const char* name, bool optional = false) {
    PyObject* o = a[next++];
    if (optional && o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
      PyErr_Format(PyExc_TypeError, "%s must be a tensor, got %s", name, Py_TYPE(o)->tp_name);
      throw NoTensor();
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda() || t.device().index() != device)
      throw std::invalid_argument(c10::str("the tensors must be on the current device, cuda:", device, ": ", name, " is on ", t.device()));
    return &t;
  }
};

void need(const at::Tensor& t, const char* name, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.sizes() != shape || !t.is_contiguous())
    throw std::invalid_argument(c10::str(name, " must be contiguous ", type, " ", shape, ", got ", t.scalar_type(), " ", t.sizes()));
}

template <class T>
T* address(const at::Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

int32_t* ints(Args& args, const char* name, std::initializer_list<int64_t> shape) {
  const at::Tensor* t = args.tensor(name);
  need(*t, name, at::kInt, shape);
  return address<int32_t>(t);
}

int32_t length(const at::Tensor& t, const char* name, int64_t dims, int64_t dim) {
  if (t.dim() != dims) throw std::invalid_argument(c10::str(name, " must have ", dims, " dimensions, got ", t.sizes()));
  if (t.size(dim) > INT32_MAX) throw std::invalid_argument(c10::str(name, " is too large: ", t.sizes()));
  return int32_t(t.size(dim));
}

// Row stride, in elements, of rows t [n][heads][dim] whose heads are contiguous (a slice of a projection's rows is).
int64_t row_stride(const at::Tensor& t, const char* name, at::ScalarType type, int64_t n, int64_t heads, int64_t dim) {
  const int64_t shape[] = {n, heads, dim};
  if (t.scalar_type() != type || t.sizes() != at::IntArrayRef(shape))
    throw std::invalid_argument(c10::str(name, " must be ", type, " ", at::IntArrayRef(shape), ", got ", t.scalar_type(), " ", t.sizes()));
  if (t.stride(2) != 1 || (heads > 1 && t.stride(1) != dim))
    throw std::invalid_argument(c10::str(name, "'s heads must be contiguous in a row, got strides ", t.strides()));
  return n > 1 ? t.stride(0) : heads * dim;
}

struct Cache {
  at::ScalarType type;
  int32_t code, pages, page_size, heads, dim;
  uint16_t *K, *V;
};

Cache cache(Args& args) {
  const at::Tensor &K = *args.tensor("K"), &V = *args.tensor("V");
  Cache c{};
  c.type = K.scalar_type();
  if ((c.type != at::kBFloat16 && c.type != at::kHalf) || K.dim() != 6 || K.size(4) != 16 || K.size(5) != 8 || !K.is_contiguous())
    throw std::invalid_argument(c10::str("K must be contiguous bfloat16 or float16 [pages, kv heads, page size / 16, head dim / 8, 16, 8], "
                                         "got ", c.type, " ", K.sizes()));
  const int64_t v[] = {K.size(0), K.size(1), 2 * K.size(2), 8 * K.size(3), 8};
  need(V, "V", c.type, v);
  c.code = c.type == at::kHalf ? TRF_F16 : TRF_BF16;
  if (K.size(0) > INT32_MAX || K.size(1) > 65535 || K.size(2) > 16 || K.size(3) > 16)
    throw std::invalid_argument(c10::str("K is too large: ", K.sizes()));
  c.pages = int32_t(K.size(0)), c.heads = int32_t(K.size(1));
  c.page_size = 16 * int32_t(K.size(2)), c.dim = 8 * int32_t(K.size(3));
  c.K = address<uint16_t>(&K), c.V = address<uint16_t>(&V);
  return c;
}

trf_stream_t stream_of(Args& args) {
  return reinterpret_cast<trf_stream_t>(PyLong_AsVoidPtr(args.a[args.next++]));
}

// Each function takes (device, stream, ...) and n arguments in all.
template <class F>
PyObject* call(PyObject* const* a, Py_ssize_t got, Py_ssize_t n, F f) {
  if (got != n || !page_plan_fn) {
    PyErr_Format(PyExc_TypeError, got != n ? "expected %zd arguments, got %zd" : "not bound", n, got);
    return nullptr;
  }
  try {
    Args args{a};
    args.device = args.number();
    const trf_stream_t stream = stream_of(args);
    const int rc = f(args, stream);
    return PyErr_Occurred() ? nullptr : PyLong_FromLong(rc);
  } catch (const NoTensor&) {  // the error is set
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// f(a...) without the interpreter's lock.  The arguments are formed with it: asking some tensors for their address throws,
// and the C functions do not.
template <class F, class... A>
int unlocked(F* f, A... a) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f(a...);
  Py_END_ALLOW_THREADS
  return rc;
}

// max_length may be left out: as long as the table's rows.
PyObject* page_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(a, n, n == 12 ? 12 : 11, [n](Args& x, trf_stream_t stream) {
    const at::Tensor &state = *x.tensor("state"), &n_new = *x.tensor("n_new"), &pool = *x.tensor("pool"), &table = *x.tensor("table");
    const int32_t page_size = x.number32("page_size"), R = length(table, "table", 2, 0), max_pages = length(table, "table", 2, 1);
    const int32_t pages = length(pool, "pool", 1, 0);
    need(state, "state", at::kInt, {2 + int64_t(R)});
    need(n_new, "n_new", at::kInt, {R});
    need(pool, "pool", at::kInt, {pages});
    need(table, "table", at::kInt, {R, max_pages});
    int32_t* out = ints(x, "state_out", {2 + int64_t(R)});
    int32_t* starts = ints(x, "starts", {int64_t(R) + 1});
    const at::Tensor& slots = *x.tensor("slots");
    const int32_t rows = length(slots, "slots", 1, 0);
    need(slots, "slots", at::kInt, {rows});
    int32_t* positions = ints(x, "positions", {rows});
    const int32_t longest = n == 12 ? x.number32("max_length") : int32_t(std::min<int64_t>(int64_t(max_pages) * page_size, INT32_MAX));
    return unlocked(page_plan_fn, address<int32_t>(&state), address<int32_t>(&n_new), R, rows, address<int32_t>(&pool), pages,
                    page_size, address<int32_t>(&table), max_pages, longest, out, starts, address<int32_t>(&slots), positions, stream);
  });
}

PyObject* page_release(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(a, n, 8, [](Args& x, trf_stream_t stream) {
    const at::Tensor &state = *x.tensor("state"), &done = *x.tensor("done"), &pool = *x.tensor("pool"), &table = *x.tensor("table");
    const int32_t page_size = x.number32("page_size"), R = length(table, "table", 2, 0), max_pages = length(table, "table", 2, 1);
    const int32_t pages = length(pool, "pool", 1, 0);
    need(state, "state", at::kInt, {2 + int64_t(R)});
    need(done, "done", done.scalar_type() == at::kByte ? at::kByte : at::kBool, {R});
    need(pool, "pool", at::kInt, {pages});
    need(table, "table", at::kInt, {R, max_pages});
    int32_t* out = ints(x, "state_out", {2 + int64_t(R)});
    return unlocked(page_release_fn, address<int32_t>(&state), address<uint8_t>(&done), R, address<int32_t>(&pool), pages, page_size,
                    address<int32_t>(&table), max_pages, out, stream);
  });
}

PyObject* paged_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(a, n, 11, [](Args& x, trf_stream_t stream) {
    const at::Tensor &k = *x.tensor("k"), &v = *x.tensor("v");
    const Cache c = cache(x);
    const int32_t rows = length(k, "k", 3, 0);
    const int64_t ks = row_stride(k, "k", c.type, rows, c.heads, c.dim), vs = row_stride(v, "v", c.type, rows, c.heads, c.dim);
    int32_t* slots = ints(x, "slots", {rows});
    const at::Tensor *positions = x.tensor("positions", true), *rope = x.tensor("rope", true);
    const at::Tensor *q = x.tensor("q", true), *q_out = x.tensor("q_out", true);
    if (positions) need(*positions, "positions", at::kInt, {rows});
    int32_t P = 0, heads = 0;
    int64_t qs = 0;
    if (rope) {
      P = length(*rope, "rope", 3, 1);
      need(*rope, "rope", at::kFloat, {2, P, c.dim / 2});
      if (!positions) throw std::invalid_argument("a rotation needs positions");
    }
    if (q) {
      heads = length(*q, "q", 3, 1);
      qs = row_stride(*q, "q", c.type, rows, heads, c.dim);
      if (!q_out) throw std::invalid_argument("q needs a q_out");
      need(*q_out, "q_out", c.type, {rows, heads, c.dim});
    }
    return unlocked(paged_append_fn, address<uint16_t>(q), qs, heads, address<uint16_t>(&k), ks, address<uint16_t>(&v), vs, c.code,
                    rows, slots, address<int32_t>(positions), address<float>(rope), P, c.K, c.V, c.pages, c.page_size, c.heads, c.dim,
                    address<uint16_t>(q_out), stream);
  });
}

// max_new, max_len: -1 for the largest that the tensors allow; scale: 0 for dim ** -0.5 (None in Python).
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return call(a, n, 16, [](Args& x, trf_stream_t stream) {
    const at::Tensor& q = *x.tensor("q");
    const Cache c = cache(x);
    const at::Tensor& table = *x.tensor("table");
    const int32_t rows = length(q, "q", 3, 0), heads = length(q, "q", 3, 1);
    const int32_t R = length(table, "table", 2, 0), max_pages = length(table, "table", 2, 1);
    const int64_t qs = row_stride(q, "q", c.type, rows, heads, c.dim);
    need(table, "table", at::kInt, {R, max_pages});
    int32_t *starts = ints(x, "starts", {int64_t(R) + 1}), *lens = ints(x, "lens", {R});
    const at::Tensor& O = *x.tensor("O");
    need(O, "O", c.type, {rows, int64_t(heads) * c.dim});
    const bool no_scale = x.a[x.next] == Py_None;
    const float scale = no_scale ? (x.next++, 1.f / sqrtf(float(c.dim))) : float(x.real());
    const int32_t causal = x.number32("causal"), window = x.number32("window");
    const at::Tensor* gate = x.tensor("gate", true);
    if (gate) need(*gate, "gate", at::kFloat, {rows, heads});
    const bool no_new = x.a[x.next] == Py_None;
    const int32_t max_new = no_new ? (x.next++, rows) : x.number32("max_new");
    const bool no_len = x.a[x.next] == Py_None;
    const int32_t max_len = no_len ? (x.next++, INT32_MAX) : x.number32("max_len");
    const at::Tensor* ws = x.tensor("ws", true);
    if (ws) need(*ws, "ws", at::kByte, {ws->numel()});
    return unlocked(paged_attention_fn, address<uint16_t>(&q), qs, heads, c.K, c.V, c.code, c.pages, c.page_size, c.heads, c.dim,
                    address<int32_t>(&table), max_pages, starts, lens, R, rows, max_new, max_len, scale, causal, window,
                    address<float>(gate), address<uint16_t>(&O), address<void>(ws), ws ? size_t(ws->numel()) : 0, stream);
  });
}

PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 4) {
    PyErr_SetString(PyExc_TypeError, "expected the addresses of 4 functions");
    return nullptr;
  }
  void* p[4];
  for (int i = 0; i < 4; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "an address is 0");
      return nullptr;
    }
  }
  page_plan_fn = reinterpret_cast<decltype(page_plan_fn)>(p[0]);
  page_release_fn = reinterpret_cast<decltype(page_release_fn)>(p[1]);
  paged_append_fn = reinterpret_cast<decltype(paged_append_fn)>(p[2]);
  paged_attention_fn = reinterpret_cast<decltype(paged_attention_fn)>(p[3]);
  Py_RETURN_NONE;
}

#define TRF_METHOD(name, doc) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, doc}

PyMethodDef methods[] = {
    TRF_METHOD(bind, "bind(page_plan_limited, page_release, paged_append, paged_attention): the C functions' addresses"),
    TRF_METHOD(page_plan,
               "page_plan(device, stream, state, n_new, pool, table, page_size, state_out, starts, slots, positions[, max_length])"),
    TRF_METHOD(page_release, "page_release(device, stream, state, done, pool, table, page_size, state_out)"),
    TRF_METHOD(paged_append, "paged_append(device, stream, k, v, K, V, slots, positions, rope, q, q_out)"),
    TRF_METHOD(paged_attention,
               "paged_attention(device, stream, q, K, V, table, starts, lens, O, scale, causal, window, gate, max_new, max_len, ws)"),
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, methods};

}  // namespace

// abi_version: of the header that this was compiled with.  functions: what bind() wants the addresses of, in its order.
PyMODINIT_FUNC PyInit__native() {
  PyObject* m = PyModule_Create(&module);
  PyObject* names = Py_BuildValue("(ssss)", "trf_page_plan_limited", "trf_page_release", "trf_paged_append", "trf_paged_attention");
  if (m && names && PyModule_AddIntConstant(m, "abi_version", TRF_ABI_VERSION) == 0 && PyModule_AddObject(m, "functions", names) == 0)
    return m;
  Py_XDECREF(names);
  Py_XDECREF(m);
  return nullptr;
}
