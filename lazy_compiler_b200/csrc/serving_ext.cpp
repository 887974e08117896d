// The calls of lazy_compiler_b200.serving: checks of the tensors, outputs, strides and the
// C-ABI call.  From Python these cost some 20 us a call, several times what the smaller
// kernels run; here a call costs about what a torch operation does.
//
// Every function takes positional arguments and returns its outputs, or the (negative)
// status of the C-ABI call.  A tensor that does not fit raises ValueError.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <cmath>
#include <string>

#include "lazyb200.h"

namespace {

// The entry points of the one loaded liblazyb200.so (bind).
struct Entries {
  decltype(&lc_window_attention) window_attention;
  decltype(&lc_paged_decode) paged_decode;
  decltype(&lc_cache_extend_recorded) cache_extend;
  decltype(&lc_cache_write_unless) cache_write;
  decltype(&lc_cache_fork_recorded) cache_fork;
  decltype(&lc_cache_release) cache_release;
  decltype(&lc_cache_compact) cache_compact;
  decltype(&lc_cache_copy) cache_copy;
} lib;
constexpr int kEntries = sizeof(Entries) / sizeof(void *);

std::string piece(const std::string &s) { return s; }
std::string piece(const char *s) { return s; }
std::string piece(int64_t v) { return std::to_string(v); }
std::string piece(const at::Device &d) { return d.str(); }
template <class... Parts>
[[noreturn]] void refuse(const Parts &...parts) {
  C10_THROW_ERROR(ValueError, (std::string() + ... + piece(parts)));
}

const at::Tensor &tensor(PyObject *o, const char *what) {
  if (!THPVariable_Check(o)) refuse(what, ": expected a tensor");
  return THPVariable_Unpack(o);
}
// None: no tensor
const at::Tensor *maybe(PyObject *o, const char *what) { return o == Py_None ? nullptr : &tensor(o, what); }

int64_t integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
bool truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v;
}
float scale_of(PyObject *o, int64_t d) {
  if (o == Py_None) return d > 0 ? (float)(1.0 / std::sqrt((double)d)) : 1.f;
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return (float)v;
}

const char *name_of(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return "float16";
    case at::kBFloat16: return "bfloat16";
    case at::kFloat: return "float32";
    case at::kDouble: return "float64";
    case at::kInt: return "int32";
    case at::kLong: return "int64";
    default: return c10::toString(t);
  }
}

std::string shape_text(at::IntArrayRef s) {
  std::string text = "(";
  for (size_t i = 0; i < s.size(); ++i) text += (i ? ", " : "") + std::to_string(s[i]);
  return text + ")";
}

void check(const at::Tensor &t, const char *what, const at::Tensor &like, at::ScalarType type, at::IntArrayRef shape) {
  if (t.scalar_type() != type || t.device() != like.device())
    refuse(what, ": ", name_of(t.scalar_type()), " on ", t.device(), ", expected ", name_of(type), " on ", like.device());
  if (t.sizes() != shape) refuse(what, ": shape ", shape_text(t.sizes()), ", expected ", shape_text(shape));
}
void check_ints(const at::Tensor &t, const char *what, const at::Tensor &like, at::IntArrayRef shape) {
  check(t, what, like, at::kInt, shape);
  if (!t.is_contiguous()) refuse(what, ": must be contiguous");
}
void check_inner(const at::Tensor &t, const char *what) {
  if (t.dim() && t.size(-1) > 1 && t.stride(-1) != 1) refuse(what, ": the last axis must be contiguous");
}
// A tensor to write has every element at its own place, as far as strides of zero go.
void check_out(const at::Tensor &t, const char *what) {
  for (int64_t i = 0; i < t.dim(); ++i)
    if (t.size(i) > 1 && t.stride(i) == 0) refuse(what, ": axis ", i, " is expanded, it cannot be written");
}
void check_cuda(const at::Tensor &t, const char *what) {
  if (!t.is_cuda()) refuse(what, ": on ", t.device(), ", the kernels run on CUDA devices only");
}
void check_axes(const at::Tensor &t, const char *what, int64_t axes) {
  if (t.dim() != axes) refuse(what, ": ", t.dim(), " axes, expected ", axes);
}
// Nothing here has a gradient: a tensor that asks for one is refused, not cut off without a word.
void check_no_gradient(const at::Tensor &t, const char *what) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(what, ": requires a gradient, which the serving operators do not compute; call them under torch.no_grad() or detach it");
}
// A tensor that a call writes: what autograd has saved of it is out of date afterwards.
void written(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
int attention_dtype(const at::Tensor &q) {
  if (q.scalar_type() != at::kHalf && q.scalar_type() != at::kBFloat16) refuse("q: ", name_of(q.scalar_type()), " is not float16 or bfloat16");
  check_cuda(q, "q");
  return q.scalar_type() == at::kHalf ? LC_F16 : LC_BF16;
}

// Makes the stream of a call current (None: the device's current one), so that what the call
// allocates is memory of the stream that it runs on: of another one, work queued there could
// still use the block, or be given it before this call has run.
struct On {
  c10::cuda::CUDAGuard device;
  c10::cuda::OptionalCUDAStreamGuard given;
  void *stream;
  On(PyObject *o, const at::Tensor &t) : device(t.device()) {
    if (o != Py_None) given.reset_stream(c10::cuda::getStreamFromExternal(reinterpret_cast<cudaStream_t>(static_cast<intptr_t>(integer(o))), t.get_device()));
    stream = c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
  }
};
// An uninitialised tensor on the device of `like`, without the dispatcher's way there.
at::Tensor fresh(at::IntArrayRef shape, at::ScalarType type, const at::Tensor &like) {
  return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), std::nullopt));
}

template <class T = void>
T *ptr(const at::Tensor *t) {
  return t ? static_cast<T *>(t->data_ptr()) : nullptr;
}
template <class T = void>
T *ptr(const at::Tensor &t) {
  return static_cast<T *>(t.data_ptr());
}

void arguments(Py_ssize_t n, Py_ssize_t expected) {
  if (n != expected) refuse("expected ", expected, " arguments, got ", n);
}

PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, kEntries);
  void **to = reinterpret_cast<void **>(&lib);
  for (int i = 0; i < kEntries; ++i) to[i] = reinterpret_cast<void *>(static_cast<intptr_t>(integer(a[i])));
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject *outputs(const at::Tensor &out, PyObject *given, const at::Tensor &lse) {
  PyObject *o = given != Py_None ? Py_NewRef(given) : THPVariable_Wrap(out);
  if (!lse.defined()) return o;
  PyObject *l = THPVariable_Wrap(lse);
  PyObject *both = PyTuple_Pack(2, o, l);
  Py_DECREF(o);
  Py_DECREF(l);
  return both;
}

// q, k, v, window, sinks, scale, q_lens, kv_lens, out, return_lse, stream
PyObject *window_attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 11);
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
  check_no_gradient(q, "q");
  check_no_gradient(k, "k");
  check_no_gradient(v, "v");
  const int dtype = attention_dtype(q);
  check_axes(q, "q", 4);
  check_axes(k, "k", 4);
  const int64_t batch = q.size(0), s_q = q.size(1), heads = q.size(2), d = q.size(3), s_kv = k.size(1), kv_heads = k.size(2);
  check(k, "k", q, q.scalar_type(), {batch, s_kv, kv_heads, d});
  check(v, "v", q, q.scalar_type(), {batch, s_kv, kv_heads, d});
  const at::Tensor *q_lens = maybe(a[6], "q_lens"), *kv_lens = maybe(a[7], "kv_lens"), *given = maybe(a[8], "out");
  if (q_lens) check_ints(*q_lens, "q_lens", q, {batch});
  if (kv_lens) check_ints(*kv_lens, "kv_lens", q, {batch});
  if (given) check(*given, "out", q, q.scalar_type(), {batch, s_q, heads, d}), check_out(*given, "out"), check_no_gradient(*given, "out");
  const On on(a[10], q);
  const at::Tensor out = given ? *given : fresh({batch, s_q, heads, d}, q.scalar_type(), q);
  const at::Tensor lse = truth(a[9]) ? fresh({batch, heads, s_q}, at::kFloat, q) : at::Tensor();
  const at::Tensor *views[4] = {&q, &k, &v, &out};
  const char *names[4] = {"q", "k", "v", "out"};
  int64_t strides[12];
  for (int x = 0; x < 4; ++x) {
    check_inner(*views[x], names[x]);
    for (int i = 0; i < 3; ++i) strides[x * 3 + i] = views[x]->stride(i);
  }
  const int status = lib.window_attention(dtype, ptr(q), ptr(k), ptr(v), ptr(out), lse.defined() ? ptr<float>(lse) : nullptr,
                                          ptr<int32_t>(q_lens), ptr<int32_t>(kv_lens), batch, s_q, s_kv, heads, kv_heads, d, strides,
                                          integer(a[3]), integer(a[4]), scale_of(a[5], d), on.stream);
  if (status) return PyLong_FromLong(status);
  if (given) written(out);
  return outputs(out, a[8], lse);
  END_HANDLE_TH_ERRORS
}

// q, k_pages, v_pages, table, lens, window, sinks, scale, out, return_lse, stream
PyObject *paged_decode(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 11);
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages");
  const at::Tensor &table = tensor(a[3], "table"), &lens = tensor(a[4], "lens");
  check_no_gradient(q, "q");
  check_no_gradient(k, "k_pages");
  check_no_gradient(v, "v_pages");
  const int dtype = attention_dtype(q);
  check_axes(q, "q", 3);
  check_axes(k, "k_pages", 4);
  check_axes(table, "table", 2);
  const int64_t slots = q.size(0), heads = q.size(1), d = q.size(2), width = table.size(1);
  const int64_t pages = k.size(0), kv_heads = k.size(1), page_size = k.size(2);
  check(k, "k_pages", q, q.scalar_type(), {pages, kv_heads, page_size, d});
  check(v, "v_pages", q, q.scalar_type(), {pages, kv_heads, page_size, d});
  check(table, "table", q, at::kInt, {slots, width});
  check_ints(lens, "lens", q, {slots});
  const at::Tensor *given = maybe(a[8], "out");
  if (given) check(*given, "out", q, q.scalar_type(), {slots, heads, d}), check_out(*given, "out"), check_no_gradient(*given, "out");
  const On on(a[10], q);
  const at::Tensor out = given ? *given : fresh({slots, heads, d}, q.scalar_type(), q);
  const at::Tensor lse = truth(a[9]) ? fresh({slots, heads}, at::kFloat, q) : at::Tensor();
  check_inner(q, "q");
  check_inner(k, "k_pages");
  check_inner(v, "v_pages");
  check_inner(out, "out");
  check_inner(table, "table");
  const int64_t strides[11] = {q.stride(0), q.stride(1), k.stride(0), k.stride(1), k.stride(2), v.stride(0),
                               v.stride(1), v.stride(2), out.stride(0), out.stride(1), table.stride(0)};
  const int status = lib.paged_decode(dtype, ptr(q), ptr(k), ptr(v), ptr(out), lse.defined() ? ptr<float>(lse) : nullptr,
                                      ptr<int32_t>(table), ptr<int32_t>(lens), slots, width, pages, page_size, heads, kv_heads, d,
                                      strides, integer(a[5]), integer(a[6]), scale_of(a[7], d), on.stream);
  if (status) return PyLong_FromLong(status);
  if (given) written(out);
  return outputs(out, a[8], lse);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- pages

// table, lens, refs, status (or None) of a cache, and of the maps to write.
struct Maps {
  at::Tensor table, lens, refs, status;
  int64_t slots, width, pages;
};
Maps maps_of(PyObject *const *a, const char *what) {
  const at::Tensor &table = tensor(a[0], what);
  check_cuda(table, what);
  check_axes(table, what, 2);
  Maps m = {table, tensor(a[1], what), tensor(a[2], what), at::Tensor(), table.size(0), table.size(1), 0};
  check_axes(m.refs, what, 1);
  m.pages = m.refs.size(0);
  check_ints(table, what, table, {m.slots, m.width});
  check_ints(m.lens, what, table, {m.slots});
  check_ints(m.refs, what, table, {m.pages});
  if (const at::Tensor *status = maybe(a[3], what)) {
    check_ints(*status, what, table, {2});
    m.status = *status;
  }
  return m;
}
// The maps to write: new ones (a[0] None), or the given ones with a status.
Maps into_of(const Maps &m, PyObject *const *a) {
  Maps to = m;
  if (a[0] == Py_None) {
    to.table = fresh({m.slots, m.width}, at::kInt, m.table);
    to.lens = fresh({m.slots}, at::kInt, m.table);
    to.refs = fresh({m.pages}, at::kInt, m.table);
    to.status = at::Tensor();
  } else {
    to = maps_of(a, "into");
    if (to.slots != m.slots || to.width != m.width || to.pages != m.pages || to.table.device() != m.table.device())
      refuse("into: other sizes or another device than the maps");
    for (const at::Tensor &t : {to.table, to.lens, to.refs, to.status})
      if (t.defined()) written(t);
  }
  if (!to.status.defined()) to.status = fresh({2}, at::kInt, m.table);
  return to;
}
// The words of a refusal (null where there are none).
int32_t *refusals_of(PyObject *o, const Maps &m) {
  const at::Tensor *t = maybe(o, "refusals");
  if (t) check_ints(*t, "refusals", m.table, {2});
  return ptr<int32_t>(t);
}
PyObject *wrapped(const Maps &m) {
  PyObject *parts[4] = {THPVariable_Wrap(m.table), THPVariable_Wrap(m.lens), THPVariable_Wrap(m.refs), THPVariable_Wrap(m.status)};
  PyObject *all = PyTuple_Pack(4, parts[0], parts[1], parts[2], parts[3]);
  for (PyObject *p : parts) Py_DECREF(p);
  return all;
}

struct Pool {
  void *data;
  int64_t planes, heads, page_size, token_bytes, strides[3];
};
Pool pool_of(const at::Tensor &t, const at::Tensor &like, int64_t pages) {
  if (t.dim() != 5 || t.device() != like.device() || t.size(1) != pages)
    refuse("pool: ", shape_text(t.sizes()), " on ", t.device(), ", expected [planes, ", pages, ", kv_heads, page_size, d] on ", like.device());
  check_no_gradient(t, "pool");
  check_inner(t, "pool");
  check_out(t, "pool");
  if (t.size(3) > 1 && t.stride(3) != t.size(4)) refuse("pool: the tokens of a head must be contiguous");
  const int64_t size = t.element_size();
  return {ptr(t), t.size(0), t.size(2), t.size(3), t.size(4) * size, {t.stride(0) * size, t.stride(1) * size, t.stride(2) * size}};
}

// maps (4), add, page_size, into (4), refusals, stream
PyObject *cache_extend(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 12);
  const Maps m = maps_of(a, "maps");
  const at::Tensor &add = tensor(a[4], "add");
  check_ints(add, "add", m.table, {m.slots});
  const On on(a[11], m.table);
  const Maps to = into_of(m, a + 6);
  const int status = lib.cache_extend(ptr<int32_t>(m.table), ptr<int32_t>(to.table), ptr<int32_t>(m.lens), ptr<int32_t>(to.lens),
                                      ptr<int32_t>(m.refs), ptr<int32_t>(to.refs), ptr<int32_t>(add), ptr<int32_t>(to.status),
                                      refusals_of(a[10], m), m.slots, m.width, m.pages, integer(a[5]), on.stream);
  return status ? PyLong_FromLong(status) : wrapped(to);
  END_HANDLE_TH_ERRORS
}

// k, v, k_pages, v_pages, maps (4), add, refusals, stream
PyObject *cache_write(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 11);
  const at::Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v"), &kp = tensor(a[2], "k_pages"), &vp = tensor(a[3], "v_pages");
  const Maps m = maps_of(a + 4, "maps");
  const at::Tensor &add = tensor(a[8], "add");
  check_ints(add, "add", m.table, {m.slots});
  check_no_gradient(k, "k");
  check_no_gradient(v, "v");
  check_no_gradient(kp, "k_pages");
  check_no_gradient(vp, "v_pages");
  check_axes(k, "k", 4);
  check_axes(kp, "k_pages", 4);
  const int64_t most = k.size(1), heads = k.size(2), d = k.size(3), page_size = kp.size(2), size = k.element_size();
  check(k, "k", m.table, k.scalar_type(), {m.slots, most, heads, d});
  check(v, "v", m.table, k.scalar_type(), {m.slots, most, heads, d});
  check(kp, "k_pages", m.table, k.scalar_type(), {m.pages, heads, page_size, d});
  check(vp, "v_pages", m.table, k.scalar_type(), {m.pages, heads, page_size, d});
  check_out(kp, "k_pages");
  check_out(vp, "v_pages");
  const at::Tensor *views[4] = {&k, &v, &kp, &vp};
  const char *names[4] = {"k", "v", "k_pages", "v_pages"};
  int64_t strides[12];
  for (int x = 0; x < 4; ++x) {
    check_inner(*views[x], names[x]);
    for (int i = 0; i < 3; ++i) strides[x * 3 + i] = views[x]->stride(i) * size;
  }
  // whether room was refused: the last extend's word, else the maps' own status
  const int32_t *refused = refusals_of(a[9], m);
  refused = refused ? refused + 1 : m.status.defined() ? ptr<int32_t>(m.status) : nullptr;
  const On on(a[10], m.table);
  const int status = lib.cache_write(ptr(k), ptr(v), ptr(kp), ptr(vp), ptr<int32_t>(m.table), ptr<int32_t>(m.lens), ptr<int32_t>(add),
                                     m.slots, most, m.width, m.pages, page_size, heads, d * size, strides, refused, on.stream);
  written(kp);
  written(vp);
  return PyLong_FromLong(status);
  END_HANDLE_TH_ERRORS
}

// pool, maps (4), parent, into (4), refusals, stream
PyObject *cache_fork(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 12);
  const Maps m = maps_of(a + 1, "maps");
  const Pool pool = pool_of(tensor(a[0], "pool"), m.table, m.pages);
  const at::Tensor &parent = tensor(a[5], "parent");
  check_ints(parent, "parent", m.table, {m.slots});
  const On on(a[11], m.table);
  const Maps to = into_of(m, a + 6);
  const int status = lib.cache_fork(pool.data, pool.planes, pool.heads, pool.token_bytes, pool.strides, ptr<int32_t>(m.table),
                                    ptr<int32_t>(to.table), ptr<int32_t>(m.lens), ptr<int32_t>(to.lens), ptr<int32_t>(m.refs),
                                    ptr<int32_t>(to.refs), ptr<int32_t>(parent), ptr<int32_t>(to.status), refusals_of(a[10], m),
                                    m.slots, m.width, m.pages, pool.page_size, on.stream);
  written(tensor(a[0], "pool"));
  return status ? PyLong_FromLong(status) : wrapped(to);
  END_HANDLE_TH_ERRORS
}

// maps (4), gone (or None), window, sinks, page_size, stream; in place
PyObject *cache_release(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 9);
  const Maps m = maps_of(a, "maps");
  const at::Tensor *gone = maybe(a[4], "gone");
  if (gone) check_ints(*gone, "gone", m.table, {m.slots});
  const On on(a[8], m.table);
  const Maps to = into_of(m, a);
  const int status = lib.cache_release(ptr<int32_t>(m.table), ptr<int32_t>(m.lens), ptr<int32_t>(m.refs), ptr<int32_t>(gone), integer(a[5]),
                                       integer(a[6]), ptr<int32_t>(to.status), m.slots, m.width, m.pages, integer(a[7]), on.stream);
  return status ? PyLong_FromLong(status) : wrapped(to);
  END_HANDLE_TH_ERRORS
}

// pool, maps (4), into (4), stream
PyObject *cache_compact(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 10);
  const Maps m = maps_of(a + 1, "maps");
  const Pool pool = pool_of(tensor(a[0], "pool"), m.table, m.pages);
  const On on(a[9], m.table);
  const Maps to = into_of(m, a + 5);
  const int status = lib.cache_compact(pool.data, pool.planes, pool.heads, pool.token_bytes, pool.strides, ptr<int32_t>(m.table),
                                       ptr<int32_t>(to.table), ptr<int32_t>(m.lens), ptr<int32_t>(to.lens), ptr<int32_t>(m.refs),
                                       ptr<int32_t>(to.refs), ptr<int32_t>(to.status), m.slots, m.width, m.pages, pool.page_size,
                                       on.stream);
  written(tensor(a[0], "pool"));
  return status ? PyLong_FromLong(status) : wrapped(to);
  END_HANDLE_TH_ERRORS
}

// pool, src, dst, stream
PyObject *cache_copy(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  arguments(n, 4);
  const at::Tensor &t = tensor(a[0], "pool"), &src = tensor(a[1], "src"), &dst = tensor(a[2], "dst");
  check_cuda(t, "pool");
  check_axes(t, "pool", 5);
  const Pool pool = pool_of(t, t, t.size(1));
  check_ints(src, "src", t, {src.numel()});
  check_ints(dst, "dst", t, {src.numel()});
  const On on(a[3], t);
  const int status = lib.cache_copy(pool.data, pool.planes, pool.heads, pool.token_bytes, pool.strides, ptr<int32_t>(src),
                                    ptr<int32_t>(dst), src.numel(), t.size(1), pool.page_size, on.stream);
  written(t);
  return PyLong_FromLong(status);
  END_HANDLE_TH_ERRORS
}

#define METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind),         METHOD(window_attention), METHOD(paged_decode),  METHOD(cache_extend), METHOD(cache_write),
                         METHOD(cache_fork),   METHOD(cache_release),    METHOD(cache_compact), METHOD(cache_copy),   {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", "Calls of lazy_compiler_b200.serving.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving() { return PyModule_Create(&module); }
