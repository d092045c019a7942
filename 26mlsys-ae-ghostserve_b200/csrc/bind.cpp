// bind.cpp — the calls of the KV-pool operators from torch tensors.
//
// A decode step makes these calls once per layer, for kernels of a few
// microseconds: checking ten tensors and marshalling twenty arguments in Python
// took longer (17 us a call for a slot plan) than the kernels run. Here the
// tensors are checked, the outputs allocated and the C ABI called (gsec.h, whose
// return codes go to the package's own exceptions). Arguments are positional; the
// Python functions of kvpool.py carry names, defaults and documentation.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <exception>
#include <string>

#include "gsec.h"

namespace {

PyObject* g_check = nullptr;  // _lib.check: raises for a return code
PyTypeObject* g_plan = nullptr;  // kvpool.SlotPlan

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  PyErr_SetString(PyExc_ValueError, buf);
  throw Refused{};
}

#define NEED(cond, ...) \
  do {                  \
    if (!(cond)) refuse(__VA_ARGS__); \
  } while (0)

const at::Tensor& tensor(PyObject* o, const char* what) {
  NEED(THPVariable_Check(o), "%s must be a tensor", what);
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o, const char* what) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  (void)what;
  return v;
}

int32_t small(PyObject* o, const char* what) {
  const int64_t v = integer(o, what);
  NEED(v >= INT32_MIN && v <= INT32_MAX, "%s=%lld does not fit 32 bits", what, (long long)v);
  return (int32_t)v;
}

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{};
  return v;
}

void no_grad(const at::Tensor& t, const char* what) {
  NEED(!(t.requires_grad() && c10::GradMode::is_enabled()), "%s requires a gradient: the operator has no backward pass", what);
  NEED(!t._fw_grad(0).defined(), "%s carries a forward-mode tangent: the operator has no derivative", what);
}

// The first tensor names the device.
struct Call {
  c10::Device device;
  c10::OptionalDeviceGuard guard;
  explicit Call(const at::Tensor& t, const char* what) : device(t.device()) {
    NEED(t.is_cuda(), "%s must be a CUDA tensor", what);
    guard.reset_device(device);
  }
  void on(const at::Tensor& t, const char* what) const {
    NEED(t.device() == device, "%s must be a tensor on %s", what, device.str().c_str());
  }
  // A contiguous tensor of the type, of `size` elements unless negative.
  void* flat(const at::Tensor& t, const char* what, at::ScalarType type, int64_t size = -1) const {
    on(t, what);
    NEED(t.scalar_type() == type && t.is_contiguous(), "%s must be a contiguous %s tensor", what, at::toString(type));
    NEED(size < 0 || t.numel() == size, "%s must have %lld elements, has %lld", what, (long long)size,
         (long long)t.numel());
    return t.data_ptr();
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
  at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    return at::detail::empty_cuda(shape, type, device, std::nullopt);
  }
};

// `count` elements from byte `from` of a new tensor, as a tensor of their own. (Two
// allocations and a split through the dispatcher took 2.5 us more.)
at::Tensor piece(const at::Tensor& t, at::ScalarType type, int64_t from, int64_t count) {
  const caffe2::TypeMeta meta = c10::scalarTypeToTypeMeta(type);
  at::Tensor r = at::detail::make_tensor<at::TensorImpl>(at::TensorImpl::VIEW, at::Storage(t.storage()), t.key_set(), meta);
  r.unsafeGetTensorImpl()->set_storage_offset(from / (int64_t)meta.itemsize());
  r.unsafeGetTensorImpl()->set_sizes_contiguous({count});
  return r;
}

void finish(int rc) {
  if (rc == GSEC_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "i", rc);  // raises
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "libgsec returned %d", rc);
  throw Refused{};
}

struct Table {
  int32_t* at;
  int64_t pitch;
  int32_t width;
};

Table table_of(const Call& c, const at::Tensor& t, int64_t batch) {
  c.on(t, "table");
  NEED(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == batch,
       "table must be an int32 tensor [%lld, pages]", (long long)batch);
  const int64_t w = t.size(1);
  NEED(w < (1ll << 31) && (w <= 1 || t.stride(1) == 1) && (batch <= 1 || t.stride(0) >= w),
       "the rows of table must be contiguous and must not overlap");
  return {static_cast<int32_t*>(t.data_ptr()), t.stride(0) > w ? t.stride(0) : w, (int32_t)w};
}

struct Pool {
  char* at;
  int64_t heads, dim, pitch, plane, rows;
};

Pool pool_of(const Call& c, const at::Tensor& t, at::ScalarType type) {
  NEED(t.dim() == 4 && t.size(1) == 2, "pool must be a CUDA tensor [slots, 2 (K, V), heads, dim]");
  c.on(t, "pool");
  NEED(t.scalar_type() == type, "pool must be a %s tensor", at::toString(type));
  const int64_t h = t.size(2), d = t.size(3), es = t.element_size();
  NEED((d <= 1 || t.stride(3) == 1) && (h <= 1 || t.stride(2) == d), "a pool row (pool[slot, plane]) must be contiguous");
  return {static_cast<char*>(t.data_ptr()), h, d, t.stride(0) * es, t.stride(1) * es, t.size(0)};
}

int code_of(at::ScalarType t, const char* what) {
  NEED(t == at::kBFloat16 || t == at::kHalf || t == at::kFloat, "%s must be a bf16, fp16 or fp32 tensor", what);
  return t == at::kBFloat16 ? GSEC_BF16 : t == at::kHalf ? GSEC_F16 : GSEC_F32;
}

// The bytes from a tensor's first element to its last.
struct Span {
  uintptr_t lo, hi;
  explicit Span(const at::Tensor& t) : lo((uintptr_t)t.data_ptr()), hi(lo) {
    if (t.numel() == 0) return;
    int64_t last = 1;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    hi = lo + last * t.element_size();
  }
};

// `out` or a new tensor; not in the memory of what the call reads (or the pool),
// which other blocks may still be reading when a result is written.
at::Tensor output(const Call& c, PyObject* o, at::IntArrayRef shape, at::ScalarType type, const at::Tensor& in,
                  const at::Tensor& pool) {
  if (o == Py_None) return c.empty(shape, type);
  const at::Tensor& t = tensor(o, "out");
  c.flat(t, "out", type);
  no_grad(t, "out");
  for (const at::Tensor* x : {&in, &pool}) {
    const Span a(t), b(*x);
    NEED(a.hi <= b.lo || b.hi <= a.lo, "out overlaps the call's input or the pool");
  }
  NEED(t.sizes() == shape, "out must have as many tokens, heads and values as the queries");
  return t;
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused&) {
  } catch (...) {  // an allocation that failed (torch.OutOfMemoryError), and the like
    torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

bool count_is(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, n);
  return false;
}

// (lens, new, table, free, cursor, page, tokens, base) -> SlotPlan(slots, positions, cu, lens, cursor, table, page)
PyObject* slots_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count_is(n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& lens = tensor(a[0], "lens");
    const Call c(lens, "lens");
    const at::Tensor &fresh = tensor(a[1], "new"), &table = tensor(a[2], "table"), &pages = tensor(a[3], "free"),
                     &cursor = tensor(a[4], "cursor");
    const int64_t batch = lens.numel(), tokens = integer(a[6], "tokens");
    NEED(lens.dim() == 1 && batch < (1ll << 30), "lens must have one dimension");
    auto* lens_at = static_cast<int32_t*>(c.flat(lens, "lens", at::kInt));
    auto* new_at = static_cast<int32_t*>(c.flat(fresh, "new", at::kInt, batch));
    const Table t = table_of(c, table, batch);
    auto* free_at = static_cast<int32_t*>(c.flat(pages, "free", at::kInt));
    auto* cursor_at = static_cast<int32_t*>(c.flat(cursor, "cursor", at::kInt, 1));
    NEED(tokens >= 0 && tokens < (1ll << 31), "tokens must be in [0, 2^31)");
    const int32_t page = small(a[5], "page"), base = small(a[7], "base");
    // the outputs share one allocation: positions and slots on 16-byte boundaries first
    const int64_t slots_from = (tokens * 4 + 15) / 16 * 16, cu_from = slots_from + tokens * 8;
    const int64_t lens_from = cu_from + (batch + 1) * 4, cursor_from = lens_from + batch * 4;
    const at::Tensor all = c.empty({cursor_from + 4}, at::kByte);
    auto* mem = static_cast<char*>(all.data_ptr());
    const auto words = [&](int64_t from) { return reinterpret_cast<int32_t*>(mem + from); };
    finish(gsec_slots_plan(lens_at, new_at, (int32_t)batch, t.at, t.pitch, t.width, free_at, pages.numel(), cursor_at,
                           page, base, reinterpret_cast<int64_t*>(mem + slots_from), words(0), tokens, words(cu_from),
                           words(lens_from), words(cursor_from), c.stream()));
    PyObject* r = PyTuple_New(7);
    if (!r) throw Refused{};
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(piece(all, at::kLong, slots_from, tokens)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(piece(all, at::kInt, 0, tokens)));
    PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(piece(all, at::kInt, cu_from, batch + 1)));
    PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(piece(all, at::kInt, lens_from, batch)));
    PyTuple_SET_ITEM(r, 4, THPVariable_Wrap(piece(all, at::kInt, cursor_from, 1)));
    for (int i = 0; i < 2; ++i) {
      Py_INCREF(a[2 + 3 * i]);  // table, page
      PyTuple_SET_ITEM(r, 5 + i, a[2 + 3 * i]);
    }
    PyObject* args = PyTuple_Pack(1, r);
    Py_DECREF(r);
    if (!args) throw Refused{};
    r = PyTuple_Type.tp_new(g_plan, args, nullptr);
    Py_DECREF(args);
    return r;
  });
}

// (qkv, pool, slots, positions, cos, sin, heads, q_weight, k_weight, eps, interleaved, out) -> q
PyObject* qk_norm_rope_store(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count_is(n, 12)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& qkv = tensor(a[0], "qkv");
    const Call c(qkv, "qkv");
    const at::Tensor &pool = tensor(a[1], "pool"), &slots = tensor(a[2], "slots"), &positions = tensor(a[3], "positions"),
                     &cos = tensor(a[4], "cos"), &sin = tensor(a[5], "sin");
    const at::ScalarType type = qkv.scalar_type();
    const int code = code_of(type, "qkv");
    no_grad(qkv, "qkv");
    no_grad(pool, "pool");
    NEED(qkv.dim() == 2 && (qkv.size(1) <= 1 || qkv.stride(1) == 1), "qkv must be a tensor [tokens, values] with contiguous rows");
    const Pool p = pool_of(c, pool, type);
    const int64_t T = qkv.size(0), values = qkv.size(1);
    const int32_t heads = small(a[6], "heads");
    NEED(heads >= 0 && values == (heads + 2 * p.heads) * p.dim,
         "qkv rows hold %lld values, %d + 2*%lld heads of %lld need %lld", (long long)values, heads, (long long)p.heads,
         (long long)p.dim, (long long)((heads + 2 * p.heads) * p.dim));
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& t = i ? positions : slots;
      const char* what = i ? "positions" : "slots";
      c.on(t, what);
      NEED((t.scalar_type() == at::kInt || t.scalar_type() == at::kLong) && t.is_contiguous(),
           "%s must be a contiguous int32 or int64 tensor", what);
      NEED(t.numel() == T, "%s has %lld entries for %lld tokens", what, (long long)t.numel(), (long long)T);
    }
    auto* cos_at = static_cast<float*>(c.flat(cos, "cos", at::kFloat));
    auto* sin_at = static_cast<float*>(c.flat(sin, "sin", at::kFloat));
    no_grad(cos, "cos");
    no_grad(sin, "sin");
    NEED(cos.dim() == 2 && cos.size(1) < (1 << 20), "cos must have shape [positions, rot / 2]");
    NEED(sin.sizes() == cos.sizes(), "sin must have the shape of cos");
    const void* w[2] = {nullptr, nullptr};
    for (int i = 0; i < 2; ++i) {
      const char* what = i ? "k_weight" : "q_weight";
      if (a[7 + i] == Py_None) continue;
      const at::Tensor& t = tensor(a[7 + i], what);
      no_grad(t, what);
      w[i] = c.flat(t, what, type, p.dim);
    }
    const double eps = real(a[9]);
    const int inter = PyObject_IsTrue(a[10]);
    if (inter < 0) throw Refused{};
    NEED(p.heads < (1 << 20) && p.dim < (1 << 20), "pool heads are too many or too wide");
    at::Tensor out = output(c, a[11], {T, heads, p.dim}, type, qkv, pool);
    const int64_t row = qkv.stride(0) > values ? qkv.stride(0) : values;
    finish(gsec_qk_norm_rope_store(qkv.data_ptr(), row * qkv.element_size(), T, code, heads, (int32_t)p.heads,
                                   (int32_t)p.dim, out.data_ptr(), p.at, p.pitch, p.plane, p.rows, slots.data_ptr(),
                                   (int32_t)slots.element_size(), positions.data_ptr(),
                                   (int32_t)positions.element_size(), cos_at, sin_at, 2 * (int32_t)cos.size(1),
                                   cos.size(0), w[0], w[1], (float)eps, inter, c.stream()));
    return THPVariable_Wrap(std::move(out));
  });
}

// (q, pool, cu, lens, table, page, prefix, prefix_len, scale, out, return_lse) -> o or (o, lse)
PyObject* prefix_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count_is(n, 11)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& q = tensor(a[0], "q");
    const Call c(q, "q");
    const at::Tensor &pool = tensor(a[1], "pool"), &cu = tensor(a[2], "cu"), &lens = tensor(a[3], "lens"),
                     &table = tensor(a[4], "table");
    const at::ScalarType type = q.scalar_type();
    const int code = code_of(type, "q");
    no_grad(q, "q");
    no_grad(pool, "pool");
    NEED(q.dim() == 3 && (q.size(2) <= 1 || q.stride(2) == 1), "q must be a tensor [tokens, heads, dim] with contiguous heads");
    const Pool p = pool_of(c, pool, type);
    const int64_t T = q.size(0), hq = q.size(1), D = q.size(2);
    NEED(p.dim == D && p.heads > 0 && hq % p.heads == 0 && hq < (1 << 20) && D < (1 << 20),
         "pool heads (%lld of %lld) do not serve queries (%lld of %lld)", (long long)p.heads, (long long)p.dim,
         (long long)hq, (long long)D);
    const int64_t batch = lens.numel();
    NEED(batch < (1ll << 30), "lens is too long");
    auto* lens_at = static_cast<int32_t*>(c.flat(lens, "lens", at::kInt));
    auto* cu_at = static_cast<int32_t*>(c.flat(cu, "cu", at::kInt, batch + 1));
    const Table t = table_of(c, table, batch);
    const int32_t page = small(a[5], "page");
    const int64_t prefix_len = integer(a[7], "prefix_len");
    NEED(prefix_len >= 0 && page >= 1, "prefix_len must not be negative, page must be positive");
    const int32_t* prefix_at = nullptr;
    if (prefix_len > 0) {
      NEED(a[6] != Py_None, "prefix_len without prefix pages");
      const at::Tensor& prefix = tensor(a[6], "prefix");
      prefix_at = static_cast<int32_t*>(c.flat(prefix, "prefix", at::kInt));
      NEED(prefix.numel() * page >= prefix_len, "%lld prefix pages of %d hold fewer than %lld keys",
           (long long)prefix.numel(), page, (long long)prefix_len);
    }
    const double scale = a[8] == Py_None ? 1.0 / std::sqrt((double)(D > 0 ? D : 1)) : real(a[8]);
    const int wants_lse = PyObject_IsTrue(a[10]);
    if (wants_lse < 0) throw Refused{};
    at::Tensor out = output(c, a[9], {T, hq, D}, type, q, pool), lse, ws;
    if (wants_lse) lse = c.empty({T, hq}, at::kFloat);
    int64_t bytes = 0;
    if (T > 0)
      finish(gsec_prefix_attention_workspace(T, (int32_t)batch, prefix_len, code, (int32_t)hq, (int32_t)p.heads,
                                             (int32_t)D, &bytes));
    if (bytes > 0) ws = c.empty({bytes}, at::kByte);
    const int64_t es = q.element_size();
    finish(gsec_prefix_attention(q.data_ptr(), q.stride(0) * es, q.stride(1) * es, T, code, (int32_t)hq,
                                 (int32_t)p.heads, (int32_t)D, p.at, p.pitch, p.plane, p.rows, cu_at, lens_at,
                                 (int32_t)batch, t.at, t.pitch, t.width, page, prefix_at, prefix_len, (float)scale,
                                 out.data_ptr(), wants_lse ? static_cast<float*>(lse.data_ptr()) : nullptr,
                                 bytes > 0 ? ws.data_ptr() : nullptr, bytes, c.stream()));
    if (!wants_lse) return THPVariable_Wrap(std::move(out));
    PyObject* r = PyTuple_New(2);
    if (!r) throw Refused{};
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(out)));
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
    return r;
  });
}

// (the function that raises for a return code, the named tuple of a plan)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count_is(n, 2)) return nullptr;
  if (!PyType_Check(a[1]) || !PyType_IsSubtype((PyTypeObject*)a[1], &PyTuple_Type)) {
    PyErr_SetString(PyExc_TypeError, "expected a tuple type");
    return nullptr;
  }
  Py_INCREF(a[0]);
  Py_XSETREF(g_check, a[0]);
  Py_INCREF(a[1]);
  Py_XSETREF(g_plan, (PyTypeObject*)a[1]);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"slots_plan", (PyCFunction)(void (*)())slots_plan, METH_FASTCALL, nullptr},
    {"qk_norm_rope_store", (PyCFunction)(void (*)())qk_norm_rope_store, METH_FASTCALL, nullptr},
    {"prefix_attention", (PyCFunction)(void (*)())prefix_attention, METH_FASTCALL, nullptr},
    {"setup", (PyCFunction)(void (*)())setup, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "gsec_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_gsec_torch(void) { return PyModule_Create(&module); }
