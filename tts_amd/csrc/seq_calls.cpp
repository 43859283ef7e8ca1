// The ordinary call of a sequence operator, from Python to the entry point without the interpreter between: a call of a few
// rows is bound by its host side, and checking, allocating and converting its arguments in Python takes longer than the
// launch.  Every function here either makes the whole call or, where an argument is anything but ordinary (another type,
// device or layout, a host list, an autograd input, a partial overlap), does nothing and returns None: the caller then goes
// through its own checks, which convert or refuse it.  What fails behind those checks is raised here: the call may have been
// queued in part, and is not made again.  The entry points are those of libttsx.so (ttsx_seq.h), bound by address.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/ttsx.h"

namespace {

struct Entries {
  decltype(&ttsx_gated_step) step;
  decltype(&ttsx_gated_scan) scan;
  decltype(&ttsx_gated_scan_backward) scan_backward;
  decltype(&ttsx_gated_scan_workspace) scan_workspace;
  decltype(&ttsx_adapter_add) add;
  decltype(&ttsx_adapter_backward) add_backward;
  decltype(&ttsx_adapter_backward_workspace) add_workspace;
} entry = {};

// An argument as the call sees it: a tensor on the current device, outside autograd, or left out.
struct Arg {
  const at::Tensor* t = nullptr;
  const at::Tensor* operator->() const { return t; }
  const at::Tensor& operator*() const { return *t; }
  explicit operator bool() const { return t != nullptr; }
  template <class T>
  T* data() const {
    return t ? static_cast<T*>(t->data_ptr()) : nullptr;
  }
};

struct Call {
  int device = -1;
  bool ok = true, grad = c10::GradMode::is_enabled(), tangents = c10::AutogradState::get_tls_state().get_fw_grad_mode();
  Call() { ok = entry.step && !c10::impl::dispatch_mode_enabled(); }
  Arg take(PyObject* o, bool optional = false) {
    Arg a;
    if (optional && o == Py_None) return a;
    if (!ok || !THPVariable_CheckExact(o)) {
      ok = false;
      return a;
    }
    const at::Tensor& t = THPVariable_Unpack(o);
    ok = t.is_cuda() && t.layout() == at::kStrided && !t.is_neg() && !(grad && t.requires_grad()) &&
         !(tangents && t._fw_grad(0).defined());
    if (ok && device < 0) device = c10::hip::current_device();
    ok = ok && t.get_device() == device;
    a.t = &t;
    return a;
  }
  void need(bool b) { ok = ok && b; }
  void* stream() const { return c10::hip::getCurrentHIPStream((c10::DeviceIndex)device).stream(); }
};

bool rows_ok(int64_t n) { return n >= 1 && n <= TTSX_SEQ_MAX_ROWS; }
bool width_ok(int64_t n) { return n >= 1 && n <= TTSX_SEQ_MAX_WIDTH; }
int type_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return TTSX_F32;
    case at::kBFloat16: return TTSX_BF16;
    case at::kHalf: return TTSX_F16;
    default: return -1;
  }
}
// The last axis contiguous, rows near enough ([B,T,n]; the batch stride is free, [B,n] has no other, a single row lies anywhere).
bool laid_out(const at::Tensor& t) {
  const int64_t d = t.dim();
  return (t.stride(d - 1) == 1 || t.size(d - 1) == 1) && (d == 2 || t.size(1) == 1 || t.stride(1) <= TTSX_SEQ_MAX_WIDTH);
}
int64_t row_stride(const at::Tensor& t) { return t.dim() == 3 ? t.stride(1) : 0; }
bool state_ok(const Arg& a, int64_t B, int64_t D) {
  return !a || (a->scalar_type() == at::kFloat && a->dim() == 2 && a->size(0) == B && a->size(1) == D && a->is_contiguous());
}
bool index_ok(const Arg& a, int64_t B) {
  return !a || (a->scalar_type() == at::kInt && a->dim() == 1 && a->size(0) == B && a->is_contiguous());
}
bool apart(const at::Tensor& a, const Arg& b) { return !b || !a.is_alias_of(*b); }
at::Tensor fresh(const at::Tensor& like, at::IntArrayRef sizes, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type));
}
struct Scratch {
  at::Tensor t;
  long bytes;
  Scratch(const at::Tensor& like, long n) : bytes(n) {
    if (n > 0) t = fresh(like, {n}, at::kByte);
  }
  void* data() const { return bytes > 0 ? t.data_ptr() : nullptr; }
};

// The results of the entry point `name`, if it returned TTSX_OK.  An argument it refused was refused before any launch.
PyObject* ordinary(int rc, const char* name, std::initializer_list<at::Tensor> out) {
  if (rc == TTSX_ERR_ARG) Py_RETURN_NONE;
  if (rc != TTSX_OK) {
    PyObject* lib = PyImport_ImportModule("tts_amd._lib");
    PyObject* done = lib ? PyObject_CallMethod(lib, "check", "is", rc, name) : nullptr;  // raises
    Py_XDECREF(lib);
    Py_XDECREF(done);
    if (done) PyErr_Format(PyExc_RuntimeError, "%s failed (%d)", name, rc);
    return nullptr;
  }
  if (out.size() == 1) return THPVariable_Wrap(*out.begin());
  PyObject* tuple = PyTuple_New((Py_ssize_t)out.size());
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : out) {
    PyObject* o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(tuple);
      return nullptr;
    }
    PyTuple_SET_ITEM(tuple, i++, o);
  }
  return tuple;
}
template <class F>
int run(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS;
  rc = f();
  Py_END_ALLOW_THREADS;
  return rc;
}

bool counts(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_Format(PyExc_TypeError, "%zd arguments, expected %zd", n, want);
  return n == want;
}

// step(x, g, h, out)
PyObject* step(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts(n, 4)) return nullptr;
  Call c;
  const Arg x = c.take(a[0]), g = c.take(a[1]), h = c.take(a[2]);
  const bool into = a[3] != Py_None;
  c.need(!into || a[3] == a[2]);
  if (!c.ok || x->dim() != 2 || g->sizes() != x->sizes()) Py_RETURN_NONE;
  const int64_t B = x->size(0), D = x->size(1);
  const int type = type_of(*x);
  if (type < 0 || g->scalar_type() != x->scalar_type() || !rows_ok(B) || !width_ok(D) || !state_ok(h, B, D) ||
      !laid_out(*x) || !laid_out(*g) || (into && !(apart(*h, x) && apart(*h, g))))
    Py_RETURN_NONE;
  const at::Tensor y = fresh(*x, {B, D}, x->scalar_type()), next = into ? *h : fresh(*x, {B, D}, at::kFloat);
  void* s = c.stream();
  const int rc = run([&] {
    return entry.step(x->data_ptr(), x->stride(0), g->data_ptr(), g->stride(0), h.data<float>(), (int)B, (int)D, type,
                      y.data_ptr(), static_cast<float*>(next.data_ptr()), s);
  });
  return ordinary(rc, "ttsx_gated_step", {y, next});
  END_HANDLE_TH_ERRORS
}

bool scan_ok(Call& c, const Arg& x, const Arg& g) {
  if (!c.ok || x->dim() != 3 || g->sizes() != x->sizes()) return false;
  const int64_t B = x->size(0), T = x->size(1), D = x->size(2);
  return type_of(*x) >= 0 && g->scalar_type() == x->scalar_type() && rows_ok(B) && rows_ok(T) && width_ok(D) && laid_out(*x) &&
         laid_out(*g);
}

// scan(x, g, h0, lengths, reverse, save_states)
PyObject* scan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts(n, 6)) return nullptr;
  Call c;
  const Arg x = c.take(a[0]), g = c.take(a[1]), h0 = c.take(a[2], true), lengths = c.take(a[3], true);
  const int reverse = PyObject_IsTrue(a[4]), save = PyObject_IsTrue(a[5]);
  if (reverse < 0 || save < 0) return nullptr;
  if (!scan_ok(c, x, g)) Py_RETURN_NONE;
  const int64_t B = x->size(0), T = x->size(1), D = x->size(2);
  if (!state_ok(h0, B, D) || !index_ok(lengths, B)) Py_RETURN_NONE;
  const int type = type_of(*x);
  const Scratch ws(*x, entry.scan_workspace((int)B, (int)T, (int)D, type, 0));
  if (ws.bytes < 0) Py_RETURN_NONE;
  const at::Tensor h = fresh(*x, {B, T, D}, x->scalar_type()), last = fresh(*x, {B, D}, at::kFloat);
  at::Tensor states;
  if (save) states = fresh(*x, {B, (T + TTSX_STATE_BLOCK - 1) / TTSX_STATE_BLOCK, D}, at::kFloat);
  void* s = c.stream();
  const int rc = run([&] {
    return entry.scan(x->data_ptr(), x->stride(0), x->stride(1), g->data_ptr(), g->stride(0), g->stride(1), h0.data<float>(),
                      lengths.data<int32_t>(), (int)B, (int)T, (int)D, type, reverse, h.data_ptr(),
                      static_cast<float*>(last.data_ptr()), save ? static_cast<float*>(states.data_ptr()) : nullptr, ws.data(),
                      (size_t)ws.bytes, s);
  });
  if (save) return ordinary(rc, "ttsx_gated_scan", {h, last, states});
  return ordinary(rc, "ttsx_gated_scan", {h, last});
  END_HANDLE_TH_ERRORS
}

// scan_backward(dh, x, g, states, dh_last, lengths, reverse)
PyObject* scan_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts(n, 7)) return nullptr;
  Call c;
  const Arg dh = c.take(a[0]), x = c.take(a[1]), g = c.take(a[2]), states = c.take(a[3]), dh_last = c.take(a[4], true),
            lengths = c.take(a[5], true);
  const int reverse = PyObject_IsTrue(a[6]);
  if (reverse < 0) return nullptr;
  if (!scan_ok(c, x, g)) Py_RETURN_NONE;
  const int64_t B = x->size(0), T = x->size(1), D = x->size(2);
  if (dh->sizes() != x->sizes() || dh->scalar_type() != x->scalar_type() || !laid_out(*dh) ||
      states->scalar_type() != at::kFloat || !states->is_contiguous() || states->dim() != 3 || states->size(0) != B ||
      states->size(1) != (T + TTSX_STATE_BLOCK - 1) / TTSX_STATE_BLOCK || states->size(2) != D || !state_ok(dh_last, B, D) ||
      !index_ok(lengths, B))
    Py_RETURN_NONE;
  const int type = type_of(*x);
  const Scratch ws(*x, entry.scan_workspace((int)B, (int)T, (int)D, type, 1));
  if (ws.bytes < 0) Py_RETURN_NONE;
  const at::Tensor dx = fresh(*x, {B, T, D}, x->scalar_type()), dg = fresh(*x, {B, T, D}, x->scalar_type()),
                   dh0 = fresh(*x, {B, D}, at::kFloat);
  void* s = c.stream();
  const int rc = run([&] {
    return entry.scan_backward(dh->data_ptr(), dh->stride(0), dh->stride(1), x->data_ptr(), x->stride(0), x->stride(1),
                               g->data_ptr(), g->stride(0), g->stride(1), states.data<float>(), dh_last.data<float>(),
                               lengths.data<int32_t>(), (int)B, (int)T, (int)D, type, reverse, dx.data_ptr(), dg.data_ptr(),
                               static_cast<float*>(dh0.data_ptr()), ws.data(), (size_t)ws.bytes, s);
  });
  return ordinary(rc, "ttsx_gated_scan_backward", {dx, dg, dh0});
  END_HANDLE_TH_ERRORS
}

struct Sizes {
  int64_t B, T, K, N, R, V;
};
// Shapes and types of an adapter's call; `wide` is y or dy.
bool adapter_ok(Call& c, const Arg& wide, const Arg& x, const Arg& down, const Arg& up, const Arg& voices, const Arg& scale,
                const Arg& lengths, Sizes& z) {
  if (!c.ok) return false;
  const int64_t d = wide->dim();
  if ((d != 2 && d != 3) || x->dim() != d || down->dim() != 3 || up->dim() != 3) return false;
  z = {wide->size(0), d == 3 ? wide->size(1) : 1, x->size(d - 1), wide->size(d - 1), down->size(1), down->size(0)};
  const at::ScalarType type = x->scalar_type();
  return x->size(0) == z.B && (d == 2 || x->size(1) == z.T) && up->size(0) == z.V && up->size(1) == z.R && down->size(2) == z.K &&
         up->size(2) == z.N && rows_ok(z.B) && rows_ok(z.T) && width_ok(z.K) && width_ok(z.N) && z.R >= 1 &&
         z.R <= TTSX_ADAPTER_MAX_RANK && z.V >= 1 && z.V <= TTSX_SEQ_MAX_VOICES &&
         type_of(*x) >= 0 && wide->scalar_type() == type && down->scalar_type() == type && up->scalar_type() == type &&
         down->is_contiguous() && up->is_contiguous() && laid_out(*x) && laid_out(*wide) && index_ok(voices, z.B) &&
         index_ok(lengths, z.B) &&
         (!scale || (scale->scalar_type() == at::kFloat && scale->dim() == 1 && scale->size(0) == z.V && scale->is_contiguous()));
}

// adapter_add(y, x, down, up, voices, scale, lengths, out)
PyObject* adapter_add(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts(n, 8)) return nullptr;
  Call c;
  const Arg y = c.take(a[0]), x = c.take(a[1]), down = c.take(a[2]), up = c.take(a[3]), voices = c.take(a[4]),
            scale = c.take(a[5], true), lengths = c.take(a[6], true);
  const bool into = a[7] != Py_None;
  c.need(!into || a[7] == a[0]);
  Sizes z;
  if (!adapter_ok(c, y, x, down, up, voices, scale, lengths, z)) Py_RETURN_NONE;
  if (into && !(y->is_contiguous() && apart(*y, x) && apart(*y, down) && apart(*y, up) && apart(*y, scale) && apart(*y, voices) &&
                apart(*y, lengths)))
    Py_RETURN_NONE;
  const at::Tensor out = into ? *y : fresh(*y, y->sizes(), y->scalar_type());
  const int type = type_of(*x);
  void* s = c.stream();
  const int rc = run([&] {
    return entry.add(y->data_ptr(), y->stride(0), row_stride(*y), x->data_ptr(), x->stride(0), row_stride(*x), down->data_ptr(),
                     up->data_ptr(), voices.data<int32_t>(), scale.data<float>(), lengths.data<int32_t>(), (int)z.B, (int)z.T,
                     (int)z.K, (int)z.N, (int)z.R, (int)z.V, type, out.data_ptr(), out.stride(0), row_stride(out), s);
  });
  return ordinary(rc, "ttsx_adapter_add", {out});
  END_HANDLE_TH_ERRORS
}

// adapter_backward(dy, x, down, up, voices, scale, lengths)
PyObject* adapter_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!counts(n, 7)) return nullptr;
  Call c;
  const Arg dy = c.take(a[0]), x = c.take(a[1]), down = c.take(a[2]), up = c.take(a[3]), voices = c.take(a[4]),
            scale = c.take(a[5], true), lengths = c.take(a[6], true);
  Sizes z;
  if (!adapter_ok(c, dy, x, down, up, voices, scale, lengths, z)) Py_RETURN_NONE;
  const int type = type_of(*x);
  const Scratch ws(*x, entry.add_workspace((int)z.B, (int)z.T, (int)z.K, (int)z.N, (int)z.R, type));
  if (ws.bytes <= 0) Py_RETURN_NONE;
  const at::Tensor dx = fresh(*x, x->sizes(), x->scalar_type()), ddown = fresh(*x, down->sizes(), x->scalar_type()),
                   dup = fresh(*x, up->sizes(), x->scalar_type());
  void* s = c.stream();
  const int rc = run([&] {
    return entry.add_backward(dy->data_ptr(), dy->stride(0), row_stride(*dy), x->data_ptr(), x->stride(0), row_stride(*x),
                              down->data_ptr(), up->data_ptr(), voices.data<int32_t>(), scale.data<float>(),
                              lengths.data<int32_t>(), (int)z.B, (int)z.T, (int)z.K, (int)z.N, (int)z.R, (int)z.V, type,
                              dx.data_ptr(), ddown.data_ptr(), dup.data_ptr(), ws.data(), (size_t)ws.bytes, s);
  });
  return ordinary(rc, "ttsx_adapter_backward", {dx, ddown, dup});
  END_HANDLE_TH_ERRORS
}

// bind(addresses of the entry points in the order of Entries)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counts(n, 7)) return nullptr;
  void* p[7];
  for (int i = 0; i < 7; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
  }
  entry = {reinterpret_cast<decltype(entry.step)>(p[0]),          reinterpret_cast<decltype(entry.scan)>(p[1]),
           reinterpret_cast<decltype(entry.scan_backward)>(p[2]), reinterpret_cast<decltype(entry.scan_workspace)>(p[3]),
           reinterpret_cast<decltype(entry.add)>(p[4]),           reinterpret_cast<decltype(entry.add_backward)>(p[5]),
           reinterpret_cast<decltype(entry.add_workspace)>(p[6])};
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(F)), METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<bind>("bind"),
                         method<step>("step"),
                         method<scan>("scan"),
                         method<scan_backward>("scan_backward"),
                         method<adapter_add>("adapter_add"),
                         method<adapter_backward>("adapter_backward"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_seqcalls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__seqcalls() { return PyModule_Create(&module); }
