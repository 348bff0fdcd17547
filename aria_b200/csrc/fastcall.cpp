// fastcall.cpp -- the short way from Python to the entry points of the paged cache and
// of the logits (module aria_b200._fastcall).
//
// One token's kernels run for 5 to 10 microseconds; checking a dozen tensors and
// converting two dozen arguments through ctypes takes the host as long again.  Here the
// checks of aria_b200/paged.py and logits.py are made in C++ and the C ABI is called
// directly (attention of one sequence: 4.8 us of host time per call instead of 11.9,
// most of it the launch and the lse's allocation; logits of one row: 6.5 instead of 16).
// A function returns None when anything is unusual and nothing was launched -- an argument
// that does not pass, a workspace that has to grow, a call that the library refuses -- and
// the Python code then goes the long way, which says what is wrong.  A CUDA error raises
// here: one of a call's kernels may have run, and sums, moves and stored rows are not to
// be made twice.  No arithmetic happens here, and of CUDA only the current device is asked:
// a launch goes there, so tensors of another one take the long way, which changes it.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>

#include <exception>

#include "../../include/aria_q4.h"

namespace {

decltype(&aria_attention_paged) f_attention = nullptr;
decltype(&aria_prompt_weights) f_prompt = nullptr;
decltype(&aria_cache_evict) f_evict = nullptr;
decltype(&aria_logits_adjust) f_logits = nullptr;

PyObject* check = nullptr;  // _lib.check(name, status): raises what the status means

thread_local bool launched = false;  // the library was called, and did not refuse

// Whether the library refused the call, so that the long way may make it again.  `failed`:
// it did not, and an exception is set.
bool refused(const char* name, int status, bool& failed) {
  failed = false;
  if (status == ARIA_Q4_OK) return false;
  if (status != ARIA_Q4_ECUDA) {
    launched = false;
    return true;
  }
  failed = true;
  PyObject* r = PyObject_CallFunction(check, "si", name, status);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, name);
  return false;
}

bool elsewhere(int dev) { return c10::cuda::current_device() != dev; }

struct Args {
  PyObject* const* a;
  int at = 0;
  PyObject* next() { return a[at++]; }
  long long integer() { return PyLong_AsLongLong(next()); }
  void* pointer() { return PyLong_AsVoidPtr(next()); }
  bool truth() { return PyObject_IsTrue(next()) > 0; }
  double real() { return PyFloat_AsDouble(next()); }
  // a tensor (null for None); `bad` is set for anything else
  const at::Tensor* tensor(bool& bad) {
    PyObject* o = next();
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) {
      bad = true;
      return nullptr;
    }
    return &THPVariable_Unpack(o);
  }
};

bool on(const at::Tensor& t, at::ScalarType type, int dev) {
  return t.is_cuda() && t.get_device() == dev && t.scalar_type() == type;
}
// contiguous [n0](n1)(n2) of this type
bool flat(const at::Tensor* t, at::ScalarType type, int dev, int64_t n0, int64_t n1 = -1, int64_t n2 = -1) {
  if (!on(*t, type, dev) || !t->is_contiguous()) return false;
  const int dims = n2 >= 0 ? 3 : n1 >= 0 ? 2 : 1;
  return t->dim() == dims && t->size(0) == n0 && (n1 < 0 || t->size(1) == n1) && (n2 < 0 || t->size(2) == n2);
}
// [M][heads][dh] with contiguous rows; its strides (those of one entry are not used)
bool rows(const at::Tensor& t, at::ScalarType type, int dev, int64_t M, int64_t heads, int64_t dh, long long& row,
          long long& head) {
  if (!on(t, type, dev) || t.dim() != 3 || t.size(0) != M || t.size(1) != heads || t.size(2) != dh ||
      t.stride(2) != 1)
    return false;
  row = M > 1 ? t.stride(0) : 8;
  head = heads > 1 ? t.stride(1) : 8;
  return true;
}
// [M][...] with contiguous rows; its row stride, or -1
long long matrix(const at::Tensor& t, at::ScalarType type, int dev, int64_t M) {
  if (!on(t, type, dev) || t.dim() != 2 || t.size(0) != M || (t.stride(1) != 1 && t.size(1) > 1)) return -1;
  return M > 1 ? t.stride(0) : t.size(1);
}
template <class T>
T* ptr(const at::Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}

int type_code(at::ScalarType t) {
  return t == at::kFloat ? ARIA_Q4_F32 : t == at::kHalf ? ARIA_Q4_F16 : t == at::kBFloat16 ? ARIA_Q4_BF16 : -1;
}

// kv, M, kv_heads, head_dim, device, scale, workspace, bytes, stream, want_lse, q, k_new,
// v_new, out, weights, weights_out, slot_pos, positions
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 18) Py_RETURN_NONE;
  Args a{args};
  const auto* kv = static_cast<const aria_paged_kv*>(a.pointer());
  const int M = (int)a.integer(), kvh = (int)a.integer(), dh = (int)a.integer(), dev = (int)a.integer();
  const float scale = (float)a.real();
  void* ws = a.pointer();
  const size_t ws_bytes = (size_t)a.integer();
  void* stream = a.pointer();
  const bool want_lse = a.truth();
  bool bad = false;
  PyObject* out_obj = args[13];
  const at::Tensor *q = a.tensor(bad), *kn = a.tensor(bad), *vn = a.tensor(bad), *out = a.tensor(bad),
                   *w = a.tensor(bad), *wo = a.tensor(bad), *sp = a.tensor(bad), *pos = a.tensor(bad);
  if (PyErr_Occurred()) return nullptr;
  if (bad || !q || q->dim() != 3 || !kn != !vn || elsewhere(dev)) Py_RETURN_NONE;
  const at::ScalarType type = kv->dtype == ARIA_Q4_BF16 ? at::kBFloat16 : at::kHalf;
  const int64_t heads = q->size(1);
  long long qr, qh, nr = 0, nh = 0, vr = 0, vh = 0, orow, oh;
  if (heads <= 0 || heads % kvh || !rows(*q, type, dev, M, heads, dh, qr, qh)) Py_RETURN_NONE;
  if (kn && (!rows(*kn, type, dev, M, kvh, dh, nr, nh) || !rows(*vn, type, dev, M, kvh, dh, vr, vh) || nr != vr ||
             nh != vh))
    Py_RETURN_NONE;
  int64_t cap = 0;
  if (w) {
    if (w->dim() != 3) Py_RETURN_NONE;
    cap = w->size(2);
    if (!flat(w, at::kFloat, dev, M, kvh, cap) || (wo && !flat(wo, at::kFloat, dev, M, kvh, cap))) Py_RETURN_NONE;
    if (sp && (!pos || !kn || !flat(sp, at::kInt, dev, M, kvh, cap) || !flat(pos, at::kInt, dev, M))) Py_RETURN_NONE;
  } else if (wo || sp) {
    Py_RETURN_NONE;
  }
  at::Tensor made, lse;
  if (!out) {
    made = at::empty({M, heads, dh}, q->options());
    out = &made;
  }
  if (!rows(*out, type, dev, M, heads, dh, orow, oh)) Py_RETURN_NONE;
  if (want_lse) lse = at::empty({M, heads}, q->options().dtype(at::kFloat));
  launched = true;
  const int status = f_attention(
      kv, M, (int)heads, ptr<const uint16_t>(q), qr, qh, ptr<const uint16_t>(kn), ptr<const uint16_t>(vn), nr, nh, scale,
      ptr<uint16_t>(out), orow, oh, want_lse ? ptr<float>(&lse) : nullptr, ptr<const float>(w),
      wo ? ptr<float>(wo) : ptr<float>(w), cap, ptr<int>(sp), sp ? ptr<const int>(pos) : nullptr, ws, ws_bytes, stream);
  bool failed;
  if (refused("aria_attention_paged", status, failed)) Py_RETURN_NONE;
  if (failed) return nullptr;
  PyObject* r = PyTuple_New(2);
  if (!r) return nullptr;
  if (made.defined()) {
    PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(made)));
  } else {
    Py_INCREF(out_obj);
    PyTuple_SET_ITEM(r, 0, out_obj);
  }
  if (want_lse) {
    PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(lse)));
  } else {
    Py_INCREF(Py_None);
    PyTuple_SET_ITEM(r, 1, Py_None);
  }
  return r;
}

// q, k, lse, out, scale, first_query, workspace, bytes, stream
PyObject* prompt(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) Py_RETURN_NONE;
  Args a{args};
  bool bad = false;
  const at::Tensor *q = a.tensor(bad), *k = a.tensor(bad), *lse = a.tensor(bad), *out = a.tensor(bad);
  const float scale = (float)a.real();
  const long long first = a.integer();
  void* ws = a.pointer();
  const size_t ws_bytes = (size_t)a.integer();
  void* stream = a.pointer();
  if (PyErr_Occurred()) return nullptr;
  if (bad || !q || !k || !lse || !out || !q->is_cuda() || q->dim() != 4 || k->dim() != 4 || out->dim() != 3 ||
      first < 0 || first > 0x7fffffff)
    Py_RETURN_NONE;
  const int dev = q->get_device();
  if (elsewhere(dev)) Py_RETURN_NONE;
  const at::ScalarType type = q->scalar_type();
  const int64_t B = q->size(0), T = q->size(1), heads = q->size(2), dh = q->size(3), kvh = k->size(2);
  if ((type != at::kHalf && type != at::kBFloat16) || !on(*k, type, dev) || k->size(0) != B || k->size(1) != T ||
      k->size(3) != dh || kvh == 0 || heads % kvh || q->stride(3) != 1 || k->stride(3) != 1 || B == 0 || T == 0)
    Py_RETURN_NONE;
  if (!flat(lse, at::kFloat, dev, B, heads, T) || !on(*out, at::kFloat, dev) || out->size(0) != B ||
      out->size(1) != kvh || out->size(2) < T || (out->stride(2) != 1 && out->size(2) > 1))
    Py_RETURN_NONE;
  auto st = [](const at::Tensor* t, int d) { return t->size(d) > 1 ? (long long)t->stride(d) : 8LL; };
  launched = true;
  const int status =
      f_prompt(ptr<const uint16_t>(q), st(q, 0), st(q, 1), st(q, 2), ptr<const uint16_t>(k), st(k, 0), st(k, 1), st(k, 2),
               type_code(type), (int)B, (int)T, (int)heads, (int)kvh, (int)dh, ptr<const float>(lse), scale, (int)first,
               ptr<float>(out), out->stride(0), out->stride(1), ws, ws_bytes, stream);
  bool failed;
  if (refused("aria_prompt_weights", status, failed)) Py_RETURN_NONE;
  if (failed) return nullptr;
  Py_RETURN_TRUE;
}

// kv, M, kv_heads, device, lens' address, keep, recent, sinks, workspace, bytes, stream,
// weights, slot_pos, next_pos, weights_out, slot_pos_out, lens_out
PyObject* evict(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 17) Py_RETURN_NONE;
  Args a{args};
  const auto* kv = static_cast<const aria_paged_kv*>(a.pointer());
  const int M = (int)a.integer(), kvh = (int)a.integer(), dev = (int)a.integer();
  const void* lens = a.pointer();
  const long long keep = a.integer(), recent = a.integer(), sinks = a.integer();
  void* ws = a.pointer();
  const size_t ws_bytes = (size_t)a.integer();
  void* stream = a.pointer();
  bool bad = false;
  const at::Tensor *w = a.tensor(bad), *p = a.tensor(bad), *next = a.tensor(bad), *wo = a.tensor(bad),
                   *po = a.tensor(bad), *lo = a.tensor(bad);
  if (PyErr_Occurred()) return nullptr;
  const long long most = 0x7fffffff;
  if (bad || !w || !p || !next || !lo || w->dim() != 3 || keep > most || recent > most || sinks > most || keep <= 0 ||
      recent < 0 || sinks < 0 || elsewhere(dev))
    Py_RETURN_NONE;
  const int64_t cap = w->size(2);
  if (!flat(w, at::kFloat, dev, M, kvh, cap) || !flat(p, at::kInt, dev, M, kvh, cap) || !flat(next, at::kInt, dev, M) ||
      !flat(lo, at::kInt, dev, M) || lo->data_ptr() == lens || (wo && !flat(wo, at::kFloat, dev, M, kvh, cap)) ||
      (po && !flat(po, at::kInt, dev, M, kvh, cap)))
    Py_RETURN_NONE;
  launched = true;
  const int status = f_evict(kv, M, ptr<const float>(w), wo ? ptr<float>(wo) : ptr<float>(w), ptr<const int>(p),
                             po ? ptr<int>(po) : ptr<int>(p), cap, ptr<const int>(next), (int)keep, (int)recent,
                             (int)sinks, ptr<int>(lo), ws, ws_bytes, stream);
  bool failed;
  if (refused("aria_cache_evict", status, failed)) Py_RETURN_NONE;
  if (failed) return nullptr;
  Py_RETURN_TRUE;
}

// workspace, bytes, stream, want_token, logits, out, history, history_lens, prompt_lens,
// repetition, frequency, presence, bias_tokens, bias_values, allowed, token
PyObject* logits(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 16) Py_RETURN_NONE;
  Args a{args};
  void* ws = a.pointer();
  const size_t ws_bytes = (size_t)a.integer();
  void* stream = a.pointer();
  const bool want = a.truth();
  bool bad = false;
  PyObject *out_obj = args[5], *token_obj = args[15];
  const at::Tensor *x = a.tensor(bad), *out = a.tensor(bad), *hist = a.tensor(bad), *hl = a.tensor(bad),
                   *pl = a.tensor(bad), *rep = a.tensor(bad), *freq = a.tensor(bad), *pres = a.tensor(bad),
                   *bt = a.tensor(bad), *bv = a.tensor(bad), *ok = a.tensor(bad), *token = a.tensor(bad);
  if (PyErr_Occurred()) return nullptr;
  if (bad || !x || !x->is_cuda() || x->dim() != 2) Py_RETURN_NONE;
  const int dev = x->get_device(), type = type_code(x->scalar_type());
  const int64_t M = x->size(0), V = x->size(1);
  if (elsewhere(dev) || type < 0 || M == 0 || M > 65535 || V <= 0 || V > 0x7fffffff) Py_RETURN_NONE;
  const long long x_row = matrix(*x, x->scalar_type(), dev, M);
  if (x_row < 0) Py_RETURN_NONE;
  aria_logit_rules r = {};
  if (hist) {
    r.history_row = matrix(*hist, at::kInt, dev, M);
    if (r.history_row < 0 || !hl || !flat(hl, at::kInt, dev, M) || (pl && !flat(pl, at::kInt, dev, M)) ||
        hist->size(1) > 0x7fffffff)
      Py_RETURN_NONE;
    r.history = ptr<const int>(hist);
    r.history_cap = (int)hist->size(1);
    r.history_lens = ptr<const int>(hl);
    r.prompt_lens = ptr<const int>(pl);
  } else if (rep || freq || pres) {
    Py_RETURN_NONE;
  }
  const at::Tensor* params[3] = {rep, freq, pres};
  for (const at::Tensor* p : params)
    if (p && !flat(p, at::kFloat, dev, M)) Py_RETURN_NONE;
  r.repetition = ptr<const float>(rep);
  r.frequency = ptr<const float>(freq);
  r.presence = ptr<const float>(pres);
  if (!bt != !bv) Py_RETURN_NONE;
  if (bt) {
    r.bias_row = matrix(*bt, at::kInt, dev, M);
    if (r.bias_row < 0 || matrix(*bv, at::kFloat, dev, M) != r.bias_row || bt->size(1) != bv->size(1) ||
        bt->size(1) > 0x7fffffff)
      Py_RETURN_NONE;
    r.biases = (int)bt->size(1);
    if (r.biases > 0) {
      r.bias_tokens = ptr<const int>(bt);
      r.bias_values = ptr<const float>(bv);
    }
  }
  if (ok) {
    if (ok->dim() != 2 || (ok->size(0) != 1 && ok->size(0) != M) || ok->size(1) != (V + 31) / 32) Py_RETURN_NONE;
    r.allowed_row = matrix(*ok, at::kInt, dev, ok->size(0));
    if (r.allowed_row < 0) Py_RETURN_NONE;
    if (ok->size(0) != M) r.allowed_row = 0;  // one row for all
    r.allowed = ptr<const uint32_t>(ok);
  }
  at::Tensor made, made_token;
  if (!out) {
    made = at::empty({M, V}, x->options());
    out = &made;
  }
  const int out_type = type_code(out->scalar_type());
  if ((out_type != type && out_type != ARIA_Q4_F32) || out->dim() != 2 || out->size(1) != V) Py_RETURN_NONE;
  const long long y_row = matrix(*out, out->scalar_type(), dev, M);
  if (y_row < 0) Py_RETURN_NONE;
  if (token) {
    if (!flat(token, at::kInt, dev, M)) Py_RETURN_NONE;
  } else if (want) {
    made_token = at::empty({M}, x->options().dtype(at::kInt));
    token = &made_token;
  }
  launched = true;
  const int status = f_logits(&r, x->data_ptr(), type, x_row, (int)M, (int)V, out->data_ptr(), out_type, y_row,
                              ptr<int>(token), ws, ws_bytes, stream);
  bool failed;
  if (refused("aria_logits_adjust", status, failed)) Py_RETURN_NONE;
  if (failed) return nullptr;
  PyObject* res = PyTuple_New(2);
  if (!res) return nullptr;
  if (made.defined()) {
    PyTuple_SET_ITEM(res, 0, THPVariable_Wrap(std::move(made)));
  } else {
    Py_INCREF(out_obj);
    PyTuple_SET_ITEM(res, 0, out_obj);
  }
  if (made_token.defined()) {
    PyTuple_SET_ITEM(res, 1, THPVariable_Wrap(std::move(made_token)));
  } else {
    Py_INCREF(token_obj);
    PyTuple_SET_ITEM(res, 1, token_obj);
  }
  return res;
}

// no C++ exception leaves a C entry: before a launch the long way meets the same trouble and
// says so, after one it raises
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  launched = false;
  try {
    return F(self, args, n);
  } catch (const std::exception& e) {
    PyErr_Clear();
    if (!launched) Py_RETURN_NONE;
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_Clear();
    if (!launched) Py_RETURN_NONE;
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

// the four entry points' addresses, and what raises the meaning of a status
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "bind takes four addresses and a function");
    return nullptr;
  }
  f_attention = reinterpret_cast<decltype(f_attention)>(PyLong_AsVoidPtr(args[0]));
  f_prompt = reinterpret_cast<decltype(f_prompt)>(PyLong_AsVoidPtr(args[1]));
  f_evict = reinterpret_cast<decltype(f_evict)>(PyLong_AsVoidPtr(args[2]));
  f_logits = reinterpret_cast<decltype(f_logits)>(PyLong_AsVoidPtr(args[3]));
  if (PyErr_Occurred()) return nullptr;
  Py_XDECREF(check);
  check = Py_NewRef(args[4]);
  Py_RETURN_NONE;
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"bind", FAST(bind), nullptr},
                         {"attention", FAST(guarded<attention>), nullptr},
                         {"prompt", FAST(guarded<prompt>), nullptr},
                         {"evict", FAST(guarded<evict>), nullptr},
                         {"logits", FAST(guarded<logits>), nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__fastcall(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "key", FASTCALL_KEY) < 0) {  // the Python and the torch that it is for
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
