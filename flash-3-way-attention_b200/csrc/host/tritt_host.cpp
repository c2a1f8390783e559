// The host side of a call from Python: checks, outputs, workspace and the library's entry point in one native call.
//
// What bounds a call of a short sequence is the time to enqueue it: a forward of 8 heads of 64 rows took 32.5 us, its kernels 15.5.  The
// interpreter's checks of the tensors' attributes, its three allocations and the conversion of 26 arguments by ctypes took 15 of them.
// With this code 17.4 us; a training step of 2 heads of 64 rows fp32 158 -> 110 us, of which 79 are autograd's own, of the dot-product-sum
// of 16 heads of 1024 rows 172 -> 125.  These functions take the calls that need no help: five or eight contiguous, 16-byte aligned CUDA tensors of one
// shape, type and device, which is the current one.  For any other call they return None and change nothing: the Python code then
// copies, converts, switches devices or raises, as its own checks say.
//
// An extension module rather than a dispatcher operator: the autograd functions, their hooks and saved tensors stay where they are.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <array>
#include <algorithm>
#include <climits>
#include <cstring>
#include <map>

#include "tritt.h"

namespace {

enum { kTdpFwd = TRITT_OP_TDP_FWD, kTdpBwd = TRITT_OP_TDP_BWD, kDpsFwd = TRITT_OP_DPS_FWD, kDpsBwd = TRITT_OP_DPS_BWD };
constexpr int kDevices = 64;
constexpr int kNotPlain = INT_MIN;   // no code of the library's

// Everything below is read and written with the interpreter's lock held.
struct Entries {   // (the addresses come from Python, which has loaded the library)
  decltype(&tritt_tdp_fwd) tdp_fwd;
  decltype(&tritt_tdp_bwd) tdp_bwd;
  decltype(&tritt_dps_fwd) dps_fwd;
  decltype(&tritt_dps_bwd) dps_bwd;
  decltype(&tritt_dps_bwd_saved) dps_bwd_saved;
  decltype(&tritt_workspace_bytes_flags) workspace_bytes;
  decltype(&tritt_tdp_fwd_workspace) tdp_fwd_workspace;
  decltype(&tritt_qk_norm_rotary_fwd) norm_fwd;
  decltype(&tritt_qk_norm_rotary_bwd) norm_bwd;
  decltype(&tritt_qk_norm_rotary_workspace) norm_workspace;
  decltype(&tritt_cache_write) cache_write;
  decltype(&tritt_cache_read) cache_read;
  decltype(&tritt_tdp_decode) tdp_decode;
  decltype(&tritt_dps_append) dps_append;
  decltype(&tritt_dps_decode) dps_decode;
  decltype(&tritt_decode_workspace) decode_workspace;
} lib{};
volatile int* status_words[kDevices] = {};
std::map<std::array<int, 12>, size_t> workspace_sizes;

// The call's tensors have one shape [B, N, T, D], type and device.
struct Shape {
  int B, N, T, D, dtype, device;
  at::ScalarType type;
};

bool usable(const at::Tensor& t) {
  return t.defined() && !t.unsafeGetTensorImpl()->is_python_dispatch() && t.layout() == at::kStrided && t.is_cuda() && t.has_storage() &&
         t.is_contiguous() && !t.is_neg() && t.numel() > 0;
}
bool aligned(const void* p) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool read_shape(const at::Tensor& q, Shape& s) {
  if (!usable(q) || q.dim() != 4) return false;
  s.type = q.scalar_type();
  s.dtype = s.type == at::kFloat ? TRITT_F32 : s.type == at::kHalf ? TRITT_F16 : s.type == at::kBFloat16 ? TRITT_BF16 : -1;
  for (int i = 0; i < 4; ++i)
    if (q.size(i) > INT_MAX) return false;
  s.B = (int)q.size(0);
  s.N = (int)q.size(1);
  s.T = (int)q.size(2);
  s.D = (int)q.size(3);
  s.device = q.device().index();
  return s.dtype >= 0 && (s.D & (s.D - 1)) == 0 && s.device >= 0 && s.device < kDevices && s.device == c10::cuda::current_device();
}

// (not a subclass: what is allocated like one of those is of its type)
bool is_tensor(PyObject* o) { return (PyObject*)Py_TYPE(o) == THPVariableClass; }

// Address of a tensor of the call's shape; null: not one.
void* operand(PyObject* o, const Shape& s) {
  if (!is_tensor(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!usable(t) || t.dim() != 4 || t.size(0) != s.B || t.size(1) != s.N || t.size(2) != s.T || t.size(3) != s.D ||
      t.scalar_type() != s.type || t.device().index() != s.device)
    return nullptr;
  void* p = t.data_ptr();
  return aligned(p) ? p : nullptr;
}

bool read_int(PyObject* o, int none, int& v) {
  if (o == Py_None) {
    v = none;
    return none >= 0;
  }
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  const long x = PyLong_AsLongAndOverflow(o, &overflow);
  if (overflow || x > INT_MAX || x < INT_MIN) return false;
  v = (int)x;
  return true;
}
bool read_float(PyObject* o, float& v) {
  if (!PyFloat_CheckExact(o)) return false;
  v = (float)PyFloat_AS_DOUBLE(o);
  return true;
}

// The scalars of a call, from argument i on: scale, causal, flags, windows (four, or the one of the dot-product-sum).
struct Scalars {
  float scale;
  int causal, flags, w[4];
  int* status;
};
bool read_scalars(PyObject* const* a, int op, const Shape& s, Scalars& c) {
  if (!read_float(a[0], c.scale) || !PyBool_Check(a[1]) || !read_int(a[2], -1, c.flags)) return false;
  c.causal = a[1] == Py_True;
  const int windows = op < kDpsFwd ? 4 : 1;
  for (int i = 0; i < windows; ++i)
    if (!read_int(a[3 + i], op < kDpsFwd ? s.T : -1, c.w[i])) return false;
  // (a kernel of an earlier call gave up, or the word is not there yet: Python reports, or makes it)
  c.status = const_cast<int*>(status_words[s.device]);
  return lib.tdp_fwd != nullptr && c.status != nullptr && *status_words[s.device] == 0;
}

size_t workspace_size(int op, const Shape& s, const Scalars& c) {
  std::array<int, 12> key = {op, s.B, s.N, s.T, s.D, s.dtype, op < kDpsFwd ? c.flags : 0, 0, 0, 0, 0, 0};
  if (op == kTdpFwd) {   // (what the forward makes use of depends on the mask)
    key[7] = c.causal;
    for (int i = 0; i < 4; ++i) key[8 + i] = c.w[i];
  }
  const auto it = workspace_sizes.find(key);
  if (it != workspace_sizes.end()) return it->second;
  if (workspace_sizes.size() >= 1024) workspace_sizes.clear();
  const size_t n = op == kTdpFwd ? lib.tdp_fwd_workspace(s.B, s.N, s.T, s.D, s.dtype, c.causal, c.w[0], c.w[1], c.w[2], c.w[3], 1, c.flags)
                                 : lib.workspace_bytes(op, s.B, s.N, s.T, s.D, s.dtype, key[6]);
  return workspace_sizes[key] = n < 256 ? 256 : n;
}

// The interpreter's lock is not held while device memory is allocated (which may wait for the device) and kernels are launched.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// An output's address; null: something stands in for plain tensors (a mode), Python's own calls shall meet it
void* fresh(const at::Tensor& t) {
  if (!usable(t)) return nullptr;
  void* p = t.data_ptr();
  return aligned(p) ? p : nullptr;
}

PyObject* wrap_all(at::Tensor* t, int n) {
  PyObject* r = PyTuple_New(n);
  if (!r) return nullptr;
  for (int i = 0; i < n; ++i) {
    PyObject* o = THPVariable_Wrap(t[i]);   // (None for one that is not there)
    if (!o) {
      Py_DECREF(r);
      return nullptr;
    }
    PyTuple_SET_ITEM(r, i, o);
  }
  return r;
}

// forward(op, q, k1, k2, v1, v2, scale, causal, flags, windows...) -> (o, log-sum-exp, workspace), the library's error code, or None
PyObject* forward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int op;
  if (n < 10 || !read_int(a[0], -1, op) || n != (op < kDpsFwd ? 13 : 10) || !is_tensor(a[1])) Py_RETURN_NONE;
  Shape s;
  Scalars c;
  const at::Tensor& q = THPVariable_Unpack(a[1]);
  if (!read_shape(q, s) || !read_scalars(a + 6, op, s, c)) Py_RETURN_NONE;
  void* in[5];
  for (int i = 0; i < 5; ++i)
    if (!(in[i] = operand(a[1 + i], s))) Py_RETURN_NONE;
  const size_t bytes = workspace_size(op, s, c);
  at::Tensor out[3];
  int rc;
  {
    Unlocked unlocked;
    out[0] = at::empty_like(q);
    out[1] = at::empty({s.B, s.N, s.T}, q.options().dtype(at::kFloat));
    out[2] = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    void *const o = fresh(out[0]), *const l = fresh(out[1]), *const w = fresh(out[2]);
    void* const stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)s.device).stream();
    if (!o || !l || !w)
      rc = kNotPlain;
    else if (op == kTdpFwd)
      rc = lib.tdp_fwd(in[0], in[1], in[2], in[3], in[4], o, (float*)l, s.B, s.N, s.T, s.D, s.dtype, c.scale, c.causal, c.w[0], c.w[1],
                       c.w[2], c.w[3], 1, 0, w, bytes, c.status, c.flags, stream);
    else
      rc = lib.dps_fwd(in[0], in[1], in[2], in[3], in[4], o, (float*)l, s.B, s.N, s.T, s.D, s.dtype, c.scale, c.causal, c.w[0], w, bytes,
                       c.status, c.flags, stream);
  }
  if (rc == kNotPlain) Py_RETURN_NONE;
  if (rc != 0) return PyLong_FromLong(rc);
  return wrap_all(out, op == kTdpFwd ? 2 : 3);
  END_HANDLE_TH_ERRORS
}

// backward(op, q, k1, k2, v1, v2, o, do, log-sum-exp, scale, causal, flags, windows..., the forward's workspace or None)
// -> the five gradients, the library's error code, or None
PyObject* backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int op;
  if (n < 14 || !read_int(a[0], -1, op) || n != (op < kDpsFwd ? 17 : 14) || !is_tensor(a[1]) || !is_tensor(a[8]))
    Py_RETURN_NONE;
  Shape s;
  Scalars c;
  const at::Tensor& q = THPVariable_Unpack(a[1]);
  if (!read_shape(q, s) || !read_scalars(a + 9, op, s, c)) Py_RETURN_NONE;
  void* in[7];
  for (int i = 0; i < 7; ++i)
    if (!(in[i] = operand(a[1 + i], s))) Py_RETURN_NONE;
  const at::Tensor& lse = THPVariable_Unpack(a[8]);
  if (!usable(lse) || lse.dim() != 3 || lse.size(0) != s.B || lse.size(1) != s.N || lse.size(2) != s.T || lse.scalar_type() != at::kFloat ||
      lse.device().index() != s.device || !aligned(lse.data_ptr()))
    Py_RETURN_NONE;
  const void* saved = nullptr;
  size_t saved_bytes = 0;
  if (a[n - 1] != Py_None) {
    if (op != kDpsBwd || !is_tensor(a[n - 1])) Py_RETURN_NONE;
    const at::Tensor& w = THPVariable_Unpack(a[n - 1]);
    if (!usable(w) || w.scalar_type() != at::kByte || w.device().index() != s.device) Py_RETURN_NONE;
    saved = w.data_ptr();
    saved_bytes = (size_t)w.numel();
  }
  const float* const l = (const float*)lse.data_ptr();
  const size_t bytes = workspace_size(op, s, c);
  at::Tensor out[6];
  int rc = 0;
  {
    Unlocked unlocked;
    void* p[6];
    for (int i = 0; i < 6; ++i) {
      out[i] = i < 5 ? at::empty_like(q) : at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
      if (!(p[i] = fresh(out[i]))) rc = kNotPlain;
    }
    void* const stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)s.device).stream();
    if (rc == kNotPlain)
      ;
    else if (op == kTdpBwd)
      rc = lib.tdp_bwd(in[0], in[1], in[2], in[3], in[4], in[5], in[6], l, p[0], p[1], p[2], p[3], p[4], s.B, s.N, s.T, s.D, s.dtype,
                       c.scale, c.causal, c.w[0], c.w[1], c.w[2], c.w[3], 1, 0, p[5], bytes, c.status, c.flags, stream);
    else if (!saved)
      rc = lib.dps_bwd(in[0], in[1], in[2], in[3], in[4], in[5], in[6], l, p[0], p[1], p[2], p[3], p[4], s.B, s.N, s.T, s.D, s.dtype,
                       c.scale, c.causal, c.w[0], p[5], bytes, c.status, c.flags, stream);
    else
      rc = lib.dps_bwd_saved(in[0], in[1], in[2], in[3], in[4], in[5], in[6], l, p[0], p[1], p[2], p[3], p[4], s.B, s.N, s.T, s.D, s.dtype,
                             c.scale, c.causal, c.w[0], p[5], bytes, saved, saved_bytes, c.status, c.flags, stream);
  }
  if (rc == kNotPlain) Py_RETURN_NONE;
  if (rc != 0) return PyLong_FromLong(rc);
  return wrap_all(out, 5);
  END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------ norms with rotation, and the cache
// The same for these: tensors whose rows are contiguous and aligned, whatever their other strides; weights may be parameters.  Anything
// else, and any argument that Python's checks would refuse, is left to them.

// A plain tensor (or a parameter: read, and nothing allocated like it); null: not one.
const at::Tensor* plain(PyObject* o, int device) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || t.unsafeGetTensorImpl()->is_python_dispatch() || t.layout() != at::kStrided || !t.is_cuda() || !t.has_storage() ||
      t.is_neg() || t.numel() == 0 || (device >= 0 && t.device().index() != device))
    return nullptr;
  return &t;
}
// A contiguous one of a shape and type, aligned; null: not one.
template <typename T>
bool dense(PyObject* o, int device, at::ScalarType type, at::IntArrayRef sizes, uintptr_t align, T*& p) {
  const at::Tensor* t = plain(o, device);
  if (!t || t->scalar_type() != type || t->sizes() != sizes || !t->is_contiguous()) return false;
  p = (T*)t->data_ptr();
  return p != nullptr && ((uintptr_t)p & (align - 1)) == 0;
}

int dtype_code(at::ScalarType t) { return t == at::kFloat ? TRITT_F32 : t == at::kHalf ? TRITT_F16 : t == at::kBFloat16 ? TRITT_BF16 : -1; }
bool head_dim(int64_t D) { return D == 16 || D == 32 || D == 64 || D == 128 || D == 256; }

bool read_rows(const at::Tensor& t, tritt_rows_t& r) {
  const int64_t unit = 16 / (int64_t)t.element_size();
  if (t.dim() != 4 || (t.size(3) > 1 && t.stride(3) != 1) || !aligned(t.data_ptr())) return false;
  long long st[3];
  for (int i = 0; i < 3; ++i) {
    st[i] = t.size(i) > 1 ? t.stride(i) : 0;
    if (st[i] % unit) return false;
  }
  r = {t.data_ptr(), st[0], st[1], st[2]};
  return true;
}
// Rows of a tensor of the call's shape.
bool read_rows(PyObject* o, const Shape& s, tritt_rows_t& r) {
  const at::Tensor* t = plain(o, s.device);
  return t && t->dim() == 4 && t->scalar_type() == s.type && t->size(0) == s.B && t->size(1) == s.N && t->size(2) == s.T && t->size(3) == s.D &&
         read_rows(*t, r);
}
bool strided_shape(PyObject* o, Shape& s) {
  if (!is_tensor(o)) return false;
  const at::Tensor* t = plain(o, -1);
  if (!t || t->dim() != 4) return false;
  s.type = t->scalar_type();
  s.dtype = dtype_code(s.type);
  for (int i = 0; i < 4; ++i)
    if (t->size(i) > INT_MAX) return false;
  s.B = (int)t->size(0), s.N = (int)t->size(1), s.T = (int)t->size(2), s.D = (int)t->size(3);
  s.device = t->device().index();
  return s.dtype >= 0 && head_dim(s.D) && s.device >= 0 && s.device < kDevices && s.device == c10::cuda::current_device();
}
int* status_of(int device) {   // null: Python reports, or makes the word
  return lib.norm_fwd && status_words[device] && *status_words[device] == 0 ? const_cast<int*>(status_words[device]) : nullptr;
}

// q, k1, k2, three weights, cos, sin, positions, eps, interleaved
bool read_norm(PyObject* const* a, Shape& s, tritt_norm_rotary_t& n) {
  if (!strided_shape(a[0], s)) return false;
  n = {};
  for (int i = 0; i < 3; ++i)
    if (!is_tensor(a[i]) || !read_rows(a[i], s, n.x[i])) return false;
  n.B = s.B, n.N = s.N, n.T = s.T, n.D = s.D, n.dtype = s.dtype;
  n.weight_dtype = s.dtype;
  const at::Tensor* first = nullptr;
  for (int i = 0; i < 3; ++i) {
    if (a[3 + i] == Py_None) continue;
    const at::Tensor* w = plain(a[3 + i], s.device);
    if (!w || !w->is_contiguous() || !aligned(w->data_ptr()) || (w->scalar_type() != s.type && w->scalar_type() != at::kFloat)) return false;
    if (!(w->dim() == 1 && w->size(0) == s.D) && !(w->dim() == 2 && w->size(0) == s.N && w->size(1) == s.D)) return false;
    if (first && (first->dim() != w->dim() || first->scalar_type() != w->scalar_type())) return false;
    first = w;
    n.w[i] = w->data_ptr();
    n.weight_heads = w->dim() == 2;
    n.weight_dtype = dtype_code(w->scalar_type());
  }
  if (a[6] != Py_None) {
    const at::Tensor *c = plain(a[6], s.device), *sn = plain(a[7], s.device);
    if (!c || !sn || c->dim() != 2 || c->sizes() != sn->sizes() || c->scalar_type() != at::kFloat || sn->scalar_type() != at::kFloat ||
        !c->is_contiguous() || !sn->is_contiguous() || !aligned(c->data_ptr()) || !aligned(sn->data_ptr()) || c->size(0) > INT_MAX)
      return false;
    n.cos = (const float*)c->data_ptr(), n.sin = (const float*)sn->data_ptr();
    n.table = (int)c->size(0);
    if (2 * c->size(1) % 16 || 2 * c->size(1) > s.D) return false;
    n.rot = 2 * (int)c->size(1);
    if (a[8] != Py_None) {
      const at::Tensor* p = plain(a[8], s.device);
      if (!p || (p->scalar_type() != at::kLong && p->scalar_type() != at::kInt)) return false;
      if (!(p->dim() == 1 && p->size(0) == s.T) && !(p->dim() == 2 && p->size(0) == s.B && p->size(1) == s.T)) return false;
      n.positions = p->data_ptr();
      n.positions64 = p->scalar_type() == at::kLong;
      n.position_stride_t = p->stride(p->dim() - 1);
      n.position_stride_b = p->dim() == 2 ? p->stride(0) : 0;
    } else if (s.T > n.table) {
      return false;
    }
  } else if (a[7] != Py_None || a[8] != Py_None) {
    return false;
  }
  if (!read_float(a[9], n.eps) || !PyBool_Check(a[10])) return false;
  n.interleaved = a[10] == Py_True;
  return true;
}

// norm_rotary(q, k1, k2, weights..., cos, sin, positions, eps, interleaved) -> the three results, the library's error code, or None
PyObject* norm_rotary(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Shape s;
  tritt_norm_rotary_t args;
  if (n != 11 || !read_norm(a, s, args)) Py_RETURN_NONE;
  int* const status = status_of(s.device);
  if (!status) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(a[0]);
  at::Tensor out[3];
  int rc = 0;
  {
    Unlocked unlocked;
    for (int i = 0; i < 3; ++i) {
      out[i] = at::empty({s.B, s.N, s.T, s.D}, q.options());
      if (!fresh(out[i]) || !read_rows(out[i], args.y[i])) rc = kNotPlain;
    }
    if (rc == 0) rc = lib.norm_fwd(&args, status, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)s.device).stream());
  }
  if (rc == kNotPlain) Py_RETURN_NONE;
  return rc != 0 ? PyLong_FromLong(rc) : wrap_all(out, 3);
  END_HANDLE_TH_ERRORS
}

// norm_rotary_backward(the same, three gradients, three truth values: gradients of the weights) -> six gradients (None where
// not wanted), the library's error code, or None
PyObject* norm_rotary_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Shape s;
  tritt_norm_rotary_t args;
  if (n != 17 || !read_norm(a, s, args)) Py_RETURN_NONE;
  for (int i = 0; i < 3; ++i)
    if (!PyBool_Check(a[14 + i]) || a[11 + i] == Py_None || !read_rows(a[11 + i], s, args.y[i])) Py_RETURN_NONE;
  int* const status = status_of(s.device);
  if (!status) Py_RETURN_NONE;
  at::Tensor out[6], scratch;
  int rc = 0;
  {
    Unlocked unlocked;
    for (int i = 0; i < 3 && rc == 0; ++i) {
      out[i] = at::empty_like(THPVariable_Unpack(a[i]));
      if (out[i].unsafeGetTensorImpl()->is_python_dispatch() || !out[i].has_storage() || !read_rows(out[i], args.dx[i])) rc = kNotPlain;
      if (a[14 + i] == Py_True && args.w[i] && rc == 0) {
        const at::Tensor& w = THPVariable_Unpack(a[3 + i]);
        out[3 + i] = at::empty(w.sizes(), w.options());
        if (!(args.dw[i] = fresh(out[3 + i]))) rc = kNotPlain;
      }
    }
    if (rc == 0) {
      const size_t bytes = lib.norm_workspace(&args);
      void* w = nullptr;
      if (bytes) {
        scratch = at::empty({(int64_t)bytes}, out[0].options().dtype(at::kByte));
        if (!(w = fresh(scratch))) rc = kNotPlain;
      }
      if (rc == 0) rc = lib.norm_bwd(&args, w, bytes, status, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)s.device).stream());
    }
  }
  if (rc == kNotPlain) Py_RETURN_NONE;
  return rc != 0 ? PyLong_FromLong(rc) : wrap_all(out, 6);
  END_HANDLE_TH_ERRORS
}

// codes, exponents, lse, table, context, counts, ancestors, of a call for n new tokens
bool read_cache(PyObject* const* a, int n, tritt_cache_t& c, int& device) {
  const at::Tensor* codes = is_tensor(a[0]) ? plain(a[0], -1) : nullptr;
  if (!codes || codes->dim() != 5 || codes->size(1) != 4 || !codes->is_contiguous() || !aligned(codes->data_ptr())) return false;
  const at::ScalarType type = codes->scalar_type();
  c = {};
  c.code = type == at::kHalf ? TRITT_CODE_F16 : type == at::kFloat8_e4m3fn ? TRITT_CODE_E4M3 : type == at::kChar ? TRITT_CODE_INT8 : -1;
  device = codes->device().index();
  const int64_t pages = codes->size(0), N = codes->size(2), page = codes->size(3), D = codes->size(4);
  if (c.code < 0 || !head_dim(D) || pages > INT_MAX || N > INT_MAX || page > INT_MAX || device < 0 || device >= kDevices ||
      device != c10::cuda::current_device())
    return false;
  c.codes = codes->data_ptr();
  c.pages = (int)pages, c.N = (int)N, c.page_size = (int)page, c.D = (int)D;
  if (!dense(a[1], device, at::kByte, {pages, 4, N, page}, 16, c.exponents)) return false;
  if (a[2] != Py_None && !dense(a[2], device, at::kFloat, {pages, N, page}, 16, c.lse)) return false;
  const at::Tensor* table = plain(a[3], device);
  if (!table || table->dim() != 2 || table->scalar_type() != at::kInt || (table->size(1) > 1 && table->stride(1) != 1) || table->size(0) > INT_MAX ||
      table->size(1) > INT_MAX)
    return false;
  c.table = (const int*)table->data_ptr();
  c.B = (int)table->size(0), c.table_pages = (int)table->size(1);
  c.table_stride = c.B > 1 ? table->stride(0) : 0;
  c.n = n;
  if (!dense(a[4], device, at::kInt, {c.B}, 4, c.context)) return false;
  if (a[5] != Py_None && !dense(a[5], device, at::kInt, {c.B}, 4, c.counts)) return false;
  if (a[6] != Py_None && (n > TRITT_MAX_ANCESTORS || !dense(a[6], device, at::kLong, {c.B, n}, 8, c.ancestors))) return false;
  return true;
}
// Four tensors [B, N, n, D] of new tokens, or one.
bool read_new(PyObject* const* a, int count, const tritt_cache_t& c, int device, Shape& s, tritt_rows_t* rows) {
  if (!strided_shape(a[0], s) || s.device != device || s.B != c.B || s.N != c.N || s.D != c.D) return false;
  for (int i = 0; i < count; ++i)
    if (!read_rows(a[i], s, rows[i])) return false;
  return true;
}
int new_count(PyObject* o) {   // new tokens of a tensor; 0: not one
  if (!is_tensor(o)) return 0;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && t.dim() == 4 && t.size(2) > 0 && t.size(2) <= INT_MAX ? (int)t.size(2) : 0;
}

// cache_write(codes, exponents, lse, table, context, counts, None, k1, k2, v1, v2) -> the library's error code (0: done), or None
PyObject* cache_write(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  tritt_cache_t c;
  tritt_rows_t rows[4];
  Shape s;
  int device, tokens;
  if (n != 11 || !(tokens = new_count(a[7])) || !read_cache(a, tokens, c, device) || !read_new(a + 7, 4, c, device, s, rows)) Py_RETURN_NONE;
  int* const status = status_of(device);
  if (!status) Py_RETURN_NONE;
  int rc;
  {
    Unlocked unlocked;
    rc = lib.cache_write(&c, rows, s.dtype, status, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
  }
  return PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// cache_read(codes, exponents, lse, table, context, counts, None, n, dtype code) -> the parts and the log-sum-exps, an error code, or None
PyObject* cache_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  tritt_cache_t c;
  int device, tokens, dtype;
  if (n != 9 || !read_int(a[7], -1, tokens) || tokens < 1 || !read_int(a[8], -1, dtype) || dtype < TRITT_F32 || dtype > TRITT_BF16 ||
      !read_cache(a, tokens, c, device))
    Py_RETURN_NONE;
  int* const status = status_of(device);
  if (!status) Py_RETURN_NONE;
  const at::ScalarType type = dtype == TRITT_F32 ? at::kFloat : dtype == TRITT_F16 ? at::kHalf : at::kBFloat16;
  const at::Tensor& codes = THPVariable_Unpack(a[0]);
  at::Tensor out[5];
  const int count = c.lse ? 5 : 4;
  int rc = 0;
  {
    Unlocked unlocked;
    void* p[5];
    for (int i = 0; i < count; ++i) {
      out[i] = i < 4 ? at::empty({c.B, c.N, tokens, c.D}, codes.options().dtype(type)) : at::empty({c.B, c.N, tokens}, codes.options().dtype(at::kFloat));
      if (!(p[i] = fresh(out[i]))) rc = kNotPlain;
    }
    if (rc == 0)
      rc = lib.cache_read(&c, p, count == 5 ? (float*)p[4] : nullptr, dtype, status, c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream());
  }
  if (rc == kNotPlain) Py_RETURN_NONE;
  return rc != 0 ? PyLong_FromLong(rc) : wrap_all(out, count);
  END_HANDLE_TH_ERRORS
}

// decode(op, codes, exponents, lse, table, context, counts, ancestors, flags, scale, then
//   tdp: q, four windows, whether the log-sum-exp is wanted;   dps: q;   append: k1, k2, v1, v2, k_diff)
// -> (o, log-sum-exp or None), for append the error code 0; the library's error code, or None
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int op, flags, tokens, device, w[4] = {0, 0, 0, 0};
  float scale;
  tritt_cache_t c;
  tritt_rows_t rows[4];
  Shape s;
  if (n < 11 || !read_int(a[0], -1, op) || n != (op == TRITT_OP_TDP_DECODE ? 16 : op == TRITT_OP_DPS_APPEND ? 15 : 11) ||
      !read_int(a[8], -1, flags) || !read_float(a[9], scale) || !(tokens = new_count(a[10])) || !read_cache(a + 1, tokens, c, device) ||
      !read_new(a + 10, op == TRITT_OP_DPS_APPEND ? 4 : 1, c, device, s, rows))
    Py_RETURN_NONE;
  const bool tdp = op == TRITT_OP_TDP_DECODE, append = op == TRITT_OP_DPS_APPEND;
  if (!tdp && !c.lse) Py_RETURN_NONE;
  if (tdp && !PyBool_Check(a[15])) Py_RETURN_NONE;
  for (int i = 0; i < (tdp ? 4 : append ? 1 : 0); ++i)
    if (!read_int(a[(tdp ? 11 : 14) + i], tdp ? 1 << 30 : -1, w[i]) || w[i] < 0) Py_RETURN_NONE;
  int* const status = status_of(device);
  if (!status) Py_RETURN_NONE;
  const at::Tensor& q = THPVariable_Unpack(a[10]);
  at::Tensor out[2], scratch;
  int rc = 0;
  {
    Unlocked unlocked;
    const size_t bytes = std::max<size_t>(lib.decode_workspace(op, &c, s.dtype, w[0], w[1], flags), 256);
    void *o = nullptr, *l = nullptr, *ws;
    if (!append) {
      out[0] = at::empty({s.B, s.N, s.T, s.D}, q.options());
      if (!(o = fresh(out[0]))) rc = kNotPlain;
      if (!tdp || a[15] == Py_True) {
        out[1] = at::empty({s.B, s.N, s.T}, q.options().dtype(at::kFloat));
        if (!(l = fresh(out[1]))) rc = kNotPlain;
      }
    }
    scratch = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    if (!(ws = fresh(scratch))) rc = kNotPlain;
    void* const stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    if (rc == kNotPlain)
      ;
    else if (tdp)
      rc = lib.tdp_decode(&c, rows, o, (float*)l, s.dtype, scale, w[0], w[1], w[2], w[3], ws, bytes, status, flags, stream);
    else if (append)
      rc = lib.dps_append(&c, rows, s.dtype, scale, w[0], ws, bytes, status, flags, stream);
    else
      rc = lib.dps_decode(&c, rows, o, (float*)l, s.dtype, scale, ws, bytes, status, flags, stream);
  }
  if (rc == kNotPlain) Py_RETURN_NONE;
  return rc != 0 || append ? PyLong_FromLong(rc) : wrap_all(out, 2);
  END_HANDLE_TH_ERRORS
}

// init(addresses of the entry points, in the order of Entries)
PyObject* init(PyObject*, PyObject* args) {
  constexpr Py_ssize_t kEntries = sizeof(Entries) / sizeof(void*);
  if (PyTuple_GET_SIZE(args) != kEntries) {
    PyErr_SetString(PyExc_TypeError, "another number of entry points");
    return nullptr;
  }
  void* f[kEntries];
  for (Py_ssize_t i = 0; i < kEntries; ++i) {
    f[i] = PyLong_AsVoidPtr(PyTuple_GET_ITEM(args, i));
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_TypeError, "a missing entry point");
      return nullptr;
    }
  }
  std::memcpy(&lib, f, sizeof(lib));
  Py_RETURN_NONE;
}

// set_status(device, address of its status word)
PyObject* set_status(PyObject*, PyObject* args) {
  int device;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "iK", &device, &address)) return nullptr;
  if (device >= 0 && device < kDevices) status_words[device] = (volatile int*)address;
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {{"init", init, METH_VARARGS, nullptr},
                         {"set_status", set_status, METH_VARARGS, nullptr},
                         {"forward", (PyCFunction)(void (*)(void))forward, METH_FASTCALL, nullptr},
                         {"backward", (PyCFunction)(void (*)(void))backward, METH_FASTCALL, nullptr},
                         {"norm_rotary", (PyCFunction)(void (*)(void))norm_rotary, METH_FASTCALL, nullptr},
                         {"norm_rotary_backward", (PyCFunction)(void (*)(void))norm_rotary_backward, METH_FASTCALL, nullptr},
                         {"cache_write", (PyCFunction)(void (*)(void))cache_write, METH_FASTCALL, nullptr},
                         {"cache_read", (PyCFunction)(void (*)(void))cache_read, METH_FASTCALL, nullptr},
                         {"decode", (PyCFunction)(void (*)(void))decode, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
  PyObject* m = PyModule_Create(&module);
  // (the version whose headers this was compiled with: objects' layouts are its own)
  if (m && PyModule_AddStringConstant(m, "torch_version", TRITT_TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
