// paged_binding.cpp — the Python calls of the paged-cache operators (ops.paged_*):
// checks the tensors, fills the C ABI's argument structure and calls it on the
// current stream. The kernels of a decode step take 4 to 8 us each, and the same
// checks written in Python took 8 us of host time a call: 12 in all, now 5.
//
// Built as a CPython module against torch's headers; libsa_b200.so stays free of
// both and is reached through the addresses that init() is given.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>

#include "../../include/sparse_attn_b200.h"

namespace {

struct Raised {};  // a Python exception is set

[[noreturn]] void raise(PyObject* type, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  PyErr_FormatV(type, fmt, ap);
  va_end(ap);
  throw Raised{};
}

decltype(&sa_paged_append) f_append;
decltype(&sa_paged_attn) f_attn;
decltype(&sa_paged_attn_workspace) f_workspace;
decltype(&sa_paged_select) f_select;

using at::Tensor;

std::string text(const Tensor& t) {
  std::string s = std::string(c10::toString(t.scalar_type())) + " [";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "] on " + t.device().str();
}

// What all tensors of a call share, and how they are read.
struct Call {
  const char* op;
  c10::Device dev{c10::kCPU};
  at::ScalarType half = at::kBFloat16;

  const Tensor& tensor(PyObject* o, const char* name) const {
    if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s: %s must be a tensor", op, name);
    return THPVariable_Unpack(o);
  }
  // The tensor that sets type and device.
  const Tensor& lead(PyObject* o, const char* name, int32_t& code) {
    const Tensor& t = tensor(o, name);
    if (!t.is_cuda())
      raise(PyExc_RuntimeError, "cuda_sparse_attention ops need CUDA tensors (there is no CPU path)");
    half = t.scalar_type();
    if (half != at::kBFloat16 && half != at::kHalf)
      raise(PyExc_TypeError, "%s: bf16 or fp16 tensors expected, got %s", op, text(t).c_str());
    dev = t.device();
    code = half == at::kBFloat16 ? SA_BF16 : SA_FP16;
    return t;
  }
  void check(const Tensor& t, const char* name, at::ScalarType type, int64_t ndim) const {
    if (t.scalar_type() != type || t.device() != dev || t.dim() != ndim)
      raise(PyExc_TypeError, "%s: %s must be %s of %lld dimensions on %s, got %s", op, name, c10::toString(type),
            (long long)ndim, dev.str().c_str(), text(t).c_str());
    if (t.size(-1) > 1 && t.stride(-1) != 1)
      raise(PyExc_ValueError, "%s: the last dimension of %s must be contiguous", op, name);
  }
  // Checks, and writes the strides of all but the last dimension.
  void strides(const Tensor& t, const char* name, at::ScalarType type, int64_t n, int64_t* out) const {
    check(t, name, type, n + 1);
    for (int64_t i = 0; i < n; ++i) out[i] = t.stride(i);
  }
  void shape(const Tensor& t, const char* name, std::initializer_list<int64_t> want) const {
    if (!t.sizes().equals(at::IntArrayRef(want))) {
      std::string s;
      for (int64_t w : want) s += (s.empty() ? "" : ", ") + std::to_string(w);
      raise(PyExc_ValueError, "%s: %s must be [%s], got %s", op, name, s.c_str(), text(t).c_str());
    }
  }
  int32_t int32(PyObject* o, const char* name) const {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    if (v < INT32_MIN || v > INT32_MAX) raise(PyExc_ValueError, "%s: %s is out of range", op, name);
    return (int32_t)v;
  }
  int32_t size(int64_t v, const char* name) const {
    if (v > INT32_MAX) raise(PyExc_ValueError, "%s: %s is out of range", op, name);
    return (int32_t)v;
  }
  double real(PyObject* o) const {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
  }

  // page_table [B, pages], cu_q [B + 1], seq_lens [B]; false for a batch without rows.
  bool batch(sa_paged_batch& b, int64_t N, PyObject* table_o, PyObject* cu_o, PyObject* lens_o, int64_t pages,
             int64_t page_size) const {
    const Tensor &table = tensor(table_o, "page_table"), &cu = tensor(cu_o, "cu_q"), &lens = tensor(lens_o, "seq_lens");
    strides(table, "page_table", at::kInt, 1, &b.table_stride);
    check(cu, "cu_q", at::kInt, 1);
    check(lens, "seq_lens", at::kInt, 1);
    const int64_t B = lens.numel();
    shape(table, "page_table", {B, table.size(1)});
    shape(cu, "cu_q", {B + 1});
    b.table = static_cast<const int32_t*>(table.data_ptr());
    b.cu_q = static_cast<const int32_t*>(cu.data_ptr());
    b.seq_lens = static_cast<const int32_t*>(lens.data_ptr());
    b.B = size(B, "the batch");
    b.N = size(N, "the batch");
    b.max_pages = size(table.size(1), "the page table");
    b.num_pages = size(pages, "the page pool");
    b.page_size = size(page_size, "page_size");
    return N > 0 && B > 0;
  }
  void pages(const Tensor& k, const Tensor& v, int64_t Hkv, int64_t D, int64_t* ks, int64_t* vs) const {
    strides(k, "k_pages", half, 3, ks);
    strides(v, "v_pages", half, 3, vs);
    shape(k, "k_pages", {k.size(0), Hkv, k.size(2), D});
    shape(v, "v_pages", {k.size(0), Hkv, k.size(2), D});
  }
  template <typename F, typename A>
  int run(F f, const A& args) const {
    const c10::cuda::OptionalCUDAGuard guard(dev);
    return f(&args, c10::cuda::getCurrentCUDAStream(dev.index()).stream());
  }
};

// The wrapped tensor, or the status of the C call where it is not 0.
PyObject* result(int rc, const Tensor& t) {
  if (rc) return PyLong_FromLong(rc);
  return THPVariable_Wrap(t);
}

template <typename F>
PyObject* guarded(Py_ssize_t have, Py_ssize_t want, F f) {
  try {
    if (have != want) raise(PyExc_TypeError, "%zd arguments expected, got %zd", want, have);
    return f();
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* torch = PyImport_ImportModule("torch");
    PyObject* type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// qkv, q_weight, k_weight, cos, sin, k_pages, v_pages, page_table, cu_q, seq_lens, Hq, Hkv, eps, k_bounds, q_out
PyObject* append(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 15, [&]() {
    Call c{"paged_qk_norm_rope_append"};
    sa_paged_append_args a{};
    const Tensor& qkv = c.lead(o[0], "qkv", a.dtype);
    a.Hq = c.int32(o[10], "Hq");
    a.Hkv = c.int32(o[11], "Hkv");
    int64_t st[2];
    c.strides(qkv, "qkv", c.half, 2, st);
    const int64_t N = qkv.size(0), D = qkv.size(2);
    c.shape(qkv, "qkv", {N, (int64_t)a.Hq + 2 * (int64_t)a.Hkv, D});
    if (st[1] != D && qkv.size(1) > 1) raise(PyExc_ValueError, "%s: the heads of qkv must be contiguous", c.op);
    a.qkv = qkv.data_ptr();
    a.qkv_st = st[0];
    const void** weight[2] = {&a.q_weight, &a.k_weight};
    for (int i = 0; i < 2; ++i) {
      if (o[1 + i] == Py_None) continue;
      const Tensor& w = c.tensor(o[1 + i], "a weight");
      c.check(w, "a weight", c.half, 1);
      c.shape(w, "a weight", {D});
      *weight[i] = w.data_ptr();
    }
    const Tensor &cos = c.tensor(o[3], "cos"), &sin = c.tensor(o[4], "sin");
    c.check(cos, "cos", c.half, 2);
    c.check(sin, "sin", c.half, 2);
    c.shape(cos, "cos", {cos.size(0), D});
    c.shape(sin, "sin", {cos.size(0), D});
    if (!cos.is_contiguous() || !sin.is_contiguous()) raise(PyExc_ValueError, "%s: cos / sin must be contiguous", c.op);
    a.cos = cos.data_ptr();
    a.sin = sin.data_ptr();
    a.positions = c.size(cos.size(0), "positions");
    const Tensor &k = c.tensor(o[5], "k_pages"), &v = c.tensor(o[6], "v_pages");
    c.pages(k, v, a.Hkv, D, a.k_strides, a.v_strides);
    a.k_pages = k.data_ptr();
    a.v_pages = v.data_ptr();
    if (o[13] != Py_None) {
      const Tensor& b = c.tensor(o[13], "k_bounds");
      c.strides(b, "k_bounds", c.half, 3, a.b_strides);
      c.shape(b, "k_bounds", {k.size(0), a.Hkv, 2, D});
      a.bounds = b.data_ptr();
    }
    const Tensor out = o[14] == Py_None ? at::empty({N, a.Hq, D}, qkv.options()) : c.tensor(o[14], "q_out");
    c.strides(out, "q_out", c.half, 2, a.q_strides);
    c.shape(out, "q_out", {N, a.Hq, D});
    a.q_out = out.data_ptr();
    a.D = c.size(D, "head_dim");
    a.eps = (float)c.real(o[12]);
    if (!c.batch(a.batch, N, o[7], o[8], o[9], k.size(0), k.size(2))) return result(0, out);
    return result(c.run(f_append, a), out);
  });
}

// q, k_bounds, page_table, cu_q, seq_lens, page_size, keep, first, recent, max_q, out
PyObject* select(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 11, [&]() {
    Call c{"paged_block_select"};
    sa_paged_select_args a{};
    const Tensor& q = c.lead(o[0], "q", a.dtype);
    const Tensor& b = c.tensor(o[1], "k_bounds");
    c.strides(q, "q", c.half, 2, a.q_strides);
    c.strides(b, "k_bounds", c.half, 3, a.b_strides);
    const int64_t N = q.size(0), Hkv = b.size(1);
    c.shape(b, "k_bounds", {b.size(0), Hkv, 2, q.size(2)});
    a.q = q.data_ptr();
    a.bounds = b.data_ptr();
    a.Hq = c.size(q.size(1), "Hq");
    a.Hkv = c.size(Hkv, "Hkv");
    a.D = c.size(q.size(2), "head_dim");
    a.keep = c.int32(o[6], "keep");
    a.first = c.int32(o[7], "first");
    a.recent = c.int32(o[8], "recent");
    a.max_q = o[9] == Py_None ? c.size(N, "the batch") : c.int32(o[9], "max_q");
    if (a.keep < 1) raise(PyExc_ValueError, "%s: keep must be at least 1", c.op);
    const Tensor out =
        o[10] == Py_None ? at::empty({N, Hkv, a.keep}, q.options().dtype(at::kInt)) : c.tensor(o[10], "out");
    c.strides(out, "out", at::kInt, 2, a.out_strides);
    c.shape(out, "out", {N, Hkv, a.keep});
    a.out = static_cast<int32_t*>(out.data_ptr());
    if (!c.batch(a.batch, N, o[2], o[3], o[4], b.size(0), c.int32(o[5], "page_size"))) return result(0, out);
    return result(c.run(f_select, a), out);
  });
}

// q, k_pages, v_pages, page_table, cu_q, seq_lens, max_q, max_len, blocks, scale, split_len, out: false for a
// batch without rows. `out` stays undefined where it is not wanted (workspace query).
bool attn_args(Call& c, PyObject* const* o, sa_paged_attn_args& a, Tensor* out) {
  const Tensor& q = c.lead(o[0], "q", a.dtype);
  const Tensor &k = c.tensor(o[1], "k_pages"), &v = c.tensor(o[2], "v_pages");
  c.strides(q, "q", c.half, 2, a.q_strides);
  const int64_t N = q.size(0), D = q.size(2);
  if (k.dim() != 4) raise(PyExc_ValueError, "%s: k_pages must have 4 dimensions, got %s", c.op, text(k).c_str());
  c.pages(k, v, k.size(1), D, a.k_strides, a.v_strides);
  a.q = q.data_ptr();
  a.k_pages = k.data_ptr();
  a.v_pages = v.data_ptr();
  a.Hq = c.size(q.size(1), "Hq");
  a.Hkv = c.size(k.size(1), "Hkv");
  a.D = c.size(D, "head_dim");
  if (o[8] != Py_None) {
    const Tensor& b = c.tensor(o[8], "blocks");
    c.strides(b, "blocks", at::kInt, 2, a.blocks_strides);
    c.shape(b, "blocks", {N, k.size(1), b.size(2)});
    // (a tensor without elements has no address, and none means no lists)
    if (b.size(2) < 1) raise(PyExc_ValueError, "%s: blocks must have room for one page at least", c.op);
    a.blocks = static_cast<const int32_t*>(b.data_ptr());
    a.n_blocks = c.size(b.size(2), "blocks");
  }
  a.scale = o[9] == Py_None ? (float)(1.0 / std::sqrt((double)D)) : (float)c.real(o[9]);
  if (out) {
    *out = o[11] == Py_None ? at::empty_like(q) : c.tensor(o[11], "out");
    c.strides(*out, "out", c.half, 2, a.o_strides);
    c.shape(*out, "out", {N, q.size(1), D});
    a.out = out->data_ptr();
  } else {
    a.out = q.data_ptr();
    a.o_strides[0] = q.size(1) * D;
    a.o_strides[1] = D;
  }
  const bool rows = c.batch(a.batch, N, o[3], o[4], o[5], k.size(0), k.size(2));
  a.max_q = o[6] == Py_None ? a.batch.N : c.int32(o[6], "max_q");
  a.max_len = o[7] == Py_None ? c.size((int64_t)a.batch.max_pages * a.batch.page_size, "max_len")
                              : c.int32(o[7], "max_len");
  a.split_len = o[10] == Py_None ? 0 : c.int32(o[10], "split_len");
  return rows;
}

// ... and workspace
PyObject* attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 13, [&]() {
    Call c{"paged_attention"};
    sa_paged_attn_args a{};
    Tensor out, ws;
    if (!attn_args(c, o, a, &out)) return result(0, out);
    int rc = SA_ERR_WORKSPACE;
    if (o[12] == Py_None) rc = c.run(f_attn, a);
    if (rc != SA_ERR_WORKSPACE) return result(rc, out);
    int64_t need = 0;
    {
      const c10::cuda::OptionalCUDAGuard guard(c.dev);
      rc = f_workspace(&a, &need);
    }
    if (rc) return result(rc, out);
    ws = o[12] == Py_None ? at::empty({need}, out.options().dtype(at::kFloat)) : c.tensor(o[12], "workspace");
    if (ws.scalar_type() != at::kFloat || ws.device() != c.dev || !ws.is_contiguous() || ws.numel() < need)
      raise(PyExc_ValueError, "%s: workspace must be %lld contiguous float32 on %s, got %s", c.op, (long long)need,
            c.dev.str().c_str(), text(ws).c_str());
    if (reinterpret_cast<uintptr_t>(ws.data_ptr()) & 15u)
      raise(PyExc_ValueError, "%s: workspace must be 16-byte aligned", c.op);
    a.workspace = static_cast<float*>(ws.data_ptr());
    return result(c.run(f_attn, a), out);
  });
}

// the floats (>= 0), or the status of the C call (< 0)
PyObject* workspace(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 12, [&]() {
    Call c{"paged_attention_workspace"};
    sa_paged_attn_args a{};
    int64_t need = 0;
    if (!attn_args(c, o, a, nullptr)) return PyLong_FromLong(0);
    const c10::cuda::OptionalCUDAGuard guard(c.dev);
    const int rc = f_workspace(&a, &need);
    return PyLong_FromLongLong(rc ? rc : need);
  });
}

// Addresses of sa_paged_append, sa_paged_attn, sa_paged_attn_workspace, sa_paged_select.
PyObject* init(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded(n, 4, [&]() {
    void* p[4];
    for (int i = 0; i < 4; ++i) {
      p[i] = PyLong_AsVoidPtr(o[i]);
      if (!p[i]) raise(PyExc_ValueError, "bad address");
    }
    f_append = reinterpret_cast<decltype(f_append)>(p[0]);
    f_attn = reinterpret_cast<decltype(f_attn)>(p[1]);
    f_workspace = reinterpret_cast<decltype(f_workspace)>(p[2]);
    f_select = reinterpret_cast<decltype(f_select)>(p[3]);
    Py_INCREF(Py_None);
    return Py_None;
  });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(init),   METHOD(append),    METHOD(select),
                         METHOD(attention), METHOD(workspace), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_sa_paged", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sa_paged() { return PyModule_Create(&module); }
