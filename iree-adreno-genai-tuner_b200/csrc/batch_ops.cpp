// The batched serving operators for torch tensors, as a CPython module (q4b._batch_ops): argument checks, the
// output and workspace allocations and the call into libq4b.so, without per-argument Python work. A step of
// single tokens runs for a few microseconds on the GPU; the same checks in Python with ctypes took 50-65 us of host time
// a call, this module takes 5 (10 to 15 for the attention, with two or three launches and its tensor maps). Refused
// arguments raise ValueError; a library error comes back as its negative code, which the Python side turns into Q4BError
// with the library's message; torch's errors keep their types.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>

#include "q4b.h"

namespace {

// The library's entry points, from the copy of libq4b.so that the Python side has loaded.
struct Api {
  decltype(&q4b_paged_rope_append) append = nullptr;
  decltype(&q4b_prefix_attention_workspace) attention_workspace = nullptr;
  decltype(&q4b_prefix_attention) attention = nullptr;
  decltype(&q4b_verify_drafts) verify = nullptr;
} api;

struct Refuse {
  std::string why;
};

const char* type_name(at::ScalarType t) { return c10::toString(t); }

int dtype_of(at::ScalarType t) {
  return t == at::kFloat ? Q4B_F32 : t == at::kHalf ? Q4B_F16 : t == at::kBFloat16 ? Q4B_BF16 : -1;
}

struct Call {
  const char* what;
  c10::Device device{c10::kCUDA, -1};

  [[noreturn]] void refuse(const std::string& why) const { throw Refuse{std::string(what) + ": " + why}; }
  void need(bool ok, const char* why) const {
    if (!ok) refuse(why);
  }

  // a CUDA tensor on the device of the first one; None is allowed where `optional`
  const at::Tensor* tensor(PyObject* o, const char* name, bool optional = false) {
    if (optional && o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) refuse(std::string(name) + " must be a CUDA tensor (there is no CPU path)");
    if (t.requires_grad() && c10::GradMode::is_enabled())
      refuse(std::string(name) + " requires grad, and there is no backward pass: detach it, or call under torch.no_grad()");
    if (device.index() < 0)
      device = t.device();
    else if (t.device() != device)
      refuse(std::string(name) + " is on " + t.device().str() + ", the others on " + device.str());
    return &t;
  }
  const at::Tensor* int32(PyObject* o, const char* name, int dim) {
    const at::Tensor* t = tensor(o, name);
    if (t->scalar_type() != at::kInt || t->dim() != dim || (t->numel() && t->size(-1) > 1 && t->stride(-1) != 1))
      refuse(std::string(name) + " must be an int32 tensor of " + std::to_string(dim) +
             " dimension(s), the last contiguous");
    return t;
  }
  int size32(int64_t n, const char* name) const {
    if (n >= (int64_t(1) << 31)) refuse(std::string(name) + " is too large");
    return (int)n;
  }
  int integer(PyObject* o, const char* name) const {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      refuse(std::string(name) + " must be an integer");
    }
    if (v < 0 || v >= (1ll << 31)) refuse(std::string(name) + " " + std::to_string(v) + " is out of range");
    return (int)v;
  }

  q4b_batch batch(PyObject* q_start, PyObject* seq_lens, PyObject* page_table, PyObject* prefix_len) {
    const at::Tensor *qs = int32(q_start, "q_start", 1), *sl = int32(seq_lens, "seq_lens", 1),
                     *pt = int32(page_table, "page_table", 2);
    const int64_t n = sl->size(0);
    if (qs->size(0) != n + 1 || pt->size(0) != n)
      refuse(std::to_string(n) + " seq_lens need q_start [" + std::to_string(n + 1) + "] and page_table [" +
             std::to_string(n) + ", ...]");
    q4b_batch b = {};
    b.q_start = static_cast<const int32_t*>(qs->data_ptr());
    b.seq_lens = static_cast<const int32_t*>(sl->data_ptr());
    b.page_table = static_cast<const int32_t*>(pt->data_ptr());
    b.batch = size32(n, "the batch");
    b.table_width = size32(pt->size(1), "page_table");
    b.table_stride = n > 1 ? pt->stride(0) : pt->size(1);
    b.prefix_len = integer(prefix_len, "prefix_len");
    return b;
  }
  q4b_paged_kv paged_kv(PyObject* k_pages, PyObject* v_pages, at::ScalarType& type) {
    const at::Tensor *k = tensor(k_pages, "k_pages"), *v = tensor(v_pages, "v_pages");
    need(k->dim() == 4 && k->sizes() == v->sizes() && k->scalar_type() == v->scalar_type(),
         "k_pages and v_pages must be [n_pages, page_size, n_kv_heads, head_dim] of one type");
    type = k->scalar_type();
    if (type != at::kHalf && type != at::kBFloat16) refuse(std::string("the cache is fp16 or bf16, not ") + type_name(type));
    need(k->strides() == v->strides() && k->stride(3) == 1,
         "k_pages and v_pages need the same strides, head_dim contiguous");
    q4b_paged_kv kv;
    kv.k = k->data_ptr();
    kv.v = v->data_ptr();
    kv.dtype = dtype_of(type);
    kv.n_pages = size32(k->size(0), "the cache");
    kv.page_size = size32(k->size(1), "the cache");
    kv.n_kv_heads = size32(k->size(2), "the cache");
    kv.head_dim = size32(k->size(3), "the cache");
    kv.page_stride = k->stride(0);
    kv.slot_stride = k->stride(1);
    kv.head_stride = k->stride(2);
    return kv;
  }
  // [rows, heads, dim] with a row's heads contiguous -> the stride between rows
  long long row_stride(const at::Tensor& t, const char* name, int64_t heads, int64_t dim) const {
    if (t.dim() != 3 || t.size(1) != heads || t.size(2) != dim)
      refuse(std::string(name) + " must be [rows, " + std::to_string(heads) + ", " + std::to_string(dim) + "]");
    if (t.numel() && ((dim > 1 && t.stride(2) != 1) || (heads > 1 && t.stride(1) != dim)))
      refuse(std::string("the heads of a row of ") + name + " must be contiguous");
    return t.size(0) > 1 ? t.stride(0) : heads * dim;
  }
  at::Tensor output(PyObject* given, const char* name, at::IntArrayRef shape, at::ScalarType type) {
    const at::Tensor* t = tensor(given, name, true);
    if (!t) return at::empty(shape, at::TensorOptions().dtype(type).device(device));
    if (t->sizes() != shape || t->scalar_type() != type || !t->is_contiguous())
      refuse(std::string(name) + " must be a contiguous tensor of the result's shape and type");
    return *t;
  }
  // Tensors that a call wrote in place count it, so that autograd notices if it had saved one (inference tensors hold no count).
  static void wrote(PyObject* o) {
    if (o == Py_None) return;
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
  }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device.index()).stream(); }
};

template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, const char* what, F&& f) {
  if (given != wanted) return PyErr_Format(PyExc_TypeError, "%s: %zd arguments, not %zd", what, wanted, given);
  if (!api.verify) return PyErr_Format(PyExc_RuntimeError, "%s: the library is not bound", what);
  try {
    Call c{what};
    return f(c);
  } catch (const Refuse& e) {
    PyErr_SetString(PyExc_ValueError, e.why.c_str());
  } catch (...) {  // torch's own, with their types: torch.OutOfMemoryError from an allocation among them
    if (!PyErr_Occurred()) torch::translate_exception_to_python(std::current_exception());
  }
  return nullptr;
}

PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 13, "paged_rope_append", [&](Call& c) -> PyObject* {
    const at::Tensor *q = c.tensor(a[0], "q"), *k = c.tensor(a[1], "k"), *v = c.tensor(a[2], "v");
    at::ScalarType type;
    const q4b_paged_kv kv = c.paged_kv(a[3], a[4], type);
    const q4b_batch b = c.batch(a[7], a[6], a[5], a[10]);
    const at::Tensor *cos = c.tensor(a[8], "cos", true), *sin = c.tensor(a[9], "sin", true);
    int inter = -1;
    if (PyUnicode_Check(a[11]))
      inter = PyUnicode_CompareWithASCIIString(a[11], "half") == 0 ? 0
              : PyUnicode_CompareWithASCIIString(a[11], "interleaved") == 0 ? 1 : -1;
    c.need(inter >= 0, "layout is 'half' or 'interleaved'");
    c.need(q->dim() == 3, "q must be [rows, heads, head_dim]");
    const int64_t rows = q->size(0), heads = q->size(1);
    const long long qs = c.row_stride(*q, "q", heads, kv.head_dim), ks = c.row_stride(*k, "k", kv.n_kv_heads, kv.head_dim),
                    vs = c.row_stride(*v, "v", kv.n_kv_heads, kv.head_dim);
    c.need(k->size(0) == rows && v->size(0) == rows && k->scalar_type() == q->scalar_type() &&
               v->scalar_type() == q->scalar_type(),
           "q, k and v need the same rows and type");
    if (q->scalar_type() != at::kFloat && q->scalar_type() != type)
      c.refuse(std::string("q, k and v are fp32 or of the cache's type, not ") + type_name(q->scalar_type()));
    c.need(!cos == !sin, "cos and sin come together");
    long long ts = 0;
    int table_rows = 0, rot = 0;
    if (cos) {
      c.need(cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->scalar_type() == at::kFloat &&
                 sin->scalar_type() == at::kFloat && cos->strides() == sin->strides() &&
                 (cos->size(1) <= 1 || cos->stride(1) == 1),
             "cos and sin must be fp32 [positions, rot / 2] with the same strides");
      table_rows = c.size32(cos->size(0), "cos");
      rot = 2 * c.size32(std::min<int64_t>(cos->size(1), 1 << 29), "cos");
      ts = cos->stride(0);
    }
    at::Tensor out = c.output(a[12], "q_out", q->sizes(), type);
    int rc = 0;
    if (rows) {
      const c10::cuda::CUDAGuard guard(c.device);
      rc = api.append(q->data_ptr(), k->data_ptr(), v->data_ptr(), dtype_of(q->scalar_type()), qs, ks, vs,
                      c.size32(rows, "q"), c.size32(heads, "q"), rot ? static_cast<const float*>(cos->data_ptr()) : nullptr,
                      rot ? static_cast<const float*>(sin->data_ptr()) : nullptr, ts, table_rows, rot, inter, &b, &kv,
                      out.data_ptr(), c.stream());
      if (!rc)
        for (int i : {3, 4, 12}) c.wrote(a[i]);
    }
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  });
}

PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 12, "prefix_attention", [&](Call& c) -> PyObject* {
    const at::Tensor* q = c.tensor(a[0], "q");
    at::ScalarType type;
    const q4b_paged_kv kv = c.paged_kv(a[1], a[2], type);
    const at::Tensor* pages = c.int32(a[3], "prefix_pages", 1);
    q4b_batch b = c.batch(a[7], a[6], a[5], a[4]);
    if (a[10] != Py_None) b.max_new = c.integer(a[10], "max_new");
    if (a[11] != Py_None) b.own_keys = c.integer(a[11], "own_keys");
    if (pages->size(0) * (long long)kv.page_size < b.prefix_len)
      c.refuse(std::to_string(pages->size(0)) + " prefix pages of " + std::to_string(kv.page_size) + " hold no " +
               std::to_string(b.prefix_len) + " keys");
    c.need(q->dim() == 3 && q->size(2) == kv.head_dim && q->scalar_type() == type &&
               (q->numel() == 0 || kv.head_dim == 1 || q->stride(2) == 1),
           "q must be [rows, heads, head_dim] of the cache's type, head_dim contiguous");
    const int64_t rows = q->size(0), heads = q->size(1);
    double scale = kv.head_dim > 0 ? 1.0 / std::sqrt((double)kv.head_dim) : 1.0;
    if (a[8] != Py_None) {
      scale = PyFloat_AsDouble(a[8]);
      if (scale == -1.0 && PyErr_Occurred()) return nullptr;
    }
    at::Tensor out = c.output(a[9], "out", {rows, heads * kv.head_dim}, type);
    int rc = 0;
    if (rows) {
      const c10::cuda::CUDAGuard guard(c.device);
      const int r = c.size32(rows, "q"), h = c.size32(heads, "q");
      // made anew for each call: the allocator keeps streams and captured graphs apart
      const size_t bytes = api.attention_workspace(r, h, &b, &kv);
      const at::Tensor ws = at::empty({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(c.device));
      rc = api.attention(q->data_ptr(), r > 1 ? q->stride(0) : 0, h > 1 ? q->stride(1) : 0, r, h, (float)scale,
                         static_cast<const int32_t*>(pages->data_ptr()), &b, &kv, out.data_ptr(), ws.data_ptr(), bytes,
                         c.stream());
      if (!rc) c.wrote(a[9]);
    }
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
  });
}

PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded(n, 6, "verify_drafts", [&](Call& c) -> PyObject* {
    const at::Tensor *p = c.tensor(a[0], "target"), *d = c.tensor(a[1], "draft", true), *tok = c.int32(a[2], "tokens", 1),
                     *u = c.tensor(a[3], "uniforms"), *qs = c.int32(a[4], "q_start", 1);
    const int dt = dtype_of(p->scalar_type());
    c.need(p->dim() == 2 && dt >= 0 && (p->size(1) <= 1 || p->stride(1) == 1),
           "target must be fp32, fp16 or bf16 [rows, vocab], the last dimension contiguous");
    const int64_t rows = p->size(0), vocab = p->size(1);
    c.need(!d || (d->sizes() == p->sizes() && d->scalar_type() == p->scalar_type() && (vocab <= 1 || d->stride(1) == 1)),
           "draft must be like target");
    c.need(tok->size(0) == rows && u->dim() == 1 && u->size(0) == rows && u->scalar_type() == at::kFloat &&
               (rows <= 1 || u->stride(0) == 1),
           "the rows need int32 tokens [rows] and contiguous fp32 uniforms [rows]");
    c.need(qs->size(0) >= 1, "q_start must be [batch + 1]");
    const int64_t batch = qs->size(0) - 1;
    at::Tensor out = c.output(a[5], "out", {rows}, at::kInt);
    at::Tensor accepted = at::empty({batch}, at::TensorOptions().dtype(at::kInt).device(c.device));
    int rc;
    {
      const c10::cuda::CUDAGuard guard(c.device);
      rc = api.verify(p->data_ptr(), d ? d->data_ptr() : nullptr, dt, rows > 1 ? p->stride(0) : vocab,
                      d && rows > 1 ? d->stride(0) : vocab, c.size32(vocab, "target"),
                      static_cast<const int32_t*>(tok->data_ptr()), static_cast<const float*>(u->data_ptr()),
                      c.size32(rows, "target"), static_cast<const int32_t*>(qs->data_ptr()), c.size32(batch, "q_start"),
                      static_cast<int32_t*>(out.data_ptr()), static_cast<int32_t*>(accepted.data_ptr()), c.stream());
    }
    if (rc) return PyLong_FromLong(rc);
    c.wrote(a[5]);
    PyObject* pair = PyTuple_New(2);
    if (!pair) return nullptr;
    PyTuple_SET_ITEM(pair, 0, THPVariable_Wrap(out));
    PyTuple_SET_ITEM(pair, 1, THPVariable_Wrap(accepted));
    return pair;
  });
}

// bind(append, attention_workspace, attention, verify): addresses in the loaded library
PyObject* bind(PyObject*, PyObject* args) {
  unsigned long long p[4];
  if (!PyArg_ParseTuple(args, "KKKK", &p[0], &p[1], &p[2], &p[3])) return nullptr;
  for (auto x : p)
    if (!x) return PyErr_Format(PyExc_ValueError, "bind: null address");
  api.append = reinterpret_cast<decltype(api.append)>(p[0]);
  api.attention_workspace = reinterpret_cast<decltype(api.attention_workspace)>(p[1]);
  api.attention = reinterpret_cast<decltype(api.attention)>(p[2]);
  api.verify = reinterpret_cast<decltype(api.verify)>(p[3]);
  Py_RETURN_NONE;
}

template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(F));
}

PyMethodDef methods[] = {{"paged_rope_append", fast<append>(), METH_FASTCALL, nullptr},
                         {"prefix_attention", fast<attention>(), METH_FASTCALL, nullptr},
                         {"verify_drafts", fast<verify>(), METH_FASTCALL, nullptr},
                         {"bind", bind, METH_VARARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_batch_ops", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__batch_ops(void) { return PyModule_Create(&module); }
