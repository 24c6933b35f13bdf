// sequence.cpp - the tensor side of the packed and paged operators' Python face
// (dinov3_b200/sequence.py): reads torch tensors' types, shapes and strides without a Python call
// each, checks them against one another, fills the argument structs of dinov3_kernels.h and calls
// the library. The library itself knows no torch types: its entry points come in by address.
//
// A call's host time is what bounds a decoder's smallest steps: checked and packed in Python these
// calls took 19 to 26 us each, as long as a dozen launches.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <sstream>
#include <string>

#include "dinov3_kernels.h"

namespace {

int (*packed_fn)(const dv3k_packed_attention *, void *);
int (*append_fn)(const dv3k_rope_append_args *, void *);
int (*paged_fn)(const dv3k_paged_attention *, void *);
size_t (*packed_workspace_fn)(const dv3k_packed_attention *);
size_t (*paged_workspace_fn)(const dv3k_paged_attention *);
PyObject *refuse_cb;  // refuse_cb(message) raises
PyObject *check_cb;   // check_cb(status) raises the library's message

// Thrown where a tensor does not fit; becomes refuse_cb(message).
struct Refused {
  std::string message;
};
template <class... A>
[[noreturn]] void refuse(const A &...a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused{s.str()};
}
// A Python error is already set.
struct Raised {};

const at::Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) refuse(name, " must be a tensor");
  return THPVariable_Unpack(o);
}

void no_gradient(const at::Tensor &t, const char *name) {
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse(name, " requires a gradient, which this operator does not compute");
  if (t._fw_grad(0).defined()) refuse(name, " carries a tangent, which this operator does not propagate");
}

uint32_t first(const at::Tensor &t, const char *name) {
  const auto type = t.scalar_type();
  if (!t.is_cuda() || (type != at::kHalf && type != at::kBFloat16))
    refuse(name, " must be a float16 or bfloat16 CUDA tensor: ", t.toString(), " on ", t.device());
  return type == at::kHalf ? DV3K_F16 : DV3K_BF16;
}

uint32_t size32(int64_t n, const char *name) {
  if (n < 0 || n > 0x7fffffff) refuse(name, " is too large: ", n);
  return static_cast<uint32_t>(n);
}

void rows(const at::Tensor &t, const char *name, const at::Tensor &like) {
  if (t.scalar_type() != like.scalar_type() || t.device() != like.device())
    refuse(name, " must have the type and device of the call's other rows: ", t.toString(), " on ", t.device());
  if (t.layout() != at::kStrided || t.dim() != 3 || (t.size(2) > 1 && t.stride(2) != 1))
    refuse(name, " must be [rows, heads, dim] with a contiguous dim: ", t.sizes(), ", strides ", t.strides());
  size32(t.size(0), name);
  size32(t.size(1), name);
  no_gradient(t, name);
}

void ints(const at::Tensor &t, const char *name, const at::Tensor &like, int64_t dims) {
  if (t.scalar_type() != at::kInt || t.device() != like.device() || t.dim() != dims)
    refuse(name, " must be int32 with ", dims, " dimension(s) on ", like.device(), ": ", t.toString(), " ", t.sizes());
  if (t.size(dims - 1) > 1 && t.stride(dims - 1) != 1) refuse(name, " must be contiguous");
  size32(t.size(0), name);
}

void cache(const at::Tensor &k, const at::Tensor &v, const at::Tensor &like, int64_t heads, int64_t dim) {
  const at::Tensor *both[2] = {&k, &v};
  const char *names[2] = {"k_cache", "v_cache"};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor &t = *both[i];
    if (t.scalar_type() != like.scalar_type() || t.device() != like.device())
      refuse(names[i], " must have the type and device of the rows: ", t.toString(), " on ", t.device());
    if (t.dim() != 4 || t.size(1) != heads || t.size(3) != dim || t.sizes() != k.sizes())
      refuse(names[i], " must be [pages, ", heads, ", page_size, ", dim, "], both alike: ", t.sizes());
    const int64_t page = t.size(2);
    if (t.numel() > 0 && ((dim > 1 && t.stride(3) != 1) || (page > 1 && t.stride(2) != dim) ||
                          (heads > 1 && t.stride(1) != page * dim)))
      refuse(names[i], " must be contiguous within a page: strides ", t.strides());
    size32(t.size(0), names[i]);
    size32(page, "page_size");
    no_gradient(t, names[i]);
  }
}

// Address of an optional contiguous tensor; null for None.
void *optional(PyObject *o, const char *name, const at::Tensor &like, at::ScalarType type,
               at::IntArrayRef shape) {
  if (o == Py_None) return nullptr;
  const at::Tensor &t = tensor(o, name);
  if (t.scalar_type() != type || t.device() != like.device() || !t.is_contiguous() || t.sizes() != shape)
    refuse(name, " must be a contiguous ", at::toString(type), " tensor of shape ", shape, " on ", like.device());
  no_gradient(t, name);
  return t.data_ptr();
}

uint32_t *status_of(PyObject *o, const at::Tensor &like) {
  if (o == Py_None) return nullptr;
  const at::Tensor &t = tensor(o, "status");
  if (t.scalar_type() != at::kInt || t.device() != like.device() || !t.is_contiguous() || t.numel() < 2)
    refuse("status must be a contiguous int32 tensor of two words on ", like.device());
  return static_cast<uint32_t *>(t.data_ptr());
}

// Counts a given tensor as written, so that autograd notices where it had kept it. Inference tensors
// have no counter.
void written(const at::Tensor &t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject *o) {
  if (o != Py_None) written(THPVariable_Unpack(o));
}

// A new tensor from torch's allocator, without the dispatcher's way to it.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor &like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}

at::Tensor output(PyObject *o, const char *name, const at::Tensor &like, const at::Tensor &q) {
  if (o == Py_None) return fresh(q.sizes(), q.scalar_type(), q);
  const at::Tensor &t = tensor(o, name);
  rows(t, name, like);
  if (t.sizes() != q.sizes()) refuse(name, " must have shape ", q.sizes(), ": ", t.sizes());
  return t;
}

float scale_of(PyObject *o, int64_t dim) {
  if (o == Py_None) return 1.f / std::sqrt(static_cast<float>(dim));
  const double s = PyFloat_AsDouble(o);
  if (s == -1.0 && PyErr_Occurred()) throw Raised{};
  return static_cast<float>(s);
}

PyObject *result(PyObject *given, at::Tensor &&t) {
  if (given != Py_None) {
    Py_INCREF(given);
    return given;
  }
  return THPVariable_Wrap(std::move(t));
}

// The call's scratch: the given tensor, or a new one of the size it needs, which the caller holds until
// the launch is out (torch's allocator then hands it on in stream order only).
template <class Args>
at::Tensor scratch_of(PyObject *given, Args &p, size_t (*need_of)(const Args *), const at::Tensor &q) {
  at::Tensor w;
  if (given != Py_None) {
    w = tensor(given, "workspace");
    if (w.scalar_type() != at::kByte || w.device() != q.device() || !w.is_contiguous())
      refuse("workspace must be a contiguous uint8 tensor on ", q.device());
  } else if (const size_t need = need_of(&p)) {
    w = fresh({static_cast<int64_t>(need)}, at::kByte, q);
  } else {
    return w;
  }
  p.workspace = w.data_ptr();
  p.workspace_bytes = static_cast<uint64_t>(w.numel());
  return w;
}

// Runs `f` on the tensors' device and its current stream; a nonzero status raises.
template <class F>
void on_device(const at::Tensor &t, F &&f) {
  const c10::cuda::CUDAGuard guard(t.device());
  const int rc = f(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
  if (rc == 0) return;
  PyObject *r = PyObject_CallFunction(check_cb, "i", rc);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "the library refused the call");
  throw Raised{};
}

// Python exceptions for everything that `f` throws.
template <class F>
PyObject *guarded(Py_ssize_t got, Py_ssize_t want, F &&f) {
  HANDLE_TH_ERRORS
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
    return nullptr;
  }
  try {
    return f();
  } catch (const Refused &e) {
    PyObject *r = PyObject_CallFunction(refuse_cb, "s", e.message.c_str());
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.message.c_str());
    return nullptr;
  } catch (const Raised &) {
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// (q, k, v, cu_q, cu_k, causal, scale, out, lse, workspace, status)
PyObject *attention_packed(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 11, [&] {
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
    const at::Tensor &cu_q = tensor(a[3], "cu_q"), &cu_k = a[4] == Py_None ? cu_q : tensor(a[4], "cu_k");
    dv3k_packed_attention p = {};
    p.dtype = first(q, "q");
    rows(q, "q", q);
    rows(k, "k", q);
    rows(v, "v", q);
    ints(cu_q, "cu_q", q, 1);
    ints(cu_k, "cu_k", q, 1);
    if (k.size(2) != q.size(2) || v.sizes() != k.sizes())
      refuse("k and v must be [rows, kv_heads, ", q.size(2), "] alike: ", k.sizes(), ", ", v.sizes());
    if (cu_q.size(0) < 1 || cu_k.size(0) != cu_q.size(0))
      refuse("cu_q and cu_k must have the same n_seq + 1 entries");
    const int causal = PyObject_IsTrue(a[5]);
    if (causal < 0) throw Raised{};
    p.scale = scale_of(a[6], q.size(2));
    p.lse = static_cast<float *>(optional(a[8], "lse", q, at::kFloat, {q.size(0), q.size(1)}));
    p.status = status_of(a[10], q);
    at::Tensor out = output(a[7], "out", q, q);
    p.q = q.data_ptr();
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.out = out.data_ptr();
    p.cu_q = static_cast<const int32_t *>(cu_q.data_ptr());
    p.cu_k = static_cast<const int32_t *>(cu_k.data_ptr());
    p.q_token = q.stride(0);
    p.q_head = q.stride(1);
    p.k_token = k.stride(0);
    p.k_head = k.stride(1);
    p.v_token = v.stride(0);
    p.v_head = v.stride(1);
    p.out_token = out.stride(0);
    p.out_head = out.stride(1);
    p.n_seq = static_cast<uint32_t>(cu_q.size(0) - 1);
    p.total_q = static_cast<uint32_t>(q.size(0));
    p.total_k = static_cast<uint32_t>(k.size(0));
    p.q_heads = static_cast<uint32_t>(q.size(1));
    p.kv_heads = static_cast<uint32_t>(k.size(1));
    p.head_dim = size32(q.size(2), "dim");
    p.causal = static_cast<uint32_t>(causal);
    at::Tensor scratch;
    on_device(q, [&](void *stream) {
      scratch = scratch_of(a[9], p, packed_workspace_fn, q);
      return packed_fn(&p, stream);
    });
    written(a[7]);
    written(a[8]);
    return result(a[7], std::move(out));
  });
}

// (q, k, v, k_cache, v_cache, page_table, lens, cos, sin, cu_new, q_out, status)
PyObject *rope_append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 12, [&]() -> PyObject * {
    const at::Tensor &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
    const at::Tensor &k_cache = tensor(a[3], "k_cache"), &v_cache = tensor(a[4], "v_cache");
    const at::Tensor &table = tensor(a[5], "page_table"), &lens = tensor(a[6], "lens");
    dv3k_rope_append_args p = {};
    p.dtype = first(k, "k");
    rows(k, "k", k);
    rows(v, "v", k);
    if (v.sizes() != k.sizes()) refuse("k and v must have the same shape: ", k.sizes(), ", ", v.sizes());
    cache(k_cache, v_cache, k, k.size(1), k.size(2));
    ints(table, "page_table", k, 2);
    ints(lens, "lens", k, 1);
    if (lens.size(0) != table.size(0)) refuse("lens must have one entry for each row of page_table");
    if (a[9] != Py_None) {
      const at::Tensor &cu = tensor(a[9], "cu_new");
      ints(cu, "cu_new", k, 1);
      if (cu.size(0) != lens.size(0) + 1) refuse("cu_new must have n_seq + 1 entries");
      p.cu_new = static_cast<const int32_t *>(cu.data_ptr());
    }
    if ((a[7] == Py_None) != (a[8] == Py_None)) refuse("cos and sin go together");
    if (a[0] == Py_None && a[10] != Py_None) refuse("q_out goes with q");
    if (a[7] != Py_None) {
      const at::Tensor &cos = tensor(a[7], "cos");
      if (cos.dim() != 2) refuse("cos must be [positions, rot_dim / 2]");
      p.cos = static_cast<const float *>(optional(a[7], "cos", k, at::kFloat, cos.sizes()));
      p.sin = static_cast<const float *>(optional(a[8], "sin", k, at::kFloat, cos.sizes()));
      p.positions = size32(cos.size(0), "positions");
      p.rot_dim = size32(2 * cos.size(1), "rot_dim");
    }
    p.status = status_of(a[11], k);
    at::Tensor out;
    if (a[0] != Py_None) {
      const at::Tensor &q = tensor(a[0], "q");
      rows(q, "q", k);
      if (q.size(0) != k.size(0) || q.size(2) != k.size(2))
        refuse("q must be [", k.size(0), ", q_heads, ", k.size(2), "]: ", q.sizes());
      out = output(a[10], "q_out", k, q);
      p.q = q.data_ptr();
      p.q_out = out.data_ptr();
      p.q_token = q.stride(0);
      p.q_head = q.stride(1);
      p.q_out_token = out.stride(0);
      p.q_out_head = out.stride(1);
      p.q_heads = static_cast<uint32_t>(q.size(1));
    }
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.k_cache = k_cache.data_ptr();
    p.v_cache = v_cache.data_ptr();
    p.lens = static_cast<const int32_t *>(lens.data_ptr());
    p.page_table = static_cast<const int32_t *>(table.data_ptr());
    p.k_token = k.stride(0);
    p.k_head = k.stride(1);
    p.v_token = v.stride(0);
    p.v_head = v.stride(1);
    p.k_page = k_cache.stride(0);
    p.v_page = v_cache.stride(0);
    p.table_stride = table.stride(0);
    p.n_seq = static_cast<uint32_t>(lens.size(0));
    p.total = static_cast<uint32_t>(k.size(0));
    p.max_pages = size32(table.size(1), "page_table");
    p.n_pages = static_cast<uint32_t>(k_cache.size(0));
    p.page_size = static_cast<uint32_t>(k_cache.size(2));
    p.kv_heads = static_cast<uint32_t>(k.size(1));
    p.head_dim = size32(k.size(2), "dim");
    on_device(k, [&](void *stream) { return append_fn(&p, stream); });
    written(k_cache);
    written(v_cache);
    written(a[10]);
    if (a[0] == Py_None) Py_RETURN_NONE;
    return result(a[10], std::move(out));
  });
}

// (q, k_cache, v_cache, page_table, lens, max_len, scale, out, lse, workspace, status)
PyObject *attention_paged(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return guarded(n, 11, [&] {
    const at::Tensor &q = tensor(a[0], "q"), &k_cache = tensor(a[1], "k_cache"), &v_cache = tensor(a[2], "v_cache");
    const at::Tensor &table = tensor(a[3], "page_table"), &lens = tensor(a[4], "lens");
    dv3k_paged_attention p = {};
    p.dtype = first(q, "q");
    rows(q, "q", q);
    cache(k_cache, v_cache, q, k_cache.dim() == 4 ? k_cache.size(1) : 0, q.size(2));
    ints(table, "page_table", q, 2);
    ints(lens, "lens", q, 1);
    if (table.size(0) != q.size(0) || lens.size(0) != q.size(0))
      refuse("page_table and lens must have one entry for each row of q");
    p.max_pages = size32(table.size(1), "page_table");
    p.page_size = static_cast<uint32_t>(k_cache.size(2));
    int64_t max_len = static_cast<int64_t>(p.max_pages) * p.page_size;
    if (a[5] != Py_None) {
      const int64_t given = PyLong_AsLongLong(a[5]);
      if (given == -1 && PyErr_Occurred()) throw Raised{};
      if (given < 0) refuse("max_len must not be negative: ", given);
      max_len = std::min(max_len, given);
    }
    p.max_len = static_cast<uint32_t>(std::min<int64_t>(max_len, 0x7fffffff));
    p.scale = scale_of(a[6], q.size(2));
    p.lse = static_cast<float *>(optional(a[8], "lse", q, at::kFloat, {q.size(0), q.size(1)}));
    p.status = status_of(a[10], q);
    at::Tensor out = output(a[7], "out", q, q);
    p.q = q.data_ptr();
    p.k_cache = k_cache.data_ptr();
    p.v_cache = v_cache.data_ptr();
    p.out = out.data_ptr();
    p.lens = static_cast<const int32_t *>(lens.data_ptr());
    p.page_table = static_cast<const int32_t *>(table.data_ptr());
    p.q_seq = q.stride(0);
    p.q_head = q.stride(1);
    p.out_seq = out.stride(0);
    p.out_head = out.stride(1);
    p.k_page = k_cache.stride(0);
    p.v_page = v_cache.stride(0);
    p.table_stride = table.stride(0);
    p.n_seq = static_cast<uint32_t>(q.size(0));
    p.n_pages = static_cast<uint32_t>(k_cache.size(0));
    p.q_heads = static_cast<uint32_t>(q.size(1));
    p.kv_heads = static_cast<uint32_t>(k_cache.size(1));
    p.head_dim = size32(q.size(2), "dim");
    at::Tensor scratch;
    on_device(q, [&](void *stream) {
      scratch = scratch_of(a[9], p, paged_workspace_fn, q);
      return paged_fn(&p, stream);
    });
    written(a[7]);
    written(a[8]);
    return result(a[7], std::move(out));
  });
}

// bind(packed, its workspace, append, paged, its workspace, refuse, check): the entry points' addresses,
// and what raises.
PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long f[5];
  PyObject *refuse_to, *check_to;
  if (!PyArg_ParseTuple(args, "KKKKKOO", &f[0], &f[1], &f[2], &f[3], &f[4], &refuse_to, &check_to)) return nullptr;
  packed_fn = reinterpret_cast<decltype(packed_fn)>(f[0]);
  packed_workspace_fn = reinterpret_cast<decltype(packed_workspace_fn)>(f[1]);
  append_fn = reinterpret_cast<decltype(append_fn)>(f[2]);
  paged_fn = reinterpret_cast<decltype(paged_fn)>(f[3]);
  paged_workspace_fn = reinterpret_cast<decltype(paged_workspace_fn)>(f[4]);
  Py_INCREF(refuse_to);
  Py_INCREF(check_to);
  Py_XSETREF(refuse_cb, refuse_to);
  Py_XSETREF(check_cb, check_to);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"attention_packed", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention_packed)), METH_FASTCALL, nullptr},
    {"rope_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_append)), METH_FASTCALL, nullptr},
    {"attention_paged", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attention_paged)), METH_FASTCALL, nullptr},
    {"bind", bind, METH_VARARGS, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_sequence", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__sequence() { return PyModule_Create(&module); }
