// torch_ops.cpp -- Python binding of the decoder-serving operators for CUDA torch tensors
// (module spinn_b200._torch_ops, wrapped by spinn_b200/runtime.py).
//
// A decoding step makes a dozen of these calls of a few microseconds each, so the arguments are
// taken apart here: reading sizes, strides and pointers through Python and ctypes cost 8 to 15 us
// a call, several times what the smallest kernels run.  Checks of types, shapes and devices raise
// TypeError / ValueError; everything else is left to the C entry points of libspinn_cuda.so,
// whose errors come back as SpinnCudaError.  Work goes to torch's current stream of the tensors'
// device; workspaces come from torch's caching allocator on that stream, so that a captured call
// has its workspace in its graph's pool.
#include <Python.h>

#include <algorithm>
#include <cmath>
#include <cstring>
#include <string>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/spinn_cuda.h"

namespace {

PyObject* g_error = nullptr;  // spinn_b200.lib.SpinnCudaError

struct Refused {};  // a Python exception is set

[[noreturn]] void refuse(PyObject* type, const char* op, const std::string& what) {
  PyErr_SetString(type, (std::string(op) + ": " + what).c_str());
  throw Refused();
}

std::string shape_of(const at::Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

const at::Tensor& tensor(PyObject* o, const char* op, const char* what) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, op, std::string(what) + " must be a torch tensor");
  return THPVariable_Unpack(o);
}
// None becomes a null pointer
const at::Tensor* maybe(PyObject* o, const char* op, const char* what) {
  return o == Py_None ? nullptr : &tensor(o, op, what);
}

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat:
      return SPINN_CUDA_FP32;
    case at::kHalf:
      return SPINN_CUDA_FP16;
    case at::kBFloat16:
      return SPINN_CUDA_BF16;
    default:
      return 0;
  }
}

int32_t narrow(int64_t v, const char* op, const char* what) {
  if (v < 0 || v > 0x7fffffff) refuse(PyExc_ValueError, op, std::string(what) + " of " + std::to_string(v) + " is out of range");
  return (int32_t)v;
}

bool rows_contiguous(const at::Tensor& t) { return t.stride(-1) == 1 || t.size(-1) <= 1; }

// The device that every tensor of a call lies on.
struct Device {
  const char* op;
  int index = -1;
  explicit Device(const char* o) : op(o) {}
  void add(const at::Tensor& t) {
    if (!t.is_cuda()) refuse(PyExc_TypeError, op, "CUDA tensors are required");
    const int d = t.get_device();
    if (index < 0) index = d;
    if (d != index) refuse(PyExc_ValueError, op, "tensors on different devices");
  }
  void add(const at::Tensor* t) {
    if (t) add(*t);
  }
};

void raise_status(int rc, const char* where) {
  if (rc >= 0) return;
  PyObject* e = PyObject_CallFunction(g_error, "iss", rc, where, spinn_cuda_last_error());
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Refused();
}

// Workspace from the caching allocator, returned to it when the call has been queued (its next
// user on the same stream runs after this call's kernels).
struct Workspace {
  void* p = nullptr;
  Workspace(size_t bytes, cudaStream_t st) {
    if (bytes) p = c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(bytes, st);
  }
  ~Workspace() {
    if (p) c10::cuda::CUDACachingAllocator::raw_delete(p);
  }
  Workspace(const Workspace&) = delete;
  Workspace& operator=(const Workspace&) = delete;
};

SpinnCudaCache cache_desc(const at::Tensor& k, const at::Tensor& v, const char* op) {
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides() || k.scalar_type() != v.scalar_type())
    refuse(PyExc_ValueError, op, "k_cache and v_cache must be [pages, page_size, heads, dim] of one shape, layout and type");
  SpinnCudaCache c;
  c.dtype = dtype_code(k.scalar_type());
  if (!c.dtype) refuse(PyExc_TypeError, op, "caches must be float32, float16 or bfloat16");
  if (!rows_contiguous(k)) refuse(PyExc_ValueError, op, "the cache's last dimension must be contiguous");
  c.k = k.data_ptr();
  c.v = v.data_ptr();
  c.page_stride = k.stride(0);
  c.token_stride = k.stride(1);
  c.head_stride = k.stride(2);
  c.num_pages = narrow(k.size(0), op, "a page count");
  c.page_size = narrow(k.size(1), op, "a page size");
  c.kv_heads = narrow(k.size(2), op, "a head count");
  c.head_dim = narrow(k.size(3), op, "a head size");
  c.reserved = 0;
  return c;
}

SpinnCudaPageTable table_desc(const at::Tensor& pages, const at::Tensor& lens, const char* op) {
  if (pages.scalar_type() != at::kInt || lens.scalar_type() != at::kInt)
    refuse(PyExc_TypeError, op, "page_table and lens must be int32");
  if (pages.dim() != 2 || lens.dim() != 1 || lens.size(0) != pages.size(0) || !lens.is_contiguous() ||
      !rows_contiguous(pages))
    refuse(PyExc_ValueError, op, "page_table must be [seqs, max_pages] with contiguous rows, lens [seqs]");
  SpinnCudaPageTable t;
  t.pages = static_cast<const int32_t*>(pages.data_ptr());
  t.lens = static_cast<const int32_t*>(lens.data_ptr());
  t.row_stride = pages.stride(0);
  t.seqs = narrow(pages.size(0), op, "a sequence count");
  t.max_pages = narrow(pages.size(1), op, "a table width");
  return t;
}

// A [n, heads, dim] tensor of the cache's type.
void check_rows(const at::Tensor& t, const at::Tensor& cache, int64_t n, int64_t heads, const char* op, const char* what) {
  if (t.scalar_type() != cache.scalar_type()) refuse(PyExc_TypeError, op, std::string(what) + " must have the cache's type");
  if (t.dim() != 3 || t.size(0) != n || t.size(1) != heads || t.size(2) != cache.size(3) || !rows_contiguous(t))
    refuse(PyExc_ValueError, op, std::string(what) + " must be [" + std::to_string(n) + ", " + std::to_string(heads) + ", " +
                                     std::to_string(cache.size(3)) + "] with contiguous rows, not " + shape_of(t));
}

void check_weights(const at::Tensor& t, int64_t seqs, int64_t heads, const char* op, const char* what) {
  if (t.scalar_type() != at::kFloat) refuse(PyExc_TypeError, op, std::string(what) + " must be float32");
  if (t.dim() != 3 || t.size(0) != seqs || t.size(1) != heads || !rows_contiguous(t))
    refuse(PyExc_ValueError, op, std::string(what) + " must be [" + std::to_string(seqs) + ", " + std::to_string(heads) +
                                     ", length] with contiguous rows, not " + shape_of(t));
}

void check_count(Py_ssize_t n, Py_ssize_t want, const char* op) {
  if (n != want) refuse(PyExc_TypeError, op, std::to_string(want) + " arguments expected");
}

int to_int(PyObject* o, const char* op, const char* what) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused();
  if (v < -0x80000000ll || v > 0x7fffffffll) refuse(PyExc_ValueError, op, std::string(what) + " is out of range");
  return (int)v;
}

// linear(x, w, y, bias, residual, act code)
void linear(PyObject* const* a, Py_ssize_t n) {
  const char* op = "linear";
  check_count(n, 6, op);
  const at::Tensor &x = tensor(a[0], op, "x"), &w = tensor(a[1], op, "w"), &y = tensor(a[2], op, "y");
  const at::Tensor *bias = maybe(a[3], op, "bias"), *res = maybe(a[4], op, "residual");
  const at::ScalarType dt = x.scalar_type();
  if (w.scalar_type() != dt || y.scalar_type() != dt || (dt != at::kHalf && dt != at::kBFloat16))
    refuse(PyExc_TypeError, op, "x, w and y must all be float16 or all bfloat16");
  if (x.dim() != 2 || w.dim() != 2 || y.dim() != 2 || x.size(1) != w.size(1) || y.size(0) != x.size(0) ||
      y.size(1) != w.size(0))
    refuse(PyExc_ValueError, op, "x must be [m, k], w [n, k] and y [m, n], not " + shape_of(x) + ", " + shape_of(w) + " and " +
                                     shape_of(y));
  if (bias && (bias->scalar_type() != dt || bias->dim() != 1 || bias->size(0) != w.size(0) || !rows_contiguous(*bias)))
    refuse(PyExc_ValueError, op, "bias must be a contiguous [n] of x's type");
  if (res && (res->scalar_type() != dt || res->sizes() != y.sizes()))
    refuse(PyExc_ValueError, op, "residual must have y's shape and type");
  if (!rows_contiguous(x) || !rows_contiguous(w) || !rows_contiguous(y) || (res && !rows_contiguous(*res)))
    refuse(PyExc_ValueError, op, "rows must be contiguous");
  Device dev(op);
  dev.add(x);
  dev.add(w);
  dev.add(y);
  dev.add(bias);
  dev.add(res);
  if (x.size(0) == 0) return;
  SpinnCudaLinear l;
  l.x = x.data_ptr();
  l.w = w.data_ptr();
  l.bias = bias ? bias->data_ptr() : nullptr;
  l.residual = res ? res->data_ptr() : nullptr;
  l.y = y.data_ptr();
  l.m = narrow(x.size(0), op, "m");
  l.n = narrow(w.size(0), op, "n");
  l.k = narrow(x.size(1), op, "k");
  // the stride of a single row means nothing
  l.x_stride = l.m > 1 ? x.stride(0) : l.k;
  l.w_stride = l.n > 1 ? w.stride(0) : l.k;
  l.y_stride = l.m > 1 ? y.stride(0) : l.n;
  l.residual_stride = res && l.m > 1 ? res->stride(0) : l.n;
  l.dtype = dtype_code(dt);
  l.act = to_int(a[5], op, "act");
  l.reserved = 0;
  const c10::cuda::OptionalCUDAGuard guard(x.device());
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index).stream();
  const size_t bytes = spinn_cuda_linear_workspace(&l);
  Workspace ws(bytes, st);
  raise_status(spinn_cuda_linear(&l, ws.p, bytes, st), "spinn_cuda_linear");
}

// cache_append(k, v, k_cache, v_cache, page_table, lens, starts)
void cache_append(PyObject* const* a, Py_ssize_t n) {
  const char* op = "cache_append";
  check_count(n, 7, op);
  const at::Tensor &k = tensor(a[0], op, "k"), &v = tensor(a[1], op, "v"), &kc = tensor(a[2], op, "k_cache"),
                   &vc = tensor(a[3], op, "v_cache"), &table = tensor(a[4], op, "page_table"),
                   &lens = tensor(a[5], op, "lens");
  const at::Tensor* starts = maybe(a[6], op, "starts");
  const SpinnCudaCache c = cache_desc(kc, vc, op);
  const SpinnCudaPageTable t = table_desc(table, lens, op);
  if (k.dim() != 3) refuse(PyExc_ValueError, op, "k must be [tokens, heads, dim]");
  const int64_t tokens = k.size(0);
  check_rows(k, kc, tokens, kc.size(2), op, "k");
  check_rows(v, kc, tokens, kc.size(2), op, "v");
  if (starts) {
    if (starts->scalar_type() != at::kInt) refuse(PyExc_TypeError, op, "starts must be int32");
    if (starts->dim() != 1 || starts->size(0) != lens.size(0) + 1 || !starts->is_contiguous())
      refuse(PyExc_ValueError, op, "starts must be [seqs + 1]");
  } else if (tokens != lens.size(0)) {
    refuse(PyExc_ValueError, op,
           std::to_string(tokens) + " rows for " + std::to_string(lens.size(0)) + " sequences without starts");
  }
  Device dev(op);
  dev.add(kc);
  dev.add(vc);
  dev.add(k);
  dev.add(v);
  dev.add(table);
  dev.add(lens);
  dev.add(starts);
  if (tokens == 0) return;
  SpinnCudaAppend r;
  r.k = k.data_ptr();
  r.v = v.data_ptr();
  r.k_token_stride = k.stride(0);
  r.k_head_stride = k.stride(1);
  r.v_token_stride = v.stride(0);
  r.v_head_stride = v.stride(1);
  r.starts = starts ? static_cast<const int32_t*>(starts->data_ptr()) : nullptr;
  r.tokens = narrow(tokens, op, "a token count");
  r.reserved = 0;
  const c10::cuda::OptionalCUDAGuard guard(kc.device());
  raise_status(spinn_cuda_cache_append(&c, &t, &r, c10::cuda::getCurrentCUDAStream(dev.index).stream()),
               "spinn_cuda_cache_append");
}

// paged_attention(q, k_cache, v_cache, page_table, lens, y, scale, weights, weights_out)
void paged_attention(PyObject* const* a, Py_ssize_t n) {
  const char* op = "paged_attention";
  check_count(n, 9, op);
  const at::Tensor &q = tensor(a[0], op, "q"), &kc = tensor(a[1], op, "k_cache"), &vc = tensor(a[2], op, "v_cache"),
                   &table = tensor(a[3], op, "page_table"), &lens = tensor(a[4], op, "lens"), &y = tensor(a[5], op, "y");
  const at::Tensor *win = maybe(a[7], op, "weights"), *wout = maybe(a[8], op, "weights_out");
  const SpinnCudaCache c = cache_desc(kc, vc, op);
  const SpinnCudaPageTable t = table_desc(table, lens, op);
  const int64_t seqs = lens.size(0), heads = kc.size(2);
  if (q.dim() != 3) refuse(PyExc_ValueError, op, "q must be [seqs, q_heads, dim]");
  check_rows(q, kc, seqs, q.size(1), op, "q");
  check_rows(y, kc, seqs, q.size(1), op, "y");
  SpinnCudaAttention d;
  std::memset(&d, 0, sizeof(d));
  if (wout) {
    check_weights(*wout, seqs, heads, op, "weights_out");
    int64_t cap = wout->size(2);
    if (win) {
      check_weights(*win, seqs, heads, op, "weights");
      cap = std::min(cap, win->size(2));
    }
    d.weights_capacity = narrow(cap, op, "a length");
  } else if (win) {
    refuse(PyExc_ValueError, op, "weights without weights_out");
  }
  if (a[6] == Py_None) {
    d.scale = (float)(1.0 / std::sqrt((double)std::max<int64_t>(kc.size(3), 1)));
  } else {
    d.scale = (float)PyFloat_AsDouble(a[6]);
    if (PyErr_Occurred()) throw Refused();
  }
  Device dev(op);
  dev.add(kc);
  dev.add(vc);
  dev.add(q);
  dev.add(table);
  dev.add(lens);
  dev.add(y);
  dev.add(win);
  dev.add(wout);
  if (seqs == 0) return;
  d.q = q.data_ptr();
  d.y = y.data_ptr();
  d.q_seq_stride = q.stride(0);
  d.q_head_stride = q.stride(1);
  d.y_seq_stride = y.stride(0);
  d.y_head_stride = y.stride(1);
  d.q_heads = narrow(q.size(1), op, "a head count");
  if (wout) {
    d.weights_out = static_cast<float*>(wout->data_ptr());
    d.wout_seq_stride = wout->stride(0);
    d.wout_head_stride = wout->stride(1);
  }
  if (win) {
    d.weights_in = static_cast<const float*>(win->data_ptr());
    d.win_seq_stride = win->stride(0);
    d.win_head_stride = win->stride(1);
  }
  const c10::cuda::OptionalCUDAGuard guard(kc.device());
  const cudaStream_t st = c10::cuda::getCurrentCUDAStream(dev.index).stream();
  const size_t bytes = spinn_cuda_paged_attention_workspace(&c, &t, &d);
  Workspace ws(bytes, st);
  raise_status(spinn_cuda_paged_attention(&c, &t, &d, ws.p, bytes, st), "spinn_cuda_paged_attention");
}

// cache_evict(k_cache, v_cache, page_table, lens, weights, weights_out, out_table, new_lens, kept, budget, recent)
void cache_evict(PyObject* const* a, Py_ssize_t n) {
  const char* op = "cache_evict";
  check_count(n, 11, op);
  const at::Tensor &kc = tensor(a[0], op, "k_cache"), &vc = tensor(a[1], op, "v_cache"),
                   &table = tensor(a[2], op, "page_table"), &lens = tensor(a[3], op, "lens"),
                   &win = tensor(a[4], op, "weights"), &wout = tensor(a[5], op, "weights_out"),
                   &out = tensor(a[6], op, "out_table"), &new_lens = tensor(a[7], op, "new_lens"),
                   &kept = tensor(a[8], op, "kept");
  const SpinnCudaCache c = cache_desc(kc, vc, op);
  const SpinnCudaPageTable t = table_desc(table, lens, op);
  const int64_t seqs = lens.size(0), heads = kc.size(2);
  SpinnCudaEvict e;
  e.budget = to_int(a[9], op, "budget");
  e.recent = to_int(a[10], op, "recent");
  check_weights(win, seqs, heads, op, "weights");
  check_weights(wout, seqs, heads, op, "weights_out");
  if (out.scalar_type() != at::kInt || new_lens.scalar_type() != at::kInt || kept.scalar_type() != at::kInt)
    refuse(PyExc_TypeError, op, "out_table, new_lens and kept must be int32");
  if (out.dim() != 2 || out.size(0) != seqs || !rows_contiguous(out))
    refuse(PyExc_ValueError, op, "out_table must be [seqs, max_pages] with contiguous rows");
  if (new_lens.dim() != 1 || new_lens.size(0) != seqs || !new_lens.is_contiguous())
    refuse(PyExc_ValueError, op, "new_lens must be [seqs]");
  if (kept.dim() != 3 || kept.size(0) != seqs || kept.size(1) != heads || kept.size(2) != e.budget || !kept.is_contiguous())
    refuse(PyExc_ValueError, op, "kept must be a contiguous [seqs, heads, budget], not " + shape_of(kept));
  Device dev(op);
  for (const at::Tensor* x : {&kc, &vc, &table, &lens, &win, &wout, &out, &new_lens, &kept}) dev.add(*x);
  if (seqs == 0) return;
  e.weights_in = static_cast<const float*>(win.data_ptr());
  e.weights_out = static_cast<float*>(wout.data_ptr());
  e.win_seq_stride = win.stride(0);
  e.win_head_stride = win.stride(1);
  e.wout_seq_stride = wout.stride(0);
  e.wout_head_stride = wout.stride(1);
  e.out_pages = static_cast<const int32_t*>(out.data_ptr());
  e.out_row_stride = out.stride(0);
  e.out_max_pages = narrow(out.size(1), op, "a table width");
  e.weights_capacity = narrow(std::min(win.size(2), wout.size(2)), op, "a length");
  e.new_lens = static_cast<int32_t*>(new_lens.data_ptr());
  e.kept = static_cast<int32_t*>(kept.data_ptr());
  const c10::cuda::OptionalCUDAGuard guard(kc.device());
  raise_status(spinn_cuda_cache_evict(&c, &t, &e, c10::cuda::getCurrentCUDAStream(dev.index).stream()),
               "spinn_cuda_cache_evict");
}

// No C++ exception leaves the module.
template <void (*F)(PyObject* const*, Py_ssize_t)>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  try {
    F(args, n);
    Py_RETURN_NONE;
  } catch (const Refused&) {
  } catch (const std::exception& e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

template <void (*F)(PyObject* const*, Py_ssize_t)>
constexpr PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F>));
}

PyMethodDef g_methods[] = {
    {"linear", fast<linear>(), METH_FASTCALL, nullptr},
    {"cache_append", fast<cache_append>(), METH_FASTCALL, nullptr},
    {"paged_attention", fast<paged_attention>(), METH_FASTCALL, nullptr},
    {"cache_evict", fast<cache_evict>(), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) {
  PyObject* lib = PyImport_ImportModule("spinn_b200.lib");
  if (!lib) return nullptr;
  g_error = PyObject_GetAttrString(lib, "SpinnCudaError");
  Py_DECREF(lib);
  return g_error ? PyModule_Create(&g_module) : nullptr;
}
