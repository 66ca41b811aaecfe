// paged_ext.cpp -- the paged KV-cache operators on torch tensors (the binding
// behind rcutetts_b200/paged.py): argument checks, outputs and workspaces from
// torch's allocator, the tensors' device and its current stream, and the call
// of the C ABI.  A call's checks read some thirty properties of tensors; from
// Python that takes longer than the small kernels do (a decode step's
// attention 14.6 us a call instead of 8, its append 9 instead of 3.5 to 4.3).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/cutetts_b200.h"

namespace {

PyObject* g_error = nullptr;  // rcutetts_b200._lib.CttsError

// What a ValueError says.
struct BadArgument : std::runtime_error {
  using std::runtime_error::runtime_error;
};
void need(bool ok, const char* what) {
  if (!ok) throw BadArgument(what);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw BadArgument(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

int type_of(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat ? CTTS_F32 : (t.scalar_type() == at::kBFloat16 ? CTTS_BF16 : -1);
}

int cuda_index(const at::Tensor& t) {
  need(t.is_cuda(), "the paged operators run on CUDA tensors");
  return t.get_device();
}

// a contiguous int32 tensor on the device
const int* ints(const at::Tensor& t, int dev, int64_t at_least, const char* what) {
  need(t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == dev && t.is_contiguous() && t.numel() >= at_least, what);
  return t.const_data_ptr<int>();
}

ctts_paged_kv pool(const at::Tensor& k, const at::Tensor& v, int dev) {
  need(k.dim() == 4 && k.sizes() == v.sizes() && k.strides() == v.strides() && k.scalar_type() == v.scalar_type() && k.is_cuda() &&
           k.get_device() == dev && v.is_cuda() && v.get_device() == dev,
       "the pools are two [pages, page_size, kv heads, head dim] tensors of one type and layout on the rows' device");
  ctts_paged_kv p{};
  p.dtype = type_of(k);
  need(p.dtype >= 0, "a cache is float32 or bf16");
  need(k.stride(3) == 1, "the head dim of a pool is contiguous");
  need(k.size(0) <= INT_MAX && k.size(1) <= INT_MAX && k.size(2) <= INT_MAX && k.size(3) <= INT_MAX, "pool too large");
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.n_pages = (int)k.size(0);
  p.page_size = (int)k.size(1);
  p.n_kv_heads = (int)k.size(2);
  p.head_dim = (int)k.size(3);
  // the stride of a dimension of one carries no meaning: one that passes the checks
  p.page_stride = p.n_pages > 1 ? k.stride(0) : (int64_t)p.page_size * p.n_kv_heads * p.head_dim;
  p.token_stride = k.stride(1);
  p.head_stride = p.n_kv_heads > 1 ? k.stride(2) : p.head_dim;
  return p;
}

// row stride of block tables [batch, pages]
int64_t table_ld(const at::Tensor& t, int64_t batch, int dev) {
  need(t.scalar_type() == at::kInt && t.is_cuda() && t.get_device() == dev && t.dim() == 2 && t.size(0) == batch &&
           t.size(1) <= INT_MAX && (t.size(1) <= 1 || t.stride(1) == 1),
       "block_tables must be an int32 [batch, pages] tensor with contiguous rows on the other tensors' device");
  return batch > 1 ? t.stride(0) : std::max(t.stride(0), t.size(1));
}

// [rows, heads, dim] with whole rows: its row stride
int64_t rows_ld(const at::Tensor& t, int64_t rows, int64_t heads, int64_t hd, const char* what) {
  need(t.dim() == 3 && t.size(0) == rows && t.size(1) == heads && t.size(2) == hd && t.stride(2) == 1 && (heads <= 1 || t.stride(1) == hd), what);
  return rows > 1 ? t.stride(0) : heads * hd;
}

int to_int(int64_t v, const char* what) {
  need(v >= INT_MIN && v <= INT_MAX, what);
  return (int)v;
}
int int_arg(PyObject* o, const char* what) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return to_int(v, what);
}
double float_arg(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

// The stream of a call -- the device's current one, or an address or a torch
// stream -- made current on its device until the call returns: outputs and
// workspaces then belong to the stream that uses them.
struct OnStream {
  c10::cuda::OptionalCUDAGuard device;
  c10::cuda::OptionalCUDAStreamGuard guard;
  void* stream;
  OnStream(PyObject* o, int dev) {
    if (dev != c10::cuda::current_device()) device.set_index((c10::DeviceIndex)dev);
    if (o == Py_None) {
      stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
      return;
    }
    if (PyLong_Check(o)) {
      stream = PyLong_AsVoidPtr(o);
    } else {
      PyObject* a = PyObject_GetAttrString(o, "cuda_stream");
      if (!a) throw python_error();
      stream = PyLong_AsVoidPtr(a);
      Py_DECREF(a);
    }
    if (!stream && PyErr_Occurred()) throw python_error();
    guard.reset_stream(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(stream), (c10::DeviceIndex)dev));
  }
};

at::Tensor empty(at::IntArrayRef size, at::ScalarType type, int dev) {
  return at::Tensor(at::detail::empty_cuda(size, type, at::Device(at::kCUDA, (c10::DeviceIndex)dev), std::nullopt));
}

// n entries of t from entry `first` on, as a tensor of their own over its storage
at::Tensor part(const at::Tensor& t, int64_t first, int64_t n) {
  auto impl = c10::make_intrusive<c10::TensorImpl>(c10::Storage(t.storage()), t.key_set(), t.dtype());
  impl->set_storage_offset(first);
  impl->set_sizes_contiguous({n});
  return at::Tensor(std::move(impl));
}

// A call has written to t: what autograd has saved of it is another version.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// A negative status as CttsError(code, message).
void done(int rc) {
  if (rc == CTTS_OK) return;
  PyObject* args = Py_BuildValue("(is)", rc, ctts_last_error());
  if (args) {
    PyErr_SetObject(g_error ? g_error : PyExc_RuntimeError, args);
    Py_DECREF(args);
  }
  throw python_error();
}

template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const BadArgument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (python_error& e) {
    e.restore();
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "paged operator failed");
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// (ctx_lens, new_lens, block_tables, free_pages, free_count, page_size, max_rows, stream)
PyObject* plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 8, "plan takes 8 arguments");
    const at::Tensor &ctx = tensor(a[0], "ctx_lens"), &nw = tensor(a[1], "new_lens"), &tab = tensor(a[2], "block_tables"),
                     &free = tensor(a[3], "free_pages"), &count = tensor(a[4], "free_count");
    const int dev = cuda_index(ctx);
    const char* what = "ctx_lens, new_lens (one entry per request), free_pages and free_count (at least one) must be contiguous int32 tensors on one device";
    ctts_paged_plan p{};
    p.batch = to_int(ctx.numel(), "too many requests");
    p.ctx_lens = ints(ctx, dev, 0, what);
    p.new_lens = ints(nw, dev, 0, what);
    need(nw.numel() == p.batch, what);
    p.free_count = ints(count, dev, 1, what);
    ints(free, dev, 0, what);
    p.free_pages = free.data_ptr<int>();
    p.free_capacity = to_int(free.numel(), "free_pages too long");
    p.table_ld = table_ld(tab, p.batch, dev);
    p.block_tables = tab.data_ptr<int>();
    p.max_pages = (int)tab.size(1);
    p.page_size = int_arg(a[5], "bad page_size");
    p.max_rows = int_arg(a[6], "bad max_rows");
    need(p.max_rows >= 0, "max_rows must not be negative");
    const OnStream on(a[7], dev);
    // one allocation: lengths, offsets, state, positions, slots
    const int64_t b = p.batch, r = p.max_rows;
    const at::Tensor out = empty({2 * b + 5 + 2 * r}, at::kInt, dev);
    p.seq_lens = out.data_ptr<int>();
    p.cu_rows = p.seq_lens + b;
    p.state = p.cu_rows + b + 1;
    p.positions = p.state + 4;
    p.slots = p.positions + r;
    done(ctts_op_paged_plan(&p, on.stream));
    written(tab);
    written(free);
    PyObject* t = PyTuple_New(5);
    if (!t) throw python_error();
    const int64_t first[5] = {0, b, 2 * b + 5, 2 * b + 5 + r, 2 * b + 1}, len[5] = {b, b + 1, r, r, 4};
    for (int i = 0; i < 5; i++) PyTuple_SET_ITEM(t, i, THPVariable_Wrap(part(out, first[i], len[i])));
    return t;
  });
}

// (x, k_pages, v_pages, positions, slots, n_heads, q_norm, k_norm, eps, theta, q type (-1: x's or out's), out, stream)
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 13, "append takes 13 arguments");
    const at::Tensor &x = tensor(a[0], "x"), &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages"), &pos = tensor(a[3], "positions"),
                     &slots = tensor(a[4], "slots");
    const int dev = cuda_index(x);
    ctts_paged_append p{};
    p.kv = pool(k, v, dev);
    p.n_heads = int_arg(a[5], "bad n_heads");
    p.x_dtype = type_of(x);
    const int64_t hd = p.kv.head_dim, width = ((int64_t)p.n_heads + 2 * p.kv.n_kv_heads) * hd;
    need(p.x_dtype >= 0 && x.dim() == 2 && p.n_heads > 0 && x.size(1) == width && x.stride(1) == 1 && x.size(0) <= INT_MAX,
         "x must be a float32 or bf16 [rows, (n_heads + 2 * kv heads) * head dim] tensor with contiguous rows");
    const int64_t rows = x.size(0);
    p.rows = (int)rows;
    p.x = x.data_ptr();
    p.x_ld = rows > 1 ? x.stride(0) : width;
    const char* what = "positions and slots must be contiguous int32 tensors with one entry per row on x's device";
    p.positions = ints(pos, dev, rows, what);
    p.slots = ints(slots, dev, rows, what);
    const float** gains[2] = {&p.q_norm, &p.k_norm};
    for (int i = 0; i < 2; i++) {
      if (a[6 + i] == Py_None) continue;
      const at::Tensor& g = tensor(a[6 + i], "q_norm and k_norm");
      need(g.scalar_type() == at::kFloat && g.is_cuda() && g.get_device() == dev && g.is_contiguous() && g.numel() == hd,
           "q_norm and k_norm are float32 [head dim] tensors on x's device");
      *gains[i] = g.const_data_ptr<float>();
    }
    p.eps = (float)float_arg(a[8]);
    p.theta = float_arg(a[9]);
    const int q_type = int_arg(a[10], "bad type");
    const OnStream on(a[12], dev);
    at::Tensor out;
    if (a[11] == Py_None) {
      p.q_dtype = q_type < 0 ? p.x_dtype : q_type;
      out = empty({rows, p.n_heads, hd}, p.q_dtype == CTTS_F32 ? at::kFloat : at::kBFloat16, dev);
    } else {
      out = tensor(a[11], "out");
      p.q_dtype = type_of(out);
      need(p.q_dtype >= 0 && (q_type < 0 || q_type == p.q_dtype) && out.is_cuda() && out.get_device() == dev,
           "out must be a float32 or bf16 [rows, n_heads, head dim] tensor of q_dtype on x's device");
    }
    p.q_ld = rows_ld(out, rows, p.n_heads, hd, "out must be a [rows, n_heads, head dim] tensor with whole rows");
    p.q = out.data_ptr();
    done(ctts_op_paged_append(&p, on.stream));
    written(k);
    written(v);
    if (a[11] != Py_None) {
      written(out);
      Py_INCREF(a[11]);
      return a[11];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// what the workspace follows from: queries [rows, heads, dim] and the pools
ctts_paged_attn attention_shape(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, int dev, int max_new) {
  ctts_paged_attn p{};
  p.kv = pool(k, v, dev);
  p.q_dtype = type_of(q);
  need(p.q_dtype >= 0 && q.dim() == 3 && q.size(2) == p.kv.head_dim && q.size(0) <= INT_MAX && q.size(1) <= INT_MAX,
       "q must be a float32 or bf16 [rows, heads, head dim] tensor on the pools' device");
  p.rows = (int)q.size(0);
  p.n_heads = (int)q.size(1);
  p.max_new = max_new;
  p.batch = p.max_pages = 1;
  p.table_ld = 1;
  return p;
}

// (q, k_pages, v_pages, block_tables, cu_rows, seq_lens, max_new, scale or None, out, workspace, stream)
PyObject* attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 11, "attention takes 11 arguments");
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages"), &tab = tensor(a[3], "block_tables"),
                     &cu = tensor(a[4], "cu_rows"), &lens = tensor(a[5], "seq_lens");
    const int dev = cuda_index(q);
    ctts_paged_attn p = attention_shape(q, k, v, dev, int_arg(a[6], "bad max_new"));
    const int64_t rows = p.rows, heads = p.n_heads, hd = p.kv.head_dim;
    p.q_ld = rows_ld(q, rows, heads, hd, "a row of q is contiguous");
    p.q = q.data_ptr();
    const char* what = "cu_rows (one entry more) and seq_lens must be contiguous int32 tensors on q's device";
    p.batch = to_int(lens.numel(), "too many requests");
    p.seq_lens = ints(lens, dev, 0, what);
    p.cu_rows = ints(cu, dev, 0, what);
    need(cu.numel() == (int64_t)p.batch + 1, what);
    p.table_ld = table_ld(tab, p.batch, dev);
    p.block_tables = tab.const_data_ptr<int>();
    p.max_pages = (int)tab.size(1);
    p.scale = a[7] == Py_None ? 1.0f / std::sqrt((float)hd) : (float)float_arg(a[7]);
    const OnStream on(a[10], dev);
    at::Tensor out, ws;
    if (a[8] == Py_None) {
      out = empty(q.sizes(), q.scalar_type(), dev);
    } else {
      out = tensor(a[8], "out");
      need(out.scalar_type() == q.scalar_type() && out.is_cuda() && out.get_device() == dev, "out must have q's shape and type, on its device");
    }
    p.out_ld = rows_ld(out, rows, heads, hd, "out must have q's shape and whole rows");
    p.out = out.data_ptr();
    if (a[9] == Py_None) {
      size_t bytes = 0;
      done(ctts_op_paged_attention_workspace(&p, &bytes));
      ws = empty({(int64_t)bytes}, at::kByte, dev);
      p.workspace_bytes = bytes;
    } else {
      ws = tensor(a[9], "workspace");
      need(ws.is_cuda() && ws.get_device() == dev && ws.is_contiguous(), "workspace must be a contiguous tensor on q's device");
      p.workspace_bytes = ws.nbytes();
    }
    p.workspace = ws.data_ptr();
    done(ctts_op_paged_attention(&p, on.stream));
    if (a[8] != Py_None) {
      written(out);
      Py_INCREF(a[8]);
      return a[8];
    }
    return THPVariable_Wrap(std::move(out));
  });
}

// (q, k_pages, v_pages, max_new)
PyObject* attention_workspace(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    need(n == 4, "attention_workspace takes 4 arguments");
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k_pages"), &v = tensor(a[2], "v_pages");
    const int dev = cuda_index(q);
    const ctts_paged_attn p = attention_shape(q, k, v, dev, int_arg(a[3], "bad max_new"));
    const OnStream on(Py_None, dev);
    size_t bytes = 0;
    done(ctts_op_paged_attention_workspace(&p, &bytes));
    return PyLong_FromSize_t(bytes);
  });
}

PyObject* set_error(PyObject*, PyObject* cls) {
  Py_XINCREF(cls);
  Py_XDECREF(g_error);
  g_error = cls;
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(plan)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(append)), METH_FASTCALL, nullptr},
    {"attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(attention)), METH_FASTCALL, nullptr},
    {"attention_workspace", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(attention_workspace)), METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_paged_ext", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

// Whether torch is the one this was built for: the layout of its classes goes
// with the version.
bool same_torch() {
  PyObject* torch = PyImport_ImportModule("torch");
  PyObject* version = torch ? PyObject_GetAttrString(torch, "__version__") : nullptr;
  const bool same = version && PyUnicode_Check(version) && PyUnicode_CompareWithASCIIString(version, PAGED_EXT_TORCH) == 0;
  if (version && !same) PyErr_Format(PyExc_ImportError, "_paged_ext.so was built for torch " PAGED_EXT_TORCH ", this is %S", version);
  Py_XDECREF(version);
  Py_XDECREF(torch);
  return same;
}

}  // namespace

PyMODINIT_FUNC PyInit__paged_ext(void) { return same_torch() ? PyModule_Create(&kModule) : nullptr; }
