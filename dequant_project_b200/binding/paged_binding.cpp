// Python binding of the paged-cache operators (dequant_project_b200/paged_ops.py):
// tensor checks, outputs and scratch memory from torch's caching allocator, and
// the call of the C ABI (include/dequant_b200.h) on torch's current stream. A
// step of a small batch runs in a few microseconds on the GPU, and checking ten
// tensors and packing twenty arguments in Python takes longer than that (13 us a
// call through ctypes), so these operators are bound natively. The library's
// entry points are handed in by address (bind), so that the process has one
// copy of the library, the one that _native.py loaded.
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <string>

#include "dequant_b200.h"

namespace {

decltype(&dqg_last_error) p_last_error = nullptr;
decltype(&dqg_rope_paged_append) p_append = nullptr;
decltype(&dqg_paged_attention_workspace) p_decode_bytes = nullptr;
decltype(&dqg_paged_attention) p_decode = nullptr;
decltype(&dqg_prompt_attention_workspace) p_prompt_bytes = nullptr;
decltype(&dqg_prompt_attention) p_prompt = nullptr;
decltype(&dqg_shared_prefix_workspace) p_prefix_bytes = nullptr;
decltype(&dqg_shared_prefix_attention) p_prefix = nullptr;

// A rejected argument: becomes RuntimeError with this message.
struct Rejected {
  std::string text;
};
[[noreturn]] void reject(const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  throw Rejected{buf};
}

void check(int rc) {
  if (rc) reject("%s", p_last_error());
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) reject("%s must be a tensor", name);
  return THPVariable_Unpack(o);
}

const char* type_name(at::ScalarType t) { return t == at::kHalf ? "float16" : "bfloat16"; }

// The operators have no backward pass: what autograd would record is refused
// instead of left out.
void forward_only(std::initializer_list<const at::Tensor*> inputs) {
  if (!at::GradMode::is_enabled()) return;
  for (const at::Tensor* t : inputs)
    if (t->requires_grad())
      reject("the paged operators are forward only: an input requires a gradient (call them under torch.no_grad())");
}

struct Pools {
  dqg_paged_kv kv;
  at::ScalarType type;
  int device;
};
Pools pools(const at::Tensor& k, const at::Tensor& v) {
  Pools p;
  p.type = k.scalar_type();
  if (p.type != at::kHalf && p.type != at::kBFloat16)
    reject("pages must be float16 or bfloat16, got %s", c10::toString(p.type));
  if (k.dim() != 4) reject("pages must be [pages, kv heads, page size, head dim]");
  if (!k.is_cuda()) reject("k_pages must be a CUDA tensor");
  if (v.sizes() != k.sizes() || v.strides() != k.strides() || v.scalar_type() != p.type || k.stride(3) != 1)
    reject("k_pages and v_pages must have one shape, type and strides, with the head dimension contiguous");
  if (v.device() != k.device()) reject("k_pages and v_pages must be on the same device");
  p.device = k.get_device();
  p.kv = dqg_paged_kv{k.data_ptr(), v.data_ptr(), k.size(0), k.size(1), k.size(2), k.size(3),
                      k.stride(0), k.stride(1), k.stride(2), p.type == at::kHalf ? DQG_FP16 : DQG_BF16};
  return p;
}

void same(const Pools& p, const at::Tensor& t, const char* name) {
  if (t.scalar_type() != p.type || !t.is_cuda() || t.get_device() != p.device)
    reject("%s must be %s on cuda:%d, as the pages are", name, type_name(p.type), p.device);
}

// A tensor of integers whose last dimension is contiguous.
void ints(const Pools& p, const at::Tensor& t, const char* name, at::ScalarType type, int64_t dims, int64_t rows) {
  if (t.scalar_type() != type || t.dim() != dims || !t.is_cuda() || t.get_device() != p.device ||
      (t.size(dims - 1) > 1 && t.stride(dims - 1) != 1))
    reject("%s must be a contiguous %d-dimensional %s tensor on cuda:%d", name, static_cast<int>(dims),
           type == at::kInt ? "int32" : "int64", p.device);
  if (rows >= 0 && t.size(0) != rows)
    reject("%s must hold %lld rows, got %lld", name, static_cast<long long>(rows), static_cast<long long>(t.size(0)));
}

// A block table's row length and stride.
int64_t row_stride(const at::Tensor& table) { return table.size(0) > 1 ? table.stride(0) : table.size(1); }

void query(const Pools& p, const at::Tensor& q, PyObject* k, PyObject* v) {
  forward_only({&q, &THPVariable_Unpack(k), &THPVariable_Unpack(v)});
  same(p, q, "q");
  if (q.dim() != 3 || q.size(2) != p.kv.head_dim || q.stride(2) != 1)
    reject("q must be [rows, heads, %d] with the head dimension contiguous", static_cast<int>(p.kv.head_dim));
}

float scale_of(PyObject* o, int64_t head_dim) {
  if (o == Py_None) return static_cast<float>(1.0 / std::sqrt(static_cast<double>(head_dim)));
  const double s = PyFloat_AsDouble(o);
  if (s == -1.0 && PyErr_Occurred()) throw python_error();
  return static_cast<float>(s);
}

struct Scratch {
  at::Tensor held;
  void* ptr;
  uint64_t bytes;
};
Scratch scratch(PyObject* given, uint64_t need, const at::Tensor& q) {
  Scratch s;
  if (given == Py_None) {
    s.held = at::empty({static_cast<int64_t>(need)}, q.options().dtype(at::kByte));
  } else {
    s.held = tensor(given, "workspace");
    if (!s.held.is_cuda() || s.held.get_device() != q.get_device() || !s.held.is_contiguous())
      reject("the workspace must be a contiguous tensor on cuda:%d", static_cast<int>(q.get_device()));
  }
  s.ptr = s.held.data_ptr();
  s.bytes = s.held.nbytes();
  return s;
}

void* stream_of(int device) {
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

void arguments(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) reject("expected %d arguments, got %d", static_cast<int>(want), static_cast<int>(n));
  if (p_last_error == nullptr) reject("the library is not bound");
}

// (qkv, cos, sin, positions, slots, k_pages, v_pages, n_q_heads, interleaved,
//  q_norm, k_norm, eps)
at::Tensor append(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 12);
  const at::Tensor &qkv = tensor(a[0], "qkv"), &cos = tensor(a[1], "cos"), &sin = tensor(a[2], "sin");
  const at::Tensor &positions = tensor(a[3], "positions"), &slots = tensor(a[4], "slots");
  const Pools p = pools(tensor(a[5], "k_pages"), tensor(a[6], "v_pages"));
  const at::Tensor &k = tensor(a[5], "k_pages"), &v = tensor(a[6], "v_pages");
  const int64_t hq = integer(a[7]), d = p.kv.head_dim;
  forward_only({&qkv, &cos, &sin, &k, &v});
  same(p, qkv, "qkv");
  const int64_t width = (hq + 2 * p.kv.n_kv_heads) * d;
  if (qkv.dim() != 2 || qkv.size(1) != width || qkv.stride(1) != 1)
    reject("qkv must be [T, %lld] with contiguous rows", static_cast<long long>(width));
  const int64_t t = qkv.size(0);
  for (const at::Tensor* x : {&cos, &sin})
    if (x->scalar_type() != at::kFloat || x->dim() != 2 || x->sizes() != cos.sizes() || !x->is_cuda() ||
        x->get_device() != p.device || !x->is_contiguous())
      reject("cos and sin must be contiguous float32 [positions, R / 2] on cuda:%d", p.device);
  ints(p, positions, "positions", at::kLong, 1, t);
  ints(p, slots, "slots", at::kLong, 1, t);
  const void* norms[2] = {nullptr, nullptr};
  const char* names[2] = {"q_norm", "k_norm"};
  for (int i = 0; i < 2; ++i) {
    if (a[9 + i] == Py_None) continue;
    const at::Tensor& w = tensor(a[9 + i], names[i]);
    forward_only({&w});
    same(p, w, names[i]);
    if (w.dim() != 1 || w.size(0) != d || w.stride(0) != 1)
      reject("%s must hold %lld contiguous weights", names[i], static_cast<long long>(d));
    norms[i] = w.data_ptr();
  }
  const int interleaved = PyObject_IsTrue(a[8]);
  const double eps = PyFloat_AsDouble(a[11]);
  if (PyErr_Occurred()) throw python_error();
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(p.device));
  at::Tensor q = at::empty({t, hq, d}, qkv.options());
  check(p_append(qkv.data_ptr(), t, t > 1 ? qkv.stride(0) : width, hq, cos.data_ptr<float>(),
                 sin.data_ptr<float>(), cos.size(0), 2 * cos.size(1), interleaved, positions.data_ptr<int64_t>(),
                 slots.data_ptr<int64_t>(), norms[0], norms[1], static_cast<float>(eps), &p.kv, q.data_ptr(),
                 stream_of(p.device)));
  // Written in place: what autograd has saved of the pages is out of date.
  for (const at::Tensor* x : {&k, &v})
    if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
  return q;
}

// (q, k_pages, v_pages, block_table, kv_lens, scale, workspace)
at::Tensor decode(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 7);
  const at::Tensor &q = tensor(a[0], "q"), &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "kv_lens");
  const Pools p = pools(tensor(a[1], "k_pages"), tensor(a[2], "v_pages"));
  query(p, q, a[1], a[2]);
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2);
  ints(p, table, "block_table", at::kInt, 2, b);
  ints(p, lens, "kv_lens", at::kInt, 1, b);
  const float scale = scale_of(a[5], d);
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(p.device));
  uint64_t need = 0;
  check(p_decode_bytes(b, hq, p.kv.n_kv_heads, d, &need));
  const Scratch ws = scratch(a[6], need, q);
  at::Tensor out = at::empty({b, hq, d}, q.options());
  check(p_decode(q.data_ptr(), q.stride(0), q.stride(1), b, hq, &p.kv, table.data_ptr<int32_t>(), table.size(1),
                 row_stride(table), lens.data_ptr<int32_t>(), scale, out.data_ptr(), ws.ptr, ws.bytes,
                 stream_of(p.device)));
  return out;
}

// (q, k_pages, v_pages, block_table, q_starts, kv_lens, causal, scale, workspace)
at::Tensor prompt(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 9);
  const at::Tensor &q = tensor(a[0], "q"), &table = tensor(a[3], "block_table");
  const at::Tensor &starts = tensor(a[4], "q_starts"), &lens = tensor(a[5], "kv_lens");
  const Pools p = pools(tensor(a[1], "k_pages"), tensor(a[2], "v_pages"));
  query(p, q, a[1], a[2]);
  const int64_t t = q.size(0), hq = q.size(1), d = q.size(2);
  ints(p, lens, "kv_lens", at::kInt, 1, -1);
  const int64_t b = lens.size(0);
  ints(p, table, "block_table", at::kInt, 2, b);
  ints(p, starts, "q_starts", at::kInt, 1, b + 1);
  const int causal = PyObject_IsTrue(a[6]);
  const float scale = scale_of(a[7], d);
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(p.device));
  uint64_t need = 0;
  check(p_prompt_bytes(d, &need));
  const Scratch ws = scratch(a[8], need, q);
  at::Tensor out = at::empty({t, hq, d}, q.options());
  check(p_prompt(q.data_ptr(), q.stride(0), q.stride(1), t, hq, &p.kv, table.data_ptr<int32_t>(), table.size(1),
                 row_stride(table), starts.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), b, causal, scale,
                 out.data_ptr(), ws.ptr, ws.bytes, stream_of(p.device)));
  return out;
}

// (q, k_pages, v_pages, prefix_table, prefix_len, block_table, kv_lens, scale,
//  workspace)
at::Tensor prefix(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 9);
  const at::Tensor &q = tensor(a[0], "q"), &pre = tensor(a[3], "prefix_table");
  const at::Tensor &table = tensor(a[5], "block_table"), &lens = tensor(a[6], "kv_lens");
  const Pools p = pools(tensor(a[1], "k_pages"), tensor(a[2], "v_pages"));
  const int64_t len = integer(a[4]);
  query(p, q, a[1], a[2]);
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2);
  ints(p, pre, "prefix_table", at::kInt, 1, -1);
  ints(p, table, "block_table", at::kInt, 2, b);
  ints(p, lens, "kv_lens", at::kInt, 1, b);
  const float scale = scale_of(a[7], d);
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(p.device));
  uint64_t need = 0;
  check(p_prefix_bytes(b, hq, p.kv.n_kv_heads, d, len, &need));
  const Scratch ws = scratch(a[8], need, q);
  at::Tensor out = at::empty({b, hq, d}, q.options());
  check(p_prefix(q.data_ptr(), q.stride(0), q.stride(1), b, hq, &p.kv, pre.data_ptr<int32_t>(), pre.size(0), len,
                 table.data_ptr<int32_t>(), table.size(1), row_stride(table), lens.data_ptr<int32_t>(), scale,
                 out.data_ptr(), ws.ptr, ws.bytes, stream_of(p.device)));
  return out;
}

template <at::Tensor (*F)(PyObject* const*, Py_ssize_t)>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::AutoDispatchBelowADInplaceOrView below;
  try {
    return THPVariable_Wrap(F(args, n));
  } catch (const Rejected& r) {
    PyErr_SetString(PyExc_RuntimeError, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// Addresses of the library's entry points, in the order below.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  void* at[8];
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "bind takes 8 addresses");
    return nullptr;
  }
  for (int i = 0; i < 8; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  p_append = reinterpret_cast<decltype(p_append)>(at[1]);
  p_decode_bytes = reinterpret_cast<decltype(p_decode_bytes)>(at[2]);
  p_decode = reinterpret_cast<decltype(p_decode)>(at[3]);
  p_prompt_bytes = reinterpret_cast<decltype(p_prompt_bytes)>(at[4]);
  p_prompt = reinterpret_cast<decltype(p_prompt)>(at[5]);
  p_prefix_bytes = reinterpret_cast<decltype(p_prefix_bytes)>(at[6]);
  p_prefix = reinterpret_cast<decltype(p_prefix)>(at[7]);
  p_last_error = reinterpret_cast<decltype(p_last_error)>(at[0]);
  Py_RETURN_NONE;
}

#define METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD("bind", bind),
                         METHOD("rope_paged_append", call<append>),
                         METHOD("paged_attention", call<decode>),
                         METHOD("prompt_attention", call<prompt>),
                         METHOD("shared_prefix_attention", call<prefix>),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_binding", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `built_for`: the torch that this was compiled against, whose layouts it knows.
PyMODINIT_FUNC PyInit__paged_binding(void) {
  PyObject* m = PyModule_Create(&module);
  if (m != nullptr && PyModule_AddStringConstant(m, "built_for", DQG_BUILT_FOR) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
