// Python binding of the paged-cache operators (dequant_project_b200/paged_ops.py,
// quantized_cache.py) and of the token draw (sampling.py): tensor checks,
// outputs and scratch memory from torch's caching allocator, and the call of the
// C ABI (include/dequant_b200.h) on torch's current stream. A
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
#include <type_traits>

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
decltype(&dqg_rope_quantized_append) p_quantized_append = nullptr;
decltype(&dqg_expand_pages) p_expand = nullptr;
decltype(&dqg_quantized_attention_workspace) p_quantized_bytes = nullptr;
decltype(&dqg_quantized_attention) p_quantized = nullptr;
decltype(&dqg_quantized_prompt_workspace) p_quantized_prompt_bytes = nullptr;
decltype(&dqg_quantized_prompt_attention) p_quantized_prompt = nullptr;
decltype(&dqg_sample_tokens) p_sample = nullptr;

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

// Written in place: what autograd has saved of these is out of date.
void changed(std::initializer_list<const at::Tensor*> tensors) {
  for (const at::Tensor* x : tensors)
    if (!x->is_inference()) x->unsafeGetTensorImpl()->bump_version();
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

template <class P>
void same(const P& p, const at::Tensor& t, const char* name) {
  if (t.scalar_type() != p.type || !t.is_cuda() || t.get_device() != p.device)
    reject("%s must be %s on cuda:%d, as the pages are", name, type_name(p.type), p.device);
}

// A tensor of integers whose last dimension is contiguous.
template <class P>
void ints(const P& p, const at::Tensor& t, const char* name, at::ScalarType type, int64_t dims, int64_t rows) {
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

// What is rotated and stored: rows of query, key and value heads, the tables
// and their rows. Returns the number of tokens.
template <class P>
int64_t rotated(const P& p, const at::Tensor& qkv, const at::Tensor& cos, const at::Tensor& sin,
                const at::Tensor& positions, int64_t hq) {
  same(p, qkv, "qkv");
  const int64_t width = (hq + 2 * p.kv.n_kv_heads) * p.kv.head_dim;
  if (qkv.dim() != 2 || qkv.size(1) != width || qkv.stride(1) != 1)
    reject("qkv must be [T, %lld] with contiguous rows", static_cast<long long>(width));
  for (const at::Tensor* x : {&cos, &sin})
    if (x->scalar_type() != at::kFloat || x->dim() != 2 || x->sizes() != cos.sizes() || !x->is_cuda() ||
        x->get_device() != p.device || !x->is_contiguous())
      reject("cos and sin must be contiguous float32 [positions, R / 2] on cuda:%d", p.device);
  ints(p, positions, "positions", at::kLong, 1, qkv.size(0));
  return qkv.size(0);
}

// Weights of the heads' norms (tensors, or None).
struct Norms {
  const void *q, *k;
};
template <class P>
Norms norms_of(const P& p, PyObject* const* a) {
  const void* norms[2] = {nullptr, nullptr};
  const char* names[2] = {"q_norm", "k_norm"};
  for (int i = 0; i < 2; ++i) {
    if (a[i] == Py_None) continue;
    const at::Tensor& w = tensor(a[i], names[i]);
    forward_only({&w});
    same(p, w, names[i]);
    if (w.dim() != 1 || w.size(0) != p.kv.head_dim || w.stride(0) != 1)
      reject("%s must hold %lld contiguous weights", names[i], static_cast<long long>(p.kv.head_dim));
    norms[i] = w.data_ptr();
  }
  return Norms{norms[0], norms[1]};
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
  const int64_t t = rotated(p, qkv, cos, sin, positions, hq);
  ints(p, slots, "slots", at::kLong, 1, t);
  const Norms norms = norms_of(p, a + 9);
  const int interleaved = PyObject_IsTrue(a[8]);
  const double eps = PyFloat_AsDouble(a[11]);
  if (PyErr_Occurred()) throw python_error();
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(p.device));
  at::Tensor q = at::empty({t, hq, d}, qkv.options());
  check(p_append(qkv.data_ptr(), t, t > 1 ? qkv.stride(0) : qkv.size(1), hq, cos.data_ptr<float>(),
                 sin.data_ptr<float>(), cos.size(0), 2 * cos.size(1), interleaved, positions.data_ptr<int64_t>(),
                 slots.data_ptr<int64_t>(), norms.q, norms.k, static_cast<float>(eps), &p.kv, q.data_ptr(),
                 stream_of(p.device)));
  changed({&k, &v});
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

PyObject* tuple(std::initializer_list<at::Tensor> tensors) {
  PyObject* t = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
  if (t == nullptr) throw python_error();
  Py_ssize_t i = 0;
  for (const at::Tensor& x : tensors) PyTuple_SET_ITEM(t, i++, THPVariable_Wrap(x));
  return t;
}

// A cache held in 8 bits: k, v, k_scale, v_scale, k_open, v_open.
struct Quantized {
  dqg_quantized_kv kv;
  const at::Tensor* t[6];
  at::ScalarType type;  // of open rows, queries and outputs
  int device;
};
Quantized quantized(PyObject* const* a) {
  static const char* names[6] = {"k", "v", "k_scale", "v_scale", "k_open", "v_open"};
  Quantized c;
  for (int i = 0; i < 6; ++i) c.t[i] = &tensor(a[i], names[i]);
  const at::Tensor &k = *c.t[0], &ks = *c.t[2], &ko = *c.t[4];
  if (!k.is_cuda()) reject("k must be a CUDA tensor");
  c.device = k.get_device();
  for (int i = 1; i < 6; ++i)
    if (!c.t[i]->is_cuda() || c.t[i]->get_device() != c.device) reject("%s must be on cuda:%d, as k is", names[i], c.device);
  if (k.scalar_type() != at::kChar && k.scalar_type() != at::kFloat8_e4m3fn)
    reject("codes must be int8 or float8_e4m3fn, got %s", c10::toString(k.scalar_type()));
  c.type = ko.scalar_type();
  if (c.type != at::kHalf && c.type != at::kBFloat16)
    reject("open blocks must be float16 or bfloat16, got %s", c10::toString(c.type));
  if (k.dim() != 4 || k.stride(3) != 1)
    reject("codes must be [pages, kv heads, page size, head dim] with the head dimension contiguous");
  if (ks.scalar_type() != at::kFloat || ks.dim() != 3 || ks.size(0) != k.size(0) || ks.size(1) != k.size(1) ||
      (ks.size(2) > 1 && ks.stride(2) != 1))
    reject("scales must be float32 [pages, kv heads, page size / block] with the blocks contiguous");
  if (ko.dim() != 4 || ko.size(1) != k.size(1) || ko.size(3) != k.size(3) || ko.stride(3) != 1 ||
      ko.stride(2) != ko.size(3))
    reject("open blocks must be [slots, kv heads, block, head dim] with the last two dimensions contiguous");
  if (ks.size(2) * ko.size(2) != k.size(2))
    reject("pages of %lld positions do not hold %lld blocks of %lld", static_cast<long long>(k.size(2)),
           static_cast<long long>(ks.size(2)), static_cast<long long>(ko.size(2)));
  for (int i = 0; i < 6; i += 2) {
    const at::Tensor &x = *c.t[i], &y = *c.t[i + 1];
    if (y.sizes() != x.sizes() || y.strides() != x.strides() || y.scalar_type() != x.scalar_type())
      reject("%s and %s must have one shape, type and strides", names[i], names[i + 1]);
  }
  c.kv = dqg_quantized_kv{k.data_ptr(), c.t[1]->data_ptr(), static_cast<float*>(ks.data_ptr()),
                          static_cast<float*>(c.t[3]->data_ptr()), ko.data_ptr(), c.t[5]->data_ptr(),
                          k.size(0), k.size(1), k.size(2), k.size(3), ko.size(2), ko.size(0),
                          k.stride(0), k.stride(1), k.stride(2), ks.stride(0), ks.stride(1), ko.stride(0), ko.stride(1),
                          k.scalar_type() == at::kChar ? DQG_INT8 : DQG_E4M3, c.type == at::kHalf ? DQG_FP16 : DQG_BF16};
  return c;
}

void forward_only_cache(const at::Tensor& x, const Quantized& c) {
  forward_only({&x, c.t[0], c.t[1], c.t[2], c.t[3], c.t[4], c.t[5]});
}

// (qkv, cos, sin, positions, cache: 6, block_table, open_slots, q_starts,
//  kv_lens, n_q_heads, interleaved, q_norm, k_norm, eps)
at::Tensor quantized_append(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 19);
  const at::Tensor &qkv = tensor(a[0], "qkv"), &cos = tensor(a[1], "cos"), &sin = tensor(a[2], "sin");
  const at::Tensor& positions = tensor(a[3], "positions");
  const Quantized c = quantized(a + 4);
  const at::Tensor &table = tensor(a[10], "block_table"), &open = tensor(a[11], "open_slots");
  const at::Tensor &starts = tensor(a[12], "q_starts"), &lens = tensor(a[13], "kv_lens");
  const int64_t hq = integer(a[14]), d = c.kv.head_dim;
  forward_only_cache(qkv, c);
  forward_only({&cos, &sin});
  const int64_t t = rotated(c, qkv, cos, sin, positions, hq);
  ints(c, lens, "kv_lens", at::kInt, 1, -1);
  const int64_t b = lens.size(0);
  ints(c, table, "block_table", at::kInt, 2, b);
  ints(c, open, "open_slots", at::kInt, 1, b);
  ints(c, starts, "q_starts", at::kInt, 1, b + 1);
  const Norms norms = norms_of(c, a + 16);
  const int interleaved = PyObject_IsTrue(a[15]);
  const double eps = PyFloat_AsDouble(a[18]);
  if (PyErr_Occurred()) throw python_error();
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.device));
  at::Tensor q = at::empty({t, hq, d}, qkv.options());
  check(p_quantized_append(qkv.data_ptr(), t, t > 1 ? qkv.stride(0) : qkv.size(1), hq, cos.data_ptr<float>(),
                           sin.data_ptr<float>(), cos.size(0), 2 * cos.size(1), interleaved,
                           positions.data_ptr<int64_t>(), norms.q, norms.k, static_cast<float>(eps), &c.kv,
                           table.data_ptr<int32_t>(), table.size(1), row_stride(table), open.data_ptr<int32_t>(),
                           starts.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), b, q.data_ptr(),
                           stream_of(c.device)));
  for (const at::Tensor* x : c.t) changed({x});
  return q;
}

// (cache: 6, block_table, open_slots, kv_lens, n_pages) -> (k_pages, v_pages,
// table)
PyObject* expand(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 10);
  const Quantized c = quantized(a);
  const at::Tensor &table = tensor(a[6], "block_table"), &open = tensor(a[7], "open_slots");
  const at::Tensor& lens = tensor(a[8], "kv_lens");
  const int64_t pages = integer(a[9]);
  forward_only_cache(*c.t[0], c);
  ints(c, lens, "kv_lens", at::kInt, 1, -1);
  const int64_t b = lens.size(0);
  ints(c, table, "block_table", at::kInt, 2, b);
  ints(c, open, "open_slots", at::kInt, 1, b);
  if (pages < 0) reject("n_pages=%lld out of range", static_cast<long long>(pages));
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.device));
  const at::TensorOptions options = c.t[4]->options();
  at::Tensor k = at::empty({pages, c.kv.n_kv_heads, c.kv.page_size, c.kv.head_dim}, options), v = at::empty_like(k);
  at::Tensor out = at::empty({b, table.size(1)}, table.options());
  check(p_expand(&c.kv, table.data_ptr<int32_t>(), table.size(1), row_stride(table), open.data_ptr<int32_t>(),
                 lens.data_ptr<int32_t>(), b, pages, k.data_ptr(), v.data_ptr(), out.data_ptr<int32_t>(),
                 stream_of(c.device)));
  return tuple({k, v, out});
}

// (q, cache: 6, block_table, open_slots, kv_lens, scale, workspace)
at::Tensor quantized_decode(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 12);
  const at::Tensor& q = tensor(a[0], "q");
  const Quantized c = quantized(a + 1);
  const at::Tensor &table = tensor(a[7], "block_table"), &open = tensor(a[8], "open_slots");
  const at::Tensor& lens = tensor(a[9], "kv_lens");
  forward_only_cache(q, c);
  same(c, q, "q");
  if (q.dim() != 3 || q.size(2) != c.kv.head_dim || q.stride(2) != 1)
    reject("q must be [rows, heads, %d] with the head dimension contiguous", static_cast<int>(c.kv.head_dim));
  const int64_t b = q.size(0), hq = q.size(1), d = q.size(2);
  ints(c, table, "block_table", at::kInt, 2, b);
  ints(c, open, "open_slots", at::kInt, 1, b);
  ints(c, lens, "kv_lens", at::kInt, 1, b);
  const float scale = scale_of(a[10], d);
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.device));
  uint64_t need = 0;
  check(p_quantized_bytes(b, hq, c.kv.n_kv_heads, d, &need));
  const Scratch ws = scratch(a[11], need, q);
  at::Tensor out = at::empty({b, hq, d}, q.options());
  check(p_quantized(q.data_ptr(), q.stride(0), q.stride(1), b, hq, &c.kv, table.data_ptr<int32_t>(), table.size(1),
                    row_stride(table), open.data_ptr<int32_t>(), lens.data_ptr<int32_t>(), scale, out.data_ptr(),
                    ws.ptr, ws.bytes, stream_of(c.device)));
  return out;
}

// (q, cache: 6, block_table, open_slots, q_starts, kv_lens, n_pages, causal,
//  scale, workspace)
at::Tensor quantized_prompt(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 15);
  const at::Tensor& q = tensor(a[0], "q");
  const Quantized c = quantized(a + 1);
  const at::Tensor &table = tensor(a[7], "block_table"), &open = tensor(a[8], "open_slots");
  const at::Tensor &starts = tensor(a[9], "q_starts"), &lens = tensor(a[10], "kv_lens");
  const int64_t pages = integer(a[11]);
  const int causal = PyObject_IsTrue(a[12]);
  forward_only_cache(q, c);
  same(c, q, "q");
  if (q.dim() != 3 || q.size(2) != c.kv.head_dim || q.stride(2) != 1)
    reject("q must be [rows, heads, %d] with the head dimension contiguous", static_cast<int>(c.kv.head_dim));
  const int64_t t = q.size(0), hq = q.size(1), d = q.size(2);
  ints(c, lens, "kv_lens", at::kInt, 1, -1);
  const int64_t b = lens.size(0);
  ints(c, table, "block_table", at::kInt, 2, b);
  ints(c, open, "open_slots", at::kInt, 1, b);
  ints(c, starts, "q_starts", at::kInt, 1, b + 1);
  const float scale = scale_of(a[13], d);
  c10::cuda::CUDAGuard guard(static_cast<c10::DeviceIndex>(c.device));
  uint64_t need = 0;
  check(p_quantized_prompt_bytes(&c.kv, b, table.size(1), pages, &need));
  const Scratch ws = scratch(a[14], need, q);
  at::Tensor out = at::empty({t, hq, d}, q.options());
  check(p_quantized_prompt(q.data_ptr(), q.stride(0), q.stride(1), t, hq, &c.kv, table.data_ptr<int32_t>(),
                           table.size(1), row_stride(table), open.data_ptr<int32_t>(), starts.data_ptr<int32_t>(),
                           lens.data_ptr<int32_t>(), b, pages, causal, scale, out.data_ptr(), ws.ptr, ws.bytes,
                           stream_of(c.device)));
  return out;
}

// A parameter of the draw: a number for all rows, or a tensor of one a row.
template <typename T>
void parameter(PyObject* o, const at::Tensor& logits, const char* name, const T** each, T* all) {
  *each = nullptr;
  if (!THPVariable_Check(o)) {
    if constexpr (std::is_same_v<T, float>) {
      *all = static_cast<float>(PyFloat_AsDouble(o));
    } else {
      const long long v = PyLong_AsLongLong(o);
      *all = static_cast<T>(v < 0 ? 0 : (v > 0x7fffffff ? 0x7fffffff : v));
    }
    if (PyErr_Occurred()) throw python_error();
    return;
  }
  const at::Tensor& t = THPVariable_Unpack(o);
  const at::ScalarType type = std::is_same_v<T, float> ? at::kFloat : at::kInt;
  if (t.scalar_type() != type || t.dim() != 1 || t.size(0) != logits.size(0) || !t.is_cuda() ||
      t.get_device() != logits.get_device() || !t.is_contiguous())
    reject("%s must be a number, or a contiguous %s tensor of %lld rows on cuda:%d", name,
           type == at::kFloat ? "float32" : "int32", static_cast<long long>(logits.size(0)),
           static_cast<int>(logits.get_device()));
  *each = static_cast<const T*>(t.data_ptr());
}

// (logits, uniform, temperature, top_k, top_p, min_p) -> (tokens, logprobs)
PyObject* sample(PyObject* const* a, Py_ssize_t n) {
  arguments(n, 6);
  const at::Tensor &logits = tensor(a[0], "logits"), &uniform = tensor(a[1], "uniform");
  if (!logits.is_cuda()) reject("logits must be a CUDA tensor");
  const at::ScalarType type = logits.scalar_type();
  if (type != at::kHalf && type != at::kBFloat16 && type != at::kFloat)
    reject("logits must be float16, bfloat16 or float32, got %s", c10::toString(type));
  if (logits.dim() != 2 || (logits.size(1) > 1 && logits.stride(1) != 1))
    reject("logits must be [rows, vocab] with contiguous rows");
  const int64_t rows = logits.size(0), vocab = logits.size(1);
  if (uniform.scalar_type() != at::kFloat || uniform.dim() != 1 || uniform.size(0) != rows || !uniform.is_cuda() ||
      uniform.get_device() != logits.get_device() || !uniform.is_contiguous())
    reject("uniform must be a contiguous float32 tensor of %lld rows on cuda:%d", static_cast<long long>(rows),
           static_cast<int>(logits.get_device()));
  if (at::GradMode::is_enabled())
    for (int i = 0; i < 6; ++i)
      if (THPVariable_Check(a[i]) && THPVariable_Unpack(a[i]).requires_grad())
        reject("a draw has no gradient: an input requires one (call it under torch.no_grad())");
  dqg_sampling s;
  parameter(a[2], logits, "temperature", &s.temperatures, &s.temperature);
  parameter(a[3], logits, "top_k", &s.top_ks, &s.top_k);
  parameter(a[4], logits, "top_p", &s.top_ps, &s.top_p);
  parameter(a[5], logits, "min_p", &s.min_ps, &s.min_p);
  c10::cuda::CUDAGuard guard(logits.device());
  at::Tensor tokens = at::empty({rows}, logits.options().dtype(at::kLong));
  at::Tensor logprobs = at::empty({rows}, logits.options().dtype(at::kFloat));
  check(p_sample(logits.data_ptr(), type == at::kHalf ? DQG_FP16 : (type == at::kFloat ? DQG_FP32 : DQG_BF16), rows,
                 vocab, rows > 1 ? logits.stride(0) : vocab, uniform.data_ptr<float>(), &s, tokens.data_ptr<int64_t>(),
                 logprobs.data_ptr<float>(), stream_of(logits.get_device())));
  return tuple({tokens, logprobs});
}

PyObject* wrapped(at::Tensor t) { return THPVariable_Wrap(t); }
PyObject* wrapped(PyObject* o) { return o; }

template <auto F>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  at::AutoDispatchBelowADInplaceOrView below;
  try {
    return wrapped(F(args, n));
  } catch (const Rejected& r) {
    PyErr_SetString(PyExc_RuntimeError, r.text.c_str());
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

template <typename F>
void set(F*& entry, void* address) {
  entry = reinterpret_cast<F*>(address);
}

// Addresses of the library's entry points, in the order below.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr int kEntries = 15;
  void* at[kEntries];
  if (n != kEntries) {
    PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kEntries);
    return nullptr;
  }
  for (int i = 0; i < kEntries; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (at[i] == nullptr) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  set(p_append, at[1]);
  set(p_decode_bytes, at[2]);
  set(p_decode, at[3]);
  set(p_prompt_bytes, at[4]);
  set(p_prompt, at[5]);
  set(p_prefix_bytes, at[6]);
  set(p_prefix, at[7]);
  set(p_quantized_append, at[8]);
  set(p_expand, at[9]);
  set(p_quantized_bytes, at[10]);
  set(p_quantized, at[11]);
  set(p_sample, at[12]);
  set(p_quantized_prompt_bytes, at[13]);
  set(p_quantized_prompt, at[14]);
  set(p_last_error, at[0]);
  Py_RETURN_NONE;
}

#define METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD("bind", bind),
                         METHOD("rope_paged_append", call<append>),
                         METHOD("paged_attention", call<decode>),
                         METHOD("prompt_attention", call<prompt>),
                         METHOD("shared_prefix_attention", call<prefix>),
                         METHOD("rope_quantized_append", call<quantized_append>),
                         METHOD("expand_pages", call<expand>),
                         METHOD("quantized_attention", call<quantized_decode>),
                         METHOD("quantized_prompt_attention", call<quantized_prompt>),
                         METHOD("sample_tokens", call<sample>),
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
