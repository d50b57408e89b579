// bind.cpp — the Python side of the operators between the packed linears (include/trellis_amd.h): argument checks,
// output and scratch tensors, the current stream, and the call into libtrellis_amd.so.
//
// A decode step makes some hundred of these calls, each a few microseconds of GPU time, so the host's share counts: a
// tensor's dtype, sizes, strides, device and address cost ~1 us together as Python attributes, and a call has up to 13
// tensors. Here they are field reads: one token's append takes 4.5 us of host time (13.4 with the same checks in
// Python and ctypes), a norm with its two outputs 5.0 (9.7), of which the launch is 2.8.
//
// Every function takes its arguments in order (norms.py and kv_cache.py hold the signatures and document them) and
// returns its result, or the library's status code as an int. Arguments that do not fit raise ValueError; nothing has
// been launched then.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/ExpandUtils.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/GradMode.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdarg>
#include <cstring>
#include <string>
#include <vector>

#include "trellis_amd.h"

namespace {

// The library's entry points, handed over by address when it has been loaded (bind()).
struct Entry {
  decltype(&trellis_residual_norm) residual_norm;
  decltype(&trellis_kv_append) kv_append;
  decltype(&trellis_attention_workspace_bytes) attention_workspace_bytes;
  decltype(&trellis_paged_attention) paged_attention;
  decltype(&trellis_evict_workspace_bytes) evict_workspace_bytes;
  decltype(&trellis_kv_evict) kv_evict;
  decltype(&trellis_tree_attention_workspace_bytes) tree_attention_workspace_bytes;
  decltype(&trellis_tree_attention) tree_attention;
  decltype(&trellis_beam_workspace_bytes) beam_workspace_bytes;
  decltype(&trellis_beam_select) beam_select;
  decltype(&trellis_kv_copy_pages) kv_copy_pages;
  decltype(&trellis_kv_keep) kv_keep;
} entry = {};

struct Refused {};   // a Python error is set

[[noreturn]] void refuse(const char* format, ...) {
  va_list args;
  va_start(args, format);
  PyErr_FormatV(PyExc_ValueError, format, args);
  va_end(args);
  throw Refused();
}

// A status other than TRELLIS_OK, for the Python side to raise.
struct Status {
  int code;
};

void check(int status) {
  if (status != TRELLIS_OK) throw Status{status};
}

const at::Tensor* optional_tensor(PyObject* o, const char* name) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse("%s must be a tensor", name);
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.requires_grad() && c10::GradMode::is_enabled())
    refuse("forward only: call it under torch.no_grad() or detach the inputs (%s wants a gradient)", name);
  // (no_grad does not switch forward-mode differentiation off; its dual numbers are of one level)
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    refuse("forward only: unpack the dual tensor (%s carries a tangent)", name);
  return &t;
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  const at::Tensor* t = optional_tensor(o, name);
  if (!t) refuse("%s must be a tensor", name);
  return *t;
}

double number(PyObject* o, const char* name) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse("%s must be a number", name);
  }
  return v;
}

int whole(PyObject* o, const char* name) {
  int overflow = 0;
  PyObject* index = PyNumber_Index(o);
  const long long v = index ? PyLong_AsLongLongAndOverflow(index, &overflow) : 0;
  if (!index) PyErr_Clear();
  if (!index || overflow || v < INT32_MIN || v > INT32_MAX) {
    Py_XDECREF(index);
    refuse("%s must be a whole number of 32 bits", name);
  }
  Py_DECREF(index);
  return static_cast<int>(v);
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? TRELLIS_F32 : t == at::kHalf ? TRELLIS_F16 : t == at::kBFloat16 ? TRELLIS_BF16 : -1;
}

int dtype_code(const at::Tensor& t, const char* name) {
  const int code = dtype_code(t.scalar_type());
  if (code < 0) refuse("%s dtype must be float32, float16 or bfloat16", name);
  return code;
}

// The dtype argument `o`, or (None) the one of `like`.
at::ScalarType dtype_or(PyObject* o, const at::Tensor& like, const char* name) {
  if (o == Py_None) return like.scalar_type();
  if (!THPDtype_Check(o)) refuse("%s must be a torch.dtype", name);
  const at::ScalarType t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  if (dtype_code(t) < 0) refuse("%s must be float32, float16 or bfloat16", name);
  return t;
}

bool on_gpu(const at::Tensor& t) { return t.is_cuda() && t.layout() == at::kStrided; }
int index_of(const at::Tensor& t) { return static_cast<int>(t.get_device()); }

void* stream_of(int device) { return c10::hip::getCurrentHIPStream(static_cast<c10::DeviceIndex>(device)).stream(); }

at::Tensor make(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
  return at::empty(sizes, like.options().dtype(dtype).requires_grad(false));
}

// A tensor that the call has written into: autograd counts such writes, so that a backward pass that saved the tensor
// before them raises an error. (Inference tensors have no count.)
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
void written(PyObject* o) {
  if (o != Py_None) written(THPVariable_Unpack(o));
}

// Sizes and type of a tensor that has to be dense and on the device.
void expect(const at::Tensor& t, const char* name, at::ScalarType dtype, at::IntArrayRef sizes, int device) {
  if (t.scalar_type() != dtype || t.sizes() != sizes || !t.is_contiguous() || !on_gpu(t) || index_of(t) != device)
    refuse("%s must be a contiguous %s tensor of sizes %s on device %d", name, at::toString(dtype),
           (std::string("[") + c10::Join(", ", sizes) + "]").c_str(), device);
}

template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused&) {
    return nullptr;
  } catch (const Status& s) {
    return PyLong_FromLong(s.code);
  } catch (...) {
    // torch's own errors as torch raises them (out of memory among them)
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
  }
}

void count(Py_ssize_t have, Py_ssize_t want, const char* name) {
  if (have != want) refuse("%s takes %d arguments", name, static_cast<int>(want));
}

// ---------------------------------------------------------------- norms

// [rows, width] with unit column stride.
at::Tensor as_rows(const at::Tensor& t) {
  at::Tensor r = t.dim() == 2 ? t : t.reshape({-1, t.size(-1)});
  return r.stride(1) == 1 || r.size(1) == 1 ? r : r.contiguous();
}

// x, residual, weight, post_weight, gate, scale, eps, out_dtype, residual_out -> (y, h)
PyObject* residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 9, "residual_norm");
    const at::Tensor& x = tensor(a[0], "x");
    const at::Tensor* residual = optional_tensor(a[1], "residual");
    const at::Tensor& weight = tensor(a[2], "weight");
    const at::Tensor* post = optional_tensor(a[3], "post_weight");
    const at::Tensor* gate = optional_tensor(a[4], "gate");
    const float scale = static_cast<float>(number(a[5], "scale")), eps = static_cast<float>(number(a[6], "eps"));
    if (!on_gpu(x)) refuse("the norms run on a GPU");
    if (x.dim() == 0) refuse("x must have at least one dim");
    const c10::DeviceGuard guard(x.device());   // launches go to the current device
    const int device = index_of(x), x_dt = dtype_code(x, "x");
    const at::ScalarType y_type = dtype_or(a[7], x, "out_dtype");
    const int64_t width = x.size(-1);
    expect(weight, "weight", at::kFloat, {width}, device);
    if (post) expect(*post, "post_weight", at::kFloat, {width}, device);
    if (x.numel() == 0 && width == 0) refuse("x must have a width");
    const at::Tensor x2 = as_rows(x);
    const int64_t rows = x2.size(0);

    at::Tensor r2, h, h2, g2;
    int r_dt = TRELLIS_F32;
    if (residual) {
      r_dt = dtype_code(*residual, "residual");
      if (residual->sizes() != x.sizes() || !on_gpu(*residual) || index_of(*residual) != device)
        refuse("residual must have x's sizes and device");
      r2 = as_rows(*residual);
      const at::Tensor* given = optional_tensor(a[8], "residual_out");
      if (given) {
        h = *given;
        if (h.sizes() != x.sizes() || h.scalar_type() != residual->scalar_type() || !on_gpu(h) || index_of(h) != device)
          refuse("residual_out must have the residual's sizes, dtype and device");
        h2 = h.dim() == 2 ? h : h.view({-1, width});
        if (h2.stride(1) != 1 && width != 1) refuse("residual_out must have unit column stride");
      } else {
        h = make(x.sizes(), residual->scalar_type(), x);
        h2 = h.dim() == 2 ? h : h.view({-1, width});
      }
    }
    int inner = 1;
    if (gate) {
      if (gate->scalar_type() != x.scalar_type() || !on_gpu(*gate) || index_of(*gate) != device)
        refuse("gate must have x's dtype and device");
      if (!at::is_expandable_to(gate->sizes(), x.sizes())) refuse("gate must broadcast against x");
      g2 = gate->sizes() == x.sizes() ? *gate : gate->expand(x.sizes());
      if (g2.dim() != 2) g2 = g2.reshape({-1, width});
      inner = g2.stride(1) == 0 || width == 1 ? 0 : 1;
      if (inner && g2.stride(1) != 1) g2 = g2.contiguous();
    }
    at::Tensor y = make(x.sizes(), y_type, x);
    check(entry.residual_norm(x2.const_data_ptr(), x2.stride(0), x_dt, residual ? r2.const_data_ptr() : nullptr,
                              residual ? r2.stride(0) : 0, r_dt, gate ? g2.const_data_ptr() : nullptr,
                              gate ? g2.stride(0) : 0, inner, post ? post->const_data_ptr<float>() : nullptr,
                              weight.const_data_ptr<float>(), scale, eps, residual ? h2.data_ptr() : nullptr,
                              residual ? h2.stride(0) : 0, y.data_ptr(), width, dtype_code(y_type), rows,
                              static_cast<int>(std::min<int64_t>(width, INT32_MAX)), stream_of(device)));
    if (residual) written(a[8]);
    if (!residual) return THPVariable_Wrap(std::move(y));
    PyObject* py = THPVariable_Wrap(std::move(y));
    PyObject* ph = a[8] == Py_None ? THPVariable_Wrap(std::move(h)) : Py_NewRef(a[8]);
    PyObject* pair = py && ph ? PyTuple_Pack(2, py, ph) : nullptr;
    Py_XDECREF(py);
    Py_XDECREF(ph);
    return pair;
  });
}

// ---------------------------------------------------------------- cache

struct CacheView {
  trellis_kv_cache c;
  int device;
};

// A call's cache (no table and lens: one that takes none); max_len None: all that the table can hold.
CacheView view_of(const at::Tensor& k, const at::Tensor& v, const at::Tensor* scores, const at::Tensor* pos,
                  const at::Tensor* table, const at::Tensor* lens, PyObject* max_len) {
  const bool rows = table != nullptr;
  if (!on_gpu(k)) refuse("the cache lives on a GPU");
  const int device = index_of(k);
  if (k.dim() != 4 || v.sizes() != k.sizes() || v.strides() != k.strides() || v.scalar_type() != k.scalar_type())
    refuse("k_pages and v_pages must be [pages, heads, page_size, head_dim], alike in dtype and strides");
  if (k.scalar_type() != at::kHalf && k.scalar_type() != at::kBFloat16) refuse("cache dtype must be float16 or bfloat16");
  if (k.stride(3) != 1) refuse("k_pages and v_pages must have unit stride over head_dim");
  if (rows && (table->scalar_type() != at::kInt || table->dim() != 2 || (table->stride(1) != 1 && table->size(1) != 1)))
    refuse("table must be int32 [rows, width] with unit column stride");
  if (!on_gpu(v) || index_of(v) != device || (rows && (!on_gpu(*table) || index_of(*table) != device)))
    refuse("k_pages, v_pages, table and lens must be on one device");
  const at::IntArrayRef plane = k.sizes().slice(0, 3);
  if (rows) expect(*lens, "lens", at::kInt, {table->size(0)}, device);
  if (scores) expect(*scores, "scores", at::kFloat, plane, device);
  if (pos) expect(*pos, "pos", at::kInt, plane, device);
  const int64_t height = rows ? table->size(0) : 0, width = rows ? table->size(1) : 1;
  for (const int64_t size : {k.size(0), k.size(1), k.size(2), k.size(3), height, width})
    if (size > INT32_MAX) refuse("the cache's sizes must fit 32 bits");
  CacheView w;
  w.device = device;
  w.c = {k.data_ptr(), v.data_ptr(), scores ? scores->data_ptr<float>() : nullptr, pos ? pos->data_ptr<int32_t>() : nullptr,
         rows ? table->const_data_ptr<int32_t>() : nullptr, rows ? lens->const_data_ptr<int32_t>() : nullptr, k.stride(0),
         k.stride(1), k.stride(2), rows ? table->stride(0) : 0, static_cast<int32_t>(k.size(0)), static_cast<int32_t>(k.size(1)),
         static_cast<int32_t>(k.size(2)), static_cast<int32_t>(k.size(3)), dtype_code(k.scalar_type()),
         static_cast<int32_t>(height), static_cast<int32_t>(width),
         max_len == Py_None ? static_cast<int32_t>(std::min<int64_t>(width * k.size(2), 1 << 30)) : whole(max_len, "max_len")};
  return w;
}

// k_pages, v_pages, scores, pos, table, lens of a call.
CacheView cache_view(PyObject* k_o, PyObject* v_o, PyObject* scores_o, PyObject* pos_o, PyObject* table_o, PyObject* lens_o,
                     PyObject* max_len) {
  const at::Tensor &k = tensor(k_o, "k_pages"), &v = tensor(v_o, "v_pages"), &table = tensor(table_o, "table"),
                   &lens = tensor(lens_o, "lens");
  return view_of(k, v, optional_tensor(scores_o, "scores"), optional_tensor(pos_o, "pos"), &table, &lens, max_len);
}

// Scratch of a call: the caller's, or a block of torch's allocator, which hands it on in stream order.
struct Scratch {
  at::Tensor own;
  void* p = nullptr;
  size_t bytes = 0;
  Scratch(PyObject* given, size_t need, const at::Tensor& like) {
    if (const at::Tensor* t = optional_tensor(given, "workspace")) {
      if (!on_gpu(*t) || index_of(*t) != index_of(like) || !t->is_contiguous())
        refuse("workspace must be contiguous on the cache's device");
      p = t->data_ptr();
      bytes = t->nbytes();
    } else if (need) {
      own = make({static_cast<int64_t>(need)}, at::kByte, like);
      p = own.data_ptr();
      bytes = need;
    }
  }
};

// [.., .., d] with unit stride over d.
at::Tensor as_heads(const at::Tensor& t) { return t.stride(2) == 1 || t.size(2) == 1 ? t : t.contiguous(); }

const int32_t* ints(PyObject* o, const char* name, int64_t n, int device) {
  const at::Tensor* t = optional_tensor(o, name);
  if (t) expect(*t, name, at::kInt, {n}, device);
  return t ? t->const_data_ptr<int32_t>() : nullptr;
}

// q, k, v, k_pages, v_pages, table, lens, starts, positions, q_norm, k_norm, eps, cos, sin, scores, pos, q_dtype -> q'
PyObject* append_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 17, "append_kv");
    const at::Tensor &q0 = tensor(a[0], "q"), &k0 = tensor(a[1], "k"), &v0 = tensor(a[2], "v");
    const CacheView w = cache_view(a[3], a[4], a[14], a[15], a[5], a[6], Py_None);
    const c10::DeviceGuard guard(THPVariable_Unpack(a[3]).device());
    const int64_t d = w.c.head_dim;
    if (q0.dim() != 3 || q0.size(2) != d) refuse("q must be [tokens, q_heads, %d]", static_cast<int>(d));
    const int64_t tokens = q0.size(0), hq = q0.size(1);
    if (tokens > INT32_MAX || hq > INT32_MAX) refuse("q's sizes must fit 32 bits");
    if (k0.sizes() != at::IntArrayRef({tokens, w.c.heads, d}) || v0.sizes() != k0.sizes())
      refuse("k and v must be [%lld, %d, %d]", static_cast<long long>(tokens), w.c.heads, static_cast<int>(d));
    for (const at::Tensor* t : {&q0, &k0, &v0})
      if (t->scalar_type() != q0.scalar_type() || !on_gpu(*t) || index_of(*t) != w.device)
        refuse("q, k and v must share a dtype on the cache's device");
    const int x_dt = dtype_code(q0, "q");
    const at::Tensor q = as_heads(q0), k = as_heads(k0), v = as_heads(v0);
    const at::Tensor *qw = optional_tensor(a[9], "q_norm"), *kw = optional_tensor(a[10], "k_norm");
    const at::Tensor *cos = optional_tensor(a[12], "cos"), *sin = optional_tensor(a[13], "sin");
    if (!qw != !kw || !cos != !sin) refuse("q_norm and k_norm, and cos and sin, go together");
    if (qw) {
      expect(*qw, "q_norm", at::kFloat, {d}, w.device);
      expect(*kw, "k_norm", at::kFloat, {d}, w.device);
    }
    int rot = 0, n_pos = 0;
    if (cos) {
      if (cos->dim() != 2 || cos->size(0) > INT32_MAX || cos->size(1) > INT16_MAX)
        refuse("cos and sin must be [positions, rotary dims / 2]");
      expect(*cos, "cos", at::kFloat, cos->sizes(), w.device);
      expect(*sin, "sin", at::kFloat, cos->sizes(), w.device);
      n_pos = static_cast<int>(cos->size(0));
      rot = 2 * static_cast<int>(cos->size(1));
    }
    const int32_t* starts = ints(a[7], "starts", static_cast<int64_t>(w.c.rows) + 1, w.device);
    const int32_t* positions = ints(a[8], "positions", tokens, w.device);
    const float eps = static_cast<float>(number(a[11], "eps"));
    const at::ScalarType out_type = dtype_or(a[16], q0, "q_dtype");
    at::Tensor out = make(q0.sizes(), out_type, q0);
    const auto f32 = [](const at::Tensor* t) { return t ? t->const_data_ptr<float>() : nullptr; };
    check(entry.kv_append(&w.c, q.const_data_ptr(), q.stride(0), q.stride(1), k.const_data_ptr(), k.stride(0), k.stride(1),
                          v.const_data_ptr(), v.stride(0), v.stride(1), x_dt, static_cast<int>(tokens), static_cast<int>(hq),
                          starts, positions, f32(qw), f32(kw), eps, f32(cos), f32(sin), rot, n_pos, out.data_ptr(),
                          dtype_code(out_type), stream_of(w.device)));
    for (const int i : {3, 4, 14, 15}) written(a[i]);
    return THPVariable_Wrap(std::move(out));
  });
}

// q, k_pages, v_pages, table, lens, scale, max_len, scores, out, out_dtype, workspace -> out
PyObject* paged_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 11, "paged_attention");
    const at::Tensor& q0 = tensor(a[0], "q");
    const CacheView w = cache_view(a[1], a[2], a[7], Py_None, a[3], a[4], a[6]);
    const c10::DeviceGuard guard(THPVariable_Unpack(a[1]).device());
    const int64_t d = w.c.head_dim;
    if (q0.dim() != 3 || q0.size(0) != w.c.rows || q0.size(2) != d || q0.size(1) > INT32_MAX || !on_gpu(q0) || index_of(q0) != w.device)
      refuse("q must be [%d, q_heads, %d] on the cache's device", w.c.rows, static_cast<int>(d));
    const int q_dt = dtype_code(q0, "q"), hq = static_cast<int>(q0.size(1)), accumulate = a[7] != Py_None;
    const at::Tensor q = as_heads(q0);
    const at::Tensor* given = optional_tensor(a[8], "out");
    at::Tensor out;
    if (given) {
      out = *given;
      if (out.sizes() != q0.sizes() || !out.is_contiguous() || !on_gpu(out) || index_of(out) != w.device)
        refuse("out must be contiguous with q's sizes and device");
    } else {
      out = make(q0.sizes(), dtype_or(a[9], q0, "out_dtype"), q0);
    }
    const int out_dt = dtype_code(out, "out");
    const double scale = a[5] == Py_None ? 1.0 / std::sqrt(static_cast<double>(d)) : number(a[5], "scale");
    size_t need = 0;
    check(entry.attention_workspace_bytes(&w.c, hq, accumulate, &need));
    const Scratch ws(a[10], need, q0);
    check(entry.paged_attention(&w.c, q.const_data_ptr(), q.stride(0), q.stride(1), q_dt, hq, static_cast<float>(scale),
                                accumulate, out.data_ptr(), out_dt, ws.p, ws.bytes, stream_of(w.device)));
    for (const int i : {7, 8, 10}) written(a[i]);
    return given ? Py_NewRef(a[8]) : THPVariable_Wrap(std::move(out));
  });
}

// k_pages, v_pages, scores, pos, table, lens, keep, recent, next_pos, out_table, max_len, workspace -> new lens
PyObject* evict_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 12, "evict_kv");
    const CacheView w = cache_view(a[0], a[1], a[2], a[3], a[4], a[5], a[10]);
    const c10::DeviceGuard guard(THPVariable_Unpack(a[0]).device());
    if (!w.c.scores || !w.c.pos) refuse("eviction goes by scores and pos");
    const int keep = whole(a[6], "keep"), recent = whole(a[7], "recent");
    const int32_t* next_pos = ints(a[8], "next_pos", w.c.rows, w.device);
    const at::Tensor* to = optional_tensor(a[9], "out_table");
    if (to && (to->scalar_type() != at::kInt || to->dim() != 2 || to->size(0) != w.c.rows || to->size(1) > INT32_MAX ||
               (to->stride(1) != 1 && to->size(1) != 1) || !on_gpu(*to) || index_of(*to) != w.device))
      refuse("out_table must be int32 [%d, width] with unit column stride on the cache's device", w.c.rows);
    const at::Tensor& lens = THPVariable_Unpack(a[5]);
    size_t need = 0;
    check(entry.evict_workspace_bytes(&w.c, keep, to != nullptr, &need));
    at::Tensor out = make(lens.sizes(), at::kInt, lens);
    const Scratch ws(a[11], need, lens);
    check(entry.kv_evict(&w.c, keep, recent, next_pos, to ? to->const_data_ptr<int32_t>() : nullptr, to ? to->stride(0) : 0,
                         to ? static_cast<int>(to->size(1)) : 0, out.data_ptr<int32_t>(), ws.p, ws.bytes, stream_of(w.device)));
    for (const int i : {0, 1, 2, 3, 11}) written(a[i]);
    return THPVariable_Wrap(std::move(out));
  });
}

// ---------------------------------------------------------------- several hypotheses

// q, k_pages, v_pages, table, lens, starts, parents, scale, max_len, out, out_dtype, workspace -> out
PyObject* tree_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 12, "tree_attention");
    const at::Tensor& q0 = tensor(a[0], "q");
    const CacheView w = cache_view(a[1], a[2], Py_None, Py_None, a[3], a[4], a[8]);
    const c10::DeviceGuard guard(THPVariable_Unpack(a[1]).device());
    const int64_t d = w.c.head_dim;
    if (q0.dim() != 3 || q0.size(2) != d || q0.size(0) > INT32_MAX || q0.size(1) > INT32_MAX || !on_gpu(q0) || index_of(q0) != w.device)
      refuse("q must be [tokens, q_heads, %d] on the cache's device", static_cast<int>(d));
    const int q_dt = dtype_code(q0, "q"), tokens = static_cast<int>(q0.size(0)), hq = static_cast<int>(q0.size(1));
    const int32_t* starts = ints(a[5], "starts", static_cast<int64_t>(w.c.rows) + 1, w.device);
    const int32_t* parents = ints(a[6], "parents", tokens, w.device);
    if (!starts && (w.c.rows == 0 ? tokens != 0 : tokens % w.c.rows != 0))
      refuse("without starts every row has the same number of tokens: %d are no multiple of %d rows", tokens, w.c.rows);
    const at::Tensor q = as_heads(q0);
    const at::Tensor* given = optional_tensor(a[9], "out");
    at::Tensor out;
    if (given) {
      out = *given;
      if (out.sizes() != q0.sizes() || !out.is_contiguous() || !on_gpu(out) || index_of(out) != w.device)
        refuse("out must be contiguous with q's sizes and device");
    } else {
      out = make(q0.sizes(), dtype_or(a[10], q0, "out_dtype"), q0);
    }
    const int out_dt = dtype_code(out, "out");
    const double scale = a[7] == Py_None ? 1.0 / std::sqrt(static_cast<double>(d)) : number(a[7], "scale");
    size_t need = 0;
    check(entry.tree_attention_workspace_bytes(&w.c, tokens, hq, q_dt, out_dt, &need));
    const Scratch ws(a[11], need, q0);
    check(entry.tree_attention(&w.c, q.const_data_ptr(), q.stride(0), q.stride(1), q_dt, tokens, hq, starts, parents,
                               static_cast<float>(scale), out.data_ptr(), out_dt, ws.p, ws.bytes, stream_of(w.device)));
    for (const int i : {9, 11}) written(a[i]);
    return given ? Py_NewRef(a[9]) : THPVariable_Wrap(std::move(out));
  });
}

// logits, scores, k, ended, end_token, workspace -> (scores, beams, tokens)
PyObject* beam_select(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 6, "beam_select");
    const at::Tensor &x0 = tensor(a[0], "logits"), &scores = tensor(a[1], "scores");
    const at::Tensor* ended = optional_tensor(a[3], "ended");
    if (!on_gpu(x0)) refuse("the selection runs on a GPU");
    const c10::DeviceGuard guard(x0.device());
    const int device = index_of(x0), x_dt = dtype_code(x0, "logits"), k = whole(a[2], "k"), end_token = whole(a[4], "end_token");
    if (x0.dim() != 3) refuse("logits must be [batch, beams, vocab]");
    const int64_t batch = x0.size(0), beams = x0.size(1), vocab = x0.size(2);
    if (batch > INT32_MAX || beams > INT32_MAX || vocab > INT32_MAX) refuse("the logits' sizes must fit 32 bits");
    expect(scores, "scores", at::kFloat, {batch, beams}, device);
    if (ended) expect(*ended, "ended", at::kBool, {batch, beams}, device);
    const at::Tensor x = as_heads(x0);
    size_t need = 0;
    check(entry.beam_workspace_bytes(static_cast<int>(batch), static_cast<int>(beams), static_cast<int>(vocab), k, &need));
    at::Tensor out = make({batch, k}, at::kFloat, x0), from = make({batch, k}, at::kInt, x0), token = make({batch, k}, at::kInt, x0);
    const Scratch ws(a[5], need, x0);
    check(entry.beam_select(x.const_data_ptr(), x.stride(0), x.stride(1), x_dt, static_cast<int>(batch), static_cast<int>(beams),
                            static_cast<int>(vocab), scores.const_data_ptr<float>(),
                            ended ? reinterpret_cast<const uint8_t*>(ended->const_data_ptr<bool>()) : nullptr, end_token, k,
                            out.data_ptr<float>(), from.data_ptr<int32_t>(), token.data_ptr<int32_t>(), ws.p, ws.bytes,
                            stream_of(device)));
    written(a[5]);
    PyObject* parts[3] = {THPVariable_Wrap(std::move(out)), THPVariable_Wrap(std::move(from)), THPVariable_Wrap(std::move(token))};
    PyObject* all = parts[0] && parts[1] && parts[2] ? PyTuple_Pack(3, parts[0], parts[1], parts[2]) : nullptr;
    for (PyObject* p : parts) Py_XDECREF(p);
    return all;
  });
}

// One cache a layer, of k_pages, v_pages, scores and pos (or None) as one layer's tensor, a list or tuple with one for each
// layer (None for a layer without scores or pos), or one tensor with the layers as its first dim. table and lens None: a
// call that takes none.
struct LayerViews {
  std::vector<trellis_kv_cache> c;
  std::vector<PyObject*> into;    // the tensors that the call writes into
  c10::Device where{c10::kCPU};
  int device = -1;

  LayerViews(PyObject* k, PyObject* v, PyObject* scores, PyObject* pos, PyObject* table_o, PyObject* lens_o) {
    const bool rows = table_o != Py_None || lens_o != Py_None;
    const at::Tensor *table = rows ? &tensor(table_o, "table") : nullptr, *lens = rows ? &tensor(lens_o, "lens") : nullptr;
    const bool listed = PyList_Check(k) || PyTuple_Check(k);
    if (!listed && tensor(k, "k_pages").dim() == 5) stacked(k, v, scores, pos, table, lens);
    else each(k, v, scores, pos, listed, table, lens);
  }

  void each(PyObject* k, PyObject* v, PyObject* scores, PyObject* pos, bool listed, const at::Tensor* table, const at::Tensor* lens) {
    PyObject* from[4] = {k, v, scores, pos};
    const char* names[4] = {"k_pages", "v_pages", "scores", "pos"};
    const Py_ssize_t layers = listed ? PySequence_Fast_GET_SIZE(k) : 1;
    if (layers < 1 || layers > INT16_MAX) refuse("k_pages must hold 1 to %d layers", INT16_MAX);
    for (int i = 1; i < 4; ++i) {
      const bool list = PyList_Check(from[i]) || PyTuple_Check(from[i]);
      if (from[i] != Py_None && (list ? PySequence_Fast_GET_SIZE(from[i]) != layers : layers != 1))
        refuse("%s must have as many layers as k_pages: %d", names[i], static_cast<int>(layers));
    }
    c.reserve(layers);
    into.reserve(4 * layers);
    for (Py_ssize_t l = 0; l < layers; ++l) {
      const at::Tensor* t[4];
      for (int i = 0; i < 4; ++i) {
        PyObject* o = PyList_Check(from[i]) || PyTuple_Check(from[i]) ? PySequence_Fast_GET_ITEM(from[i], l) : from[i];
        t[i] = i < 2 ? &tensor(o, names[i]) : optional_tensor(o, names[i]);
        if (t[i]) into.push_back(o);
      }
      take(view_of(*t[0], *t[1], t[2], t[3], table, lens, Py_None), *t[0]);
    }
  }

  void stacked(PyObject* k_o, PyObject* v_o, PyObject* scores_o, PyObject* pos_o, const at::Tensor* table, const at::Tensor* lens) {
    const at::Tensor &k = tensor(k_o, "k_pages"), &v = tensor(v_o, "v_pages");
    const at::Tensor *scores = optional_tensor(scores_o, "scores"), *pos = optional_tensor(pos_o, "pos");
    const int64_t layers = k.size(0);
    if (layers < 1 || layers > INT16_MAX) refuse("k_pages must hold 1 to %d layers", INT16_MAX);
    for (const at::Tensor* t : {&v, scores, pos})
      if (t && (t->dim() != (t == &v ? 5 : 4) || t->size(0) != layers))
        refuse("v_pages, scores and pos must hold the layers as k_pages does: %lld first", static_cast<long long>(layers));
    const auto first = [](const at::Tensor* t) { return t ? t->select(0, 0) : at::Tensor(); };
    const at::Tensor k0 = first(&k), v0 = first(&v), s0 = first(scores), p0 = first(pos);
    take(view_of(k0, v0, scores ? &s0 : nullptr, pos ? &p0 : nullptr, table, lens, Py_None), k0);
    c.reserve(layers);
    for (int64_t l = 1; l < layers; ++l) {
      trellis_kv_cache one = c[0];
      one.k = static_cast<char*>(one.k) + l * k.stride(0) * 2;
      one.v = static_cast<char*>(one.v) + l * v.stride(0) * 2;
      if (scores) one.scores += l * scores->stride(0);
      if (pos) one.pos += l * pos->stride(0);
      c.push_back(one);
    }
    for (PyObject* o : {k_o, v_o, scores_o, pos_o})
      if (o != Py_None) into.push_back(o);
  }

  void take(const CacheView& w, const at::Tensor& k) {
    if (!c.empty() && w.device != device) refuse("the layers must be on one device");
    device = w.device;
    where = k.device();
    c.push_back(w.c);
  }

  void all_written() const {
    for (PyObject* o : into) written(o);
  }
};

// k_pages, v_pages, src, dst, counts, scores, pos -> None
PyObject* copy_pages(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 7, "copy_pages");
    const LayerViews w(a[0], a[1], a[5], a[6], Py_None, Py_None);
    const at::Tensor& src = tensor(a[2], "src");
    const c10::DeviceGuard guard(w.where);
    if (src.dim() != 1 || src.size(0) > INT32_MAX) refuse("src must be int32 [n]");
    const int64_t pages = src.size(0);
    tensor(a[3], "dst");
    check(entry.kv_copy_pages(w.c.data(), static_cast<int>(w.c.size()), ints(a[2], "src", pages, w.device),
                              ints(a[3], "dst", pages, w.device), ints(a[4], "counts", pages, w.device),
                              static_cast<int>(pages), stream_of(w.device)));
    w.all_written();
    Py_RETURN_NONE;
  });
}

// k_pages, v_pages, table, lens, starts, path, scores, pos -> new lens
PyObject* keep_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    count(n, 8, "keep_kv");
    tensor(a[2], "table");
    const LayerViews w(a[0], a[1], a[6], a[7], a[2], a[3]);
    const c10::DeviceGuard guard(w.where);
    const at::Tensor &path = tensor(a[5], "path"), &lens = THPVariable_Unpack(a[3]);
    const int rows = w.c[0].rows;
    tensor(a[4], "starts");
    if (path.scalar_type() != at::kInt || path.dim() != 2 || path.size(0) != rows || path.size(1) > INT32_MAX ||
        (path.stride(1) != 1 && path.size(1) > 1) || !on_gpu(path) || index_of(path) != w.device)
      refuse("path must be int32 [%d, width] with unit column stride on the cache's device", rows);
    at::Tensor out = make(lens.sizes(), at::kInt, lens);
    check(entry.kv_keep(w.c.data(), static_cast<int>(w.c.size()), ints(a[4], "starts", static_cast<int64_t>(rows) + 1, w.device),
                        path.const_data_ptr<int32_t>(), path.stride(0), static_cast<int>(path.size(1)), out.data_ptr<int32_t>(),
                        stream_of(w.device)));
    w.all_written();
    return THPVariable_Wrap(std::move(out));
  });
}

// The addresses of the library's entry points, in the order of Entry.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    constexpr Py_ssize_t have = sizeof(Entry) / sizeof(void*);
    count(n, have, "bind");
    void* p[have];
    for (Py_ssize_t i = 0; i < have; ++i) {
      p[i] = PyLong_AsVoidPtr(a[i]);
      if (!p[i]) refuse("bind takes addresses");
    }
    static_assert(sizeof(p) == sizeof(entry), "every entry is one address");
    std::memcpy(&entry, p, sizeof(entry));
    Py_RETURN_NONE;
  });
}

#define METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {METHOD(bind), METHOD(residual_norm), METHOD(append_kv), METHOD(paged_attention), METHOD(evict_kv),
                         METHOD(tree_attention), METHOD(beam_select), METHOD(copy_pages), METHOD(keep_kv),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serve", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serve() { return PyModule_Create(&module); }
