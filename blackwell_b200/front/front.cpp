// Torch front end of the rotary and cache entry points: checks tensors and calls
// the C ABI (include/bw_attn.h) on the current CUDA stream.  A CPython module
// (blackwell_b200/_front.so) and not Python code because the checks of a decode
// step's calls cost more there than the launches: 4 to 6 us a call against 0.3.
//
// Every function takes its arguments by position and returns the entry point's
// status code; what is wrong with a tensor raises ValueError or TypeError before
// anything touches the device.  blackwell_b200/cache.py documents the arguments.
#include <Python.h>

#include <initializer_list>
#include <string>

#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <ATen/core/grad_mode.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/bw_attn.h"

namespace {

using at::Tensor;

struct Refused {};   // a Python exception is set

[[noreturn]] void refuse(PyObject* type, const std::string& what) {
  PyErr_SetString(type, what.c_str());
  throw Refused{};
}

std::string shape_of(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}
std::string shape_of(std::initializer_list<int64_t> n) {
  std::string s = "[";
  for (auto it = n.begin(); it != n.end(); ++it) s += (it != n.begin() ? ", " : "") + std::to_string(*it);
  return s + "]";
}

// Tensor argument; None gives nullptr where it is allowed.
const Tensor* tensor(PyObject* o, const char* name, bool or_none = false) {
  if (or_none && o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a tensor");
  return &THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  return v;
}
int int32(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse(PyExc_ValueError, std::string(name) + " is out of range");
  return (int)v;
}
int truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused{};
  return v;
}

void want(const char* name, const Tensor& t, at::ScalarType dtype, std::initializer_list<int64_t> shape) {
  if (t.scalar_type() != dtype)
    refuse(PyExc_TypeError, std::string(name) + " must be " + c10::toString(dtype) + ", got " + c10::toString(t.scalar_type()));
  if (!t.sizes().equals(c10::IntArrayRef(shape)) || !t.is_contiguous())
    refuse(PyExc_ValueError, std::string(name) + " must be a contiguous " + shape_of(shape) + " tensor, got " + shape_of(t));
}

// The current stream of the current device, on which every tensor given lies.
void* stream_for(std::initializer_list<const Tensor*> tensors) {
  int dev = -1;
  for (const Tensor* t : tensors)
    if (t) {
      if (!t->is_cuda())
        refuse(PyExc_ValueError, "expected CUDA tensors, got a " + shape_of(*t) + " tensor on " + t->device().str());
      const int d = (int)t->get_device();
      if (dev >= 0 && d != dev)
        refuse(PyExc_ValueError, "the tensors are on different devices (" + std::to_string(dev) + " and " + std::to_string(d) + ")");
      dev = d;
    }
  const int now = (int)c10::cuda::current_device();
  if (dev >= 0 && dev != now)
    refuse(PyExc_ValueError, "the tensors are on device " + std::to_string(dev) + ", the current device is " + std::to_string(now));
  return c10::cuda::getCurrentCUDAStream().stream();
}

void* ptr(const Tensor* t) { return t ? t->data_ptr() : nullptr; }

void want_table(const Tensor& t) {
  if (t.scalar_type() != at::kFloat || t.dim() != 2 || !t.is_contiguous())
    refuse(PyExc_ValueError, "cos_sin_cache must be a contiguous fp32 [length, rotary_dim] tensor");
}
int small(const char* name, int64_t v) {
  if (v < 0 || v > INT32_MAX) refuse(PyExc_ValueError, std::string(name) + " is out of range");
  return (int)v;
}

// ------------------------------------------------------------------ the functions

double real(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{};
  return v;
}

// rope_table(out, first, kind, and the eight numbers of bw_rope_scaling in their order)
int rope_table(PyObject* const* a) {
  const Tensor* out = tensor(a[0], "out");
  if (out->dim() != 2) refuse(PyExc_ValueError, "out must be [length, rotary_dim]");
  want("out", *out, at::kFloat, {out->size(0), out->size(1)});
  bw_rope_scaling s{int32(a[2], "kind"), real(a[3]), real(a[4]), real(a[5]), real(a[6]), real(a[7]), real(a[8]), real(a[9]),
                    real(a[10])};
  void* stream = stream_for({out});
  return bw_rope_table(static_cast<float*>(ptr(out)), out->size(0), small("rotary_dim", out->size(1)), integer(a[1]), &s,
                       stream);
}

// Strides of the (b, h, s) axes of a [B, H, S, D] tensor; of [tokens, H, D]: B =
// tokens and S = 1, or, where the positions are 0, 1, ..., B = 1 and S = tokens.
void bhs(const char* name, const Tensor& t, bool one_sequence, int64_t* st) {
  const int64_t n = t.dim();
  if (t.stride(n - 1) != 1 && t.size(n - 1) > 1)
    refuse(PyExc_ValueError, std::string(name) + " must have a contiguous last dimension");
  st[0] = one_sequence ? 0 : t.stride(0);
  st[1] = t.stride(1);
  st[2] = n == 4 ? t.stride(2) : one_sequence ? t.stride(0) : 0;
}

// Status of rope where gradients are on and an argument requires them: the call is
// left to the caller's autograd function.  No status of the C ABI is negative.
constexpr int kWantsGradient = -1;

// rope(q, q_out, k, k_out, cos_sin_cache, positions, pos_offset, interleaved, inverse)
int rope(PyObject* const* a) {
  const Tensor *q = tensor(a[0], "q"), *q_out = tensor(a[1], "q_out"), *k = tensor(a[2], "k", true),
               *k_out = tensor(a[3], "k_out", true), *table = tensor(a[4], "cos_sin_cache"),
               *positions = tensor(a[5], "positions", true);
  if (at::GradMode::is_enabled())
    for (const Tensor* t : {q, k, table, q_out, k_out})
      if (t && t->requires_grad()) return kWantsGradient;
  const int64_t nd = q->dim();
  if (nd != 3 && nd != 4) refuse(PyExc_ValueError, "q must be [B, H, S, D] or [tokens, H, D], got " + shape_of(*q));
  const auto dtype = q->scalar_type();
  if (dtype != at::kBFloat16 && dtype != at::kFloat)
    refuse(PyExc_TypeError, std::string("q must be bfloat16 or float32, got ") + c10::toString(dtype));
  want_table(*table);
  const bool one = nd == 3 && !positions;
  const int64_t Hq = q->size(1), D = q->size(nd - 1);
  const int64_t B = one ? 1 : q->size(0), S = nd == 4 ? q->size(2) : one ? q->size(0) : 1;
  const auto same = [&](const char* name, const Tensor& t, const Tensor& ref) {
    if (t.scalar_type() != ref.scalar_type() || !t.sizes().equals(ref.sizes()))
      refuse(PyExc_ValueError, std::string(name) + " must be a " + c10::toString(ref.scalar_type()) + " " + shape_of(ref) + " tensor");
  };
  same("q_out", *q_out, *q);
  if (!k != !k_out) refuse(PyExc_ValueError, "k_out without k");
  int64_t Hkv = 0, qs[3], qos[3], ks[3], kos[3];
  if (k) {
    bool ok = k->dim() == nd && k->scalar_type() == dtype;
    for (int64_t i = 0; ok && i < nd; ++i) ok = i == 1 || k->size(i) == q->size(i);
    if (!ok) refuse(PyExc_ValueError, "k must be like q but for the number of heads, got " + shape_of(*k) + " beside " + shape_of(*q));
    same("k_out", *k_out, *k);
    Hkv = k->size(1);
    bhs("k", *k, one, ks);
    bhs("k_out", *k_out, one, kos);
  }
  bhs("q", *q, one, qs);
  bhs("q_out", *q_out, one, qos);
  if (positions) {
    if (nd == 4) want("positions", *positions, at::kInt, {B, S});
    else want("positions", *positions, at::kInt, {B});
  }
  if (q->numel() == 0 && k && k->numel() != 0) refuse(PyExc_ValueError, "q has no heads: give the tensor that has as q");
  void* stream = stream_for({q, k, table, positions, q_out, k_out});
  if (q->numel() == 0) return BW_OK;
  return bw_rope(ptr(q), ptr(q_out), ptr(k), ptr(k_out), dtype == at::kBFloat16 ? BW_BF16 : BW_F32, small("B", B),
                 small("Hq", Hq), small("Hkv", Hkv), small("S", S), small("D", D), qs, qos, k ? ks : nullptr,
                 k ? kos : nullptr, static_cast<const float*>(ptr(table)), table->size(0),
                 small("rotary_dim", table->size(1)), static_cast<const int*>(ptr(positions)), int32(a[6], "pos_offset"),
                 truth(a[7]), truth(a[8]), stream);
}

struct Cache {
  int dtype, num_pages, page_size, Hkv, D;
};
Cache cache_of(const Tensor& k, const Tensor& v, const Tensor* scales) {
  const auto t = k.scalar_type();
  if (k.dim() != 4 || (t != at::kBFloat16 && t != at::kFloat8_e4m3fn))
    refuse(PyExc_ValueError, "k_cache must be a bfloat16 or float8_e4m3fn [num_pages, page_size, Hkv, D] tensor");
  if (!k.is_contiguous()) refuse(PyExc_ValueError, "k_cache must be contiguous");
  want("v_cache", v, t, {k.size(0), k.size(1), k.size(2), k.size(3)});
  Cache c{t == at::kBFloat16 ? BW_BF16 : BW_E4M3, small("num_pages", k.size(0)), small("page_size", k.size(1)),
          small("Hkv", k.size(2)), small("D", k.size(3))};
  if (c.dtype == BW_BF16) {
    if (scales) refuse(PyExc_ValueError, "a bfloat16 cache has no scales");
  } else {
    if (!scales) refuse(PyExc_ValueError, "a float8_e4m3fn cache needs scales");
    want("scales", *scales, at::kByte, {c.num_pages, c.Hkv, 2, c.page_size});
  }
  return c;
}

// kv_cache_write(k, v, k_cache, v_cache, slots, scales, cos_sin_cache, positions, interleaved)
int kv_cache_write(PyObject* const* a) {
  const Tensor *k = tensor(a[0], "k"), *v = tensor(a[1], "v"), *kc = tensor(a[2], "k_cache"),
               *vc = tensor(a[3], "v_cache"), *slots = tensor(a[4], "slots"), *scales = tensor(a[5], "scales", true),
               *table = tensor(a[6], "cos_sin_cache", true), *positions = tensor(a[7], "positions", true);
  const Cache c = cache_of(*kc, *vc, scales);
  if (k->dim() != 3 || k->size(1) != c.Hkv || k->size(2) != c.D || !v->sizes().equals(k->sizes()))
    refuse(PyExc_ValueError, "k and v must be [tokens, " + std::to_string(c.Hkv) + ", " + std::to_string(c.D) + "], got " +
                                 shape_of(*k) + " and " + shape_of(*v));
  if (k->scalar_type() != at::kBFloat16 || v->scalar_type() != at::kBFloat16)
    refuse(PyExc_TypeError, "k and v must be bfloat16");
  if (k->stride(2) != 1 || v->stride(2) != 1) refuse(PyExc_ValueError, "k and v must have a contiguous last dimension");
  const int64_t T = k->size(0);
  want("slots", *slots, at::kLong, {T});
  if (table) {
    want_table(*table);
    if (!positions) refuse(PyExc_ValueError, "cos_sin_cache needs positions");
    want("positions", *positions, at::kInt, {T});
  } else if (positions) {
    refuse(PyExc_ValueError, "positions need cos_sin_cache");
  }
  void* stream = stream_for({k, v, kc, vc, slots, scales, table, positions});
  const int64_t ks[2] = {k->stride(0), k->stride(1)}, vs[2] = {v->stride(0), v->stride(1)};
  return bw_kv_cache_write(ptr(k), ptr(v), ks, vs, small("tokens", T), c.Hkv, c.D, ptr(kc), ptr(vc),
                           static_cast<uint8_t*>(ptr(scales)), c.dtype, c.page_size, c.num_pages,
                           static_cast<const int64_t*>(ptr(slots)), static_cast<const float*>(ptr(table)),
                           table ? table->size(0) : 0, table ? small("rotary_dim", table->size(1)) : 0,
                           static_cast<const int*>(ptr(positions)), truth(a[8]), stream);
}

int table_width(const Tensor& bt, int64_t B) {
  if (bt.dim() != 2) refuse(PyExc_ValueError, "block_table must be [B, max_pages]");
  want("block_table", bt, at::kInt, {B, bt.size(1)});
  return small("max_pages", bt.size(1));
}

// kv_cache_read(k_cache, v_cache, block_table, kv_lens, out_offsets, scales, kv_starts, k_out, v_out)
int kv_cache_read(PyObject* const* a) {
  const Tensor *kc = tensor(a[0], "k_cache"), *vc = tensor(a[1], "v_cache"), *bt = tensor(a[2], "block_table"),
               *lens = tensor(a[3], "kv_lens"), *offs = tensor(a[4], "out_offsets"),
               *scales = tensor(a[5], "scales", true), *starts = tensor(a[6], "kv_starts", true),
               *k_out = tensor(a[7], "k_out"), *v_out = tensor(a[8], "v_out");
  const Cache c = cache_of(*kc, *vc, scales);
  const int64_t B = lens->numel();
  const int width = table_width(*bt, B);
  want("kv_lens", *lens, at::kInt, {B});
  want("out_offsets", *offs, at::kLong, {B});
  if (starts) want("kv_starts", *starts, at::kInt, {B});
  if (k_out->dim() != 3) refuse(PyExc_ValueError, "k_out must be [total_rows, Hkv, D]");
  want("k_out", *k_out, at::kBFloat16, {k_out->size(0), c.Hkv, c.D});
  want("v_out", *v_out, at::kBFloat16, {k_out->size(0), c.Hkv, c.D});
  void* stream = stream_for({kc, vc, bt, lens, offs, scales, starts, k_out, v_out});
  return bw_kv_cache_read(ptr(kc), ptr(vc), static_cast<const uint8_t*>(ptr(scales)), c.dtype, c.page_size, c.num_pages,
                          static_cast<const int*>(ptr(bt)), width, static_cast<const int*>(ptr(lens)),
                          static_cast<const int*>(ptr(starts)), static_cast<const int64_t*>(ptr(offs)), small("B", B),
                          c.Hkv, c.D, ptr(k_out), ptr(v_out), k_out->size(0), stream);
}

// gqa_decode_paged_fp8(q, k_cache, v_cache, scales, block_table, kv_lens, scale, workspace, out, lse)
int gqa_decode_paged_fp8(PyObject* const* a) {
  const Tensor *q = tensor(a[0], "q"), *kc = tensor(a[1], "k_cache"), *vc = tensor(a[2], "v_cache"),
               *scales = tensor(a[3], "scales", true), *bt = tensor(a[4], "block_table"), *lens = tensor(a[5], "kv_lens"),
               *ws = tensor(a[7], "workspace"), *out = tensor(a[8], "out"), *lse = tensor(a[9], "lse");
  const Cache c = cache_of(*kc, *vc, scales);
  if (c.dtype != BW_E4M3)
    refuse(PyExc_TypeError, "k_cache and v_cache must be float8_e4m3fn (gqa_decode_paged reads a bfloat16 cache)");
  if (q->dim() != 3 || q->size(2) != c.D) refuse(PyExc_ValueError, "q must be [B, Hq, " + std::to_string(c.D) + "], got " + shape_of(*q));
  const int64_t B = q->size(0), Hq = q->size(1);
  want("q", *q, at::kBFloat16, {B, Hq, c.D});
  const int width = table_width(*bt, B);
  want("kv_lens", *lens, at::kInt, {B});
  want("out", *out, at::kBFloat16, {B, Hq, c.D});
  want("lse", *lse, at::kFloat, {B, Hq});
  if (!ws->is_contiguous()) refuse(PyExc_ValueError, "workspace must be contiguous");
  const double scale = real(a[6]);
  void* stream = stream_for({q, kc, vc, scales, bt, lens, ws, out, lse});
  if (B == 0) return BW_OK;   // no sequence
  return bw_gqa_decode_paged_fp8(ptr(q), ptr(kc), ptr(vc), static_cast<const uint8_t*>(ptr(scales)),
                                 static_cast<const int*>(ptr(bt)), static_cast<const int*>(ptr(lens)), ptr(out),
                                 static_cast<float*>(ptr(lse)), small("B", B), small("Hq", Hq), c.Hkv, c.D, c.page_size,
                                 c.num_pages, width, (float)scale, ptr(ws), ws->nbytes(), stream);
}

// No exception leaves the module: Refused has set a Python one, others become RuntimeError.
template <int (*F)(PyObject* const*), int N>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "expected %d arguments, got %zd", N, n);
    return nullptr;
  }
  try {
    return PyLong_FromLong(F(args));
  } catch (const Refused&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown error");
  }
  return nullptr;
}

#define BW_METHOD(f, n) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&call<f, n>)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {BW_METHOD(rope_table, 11), BW_METHOD(rope, 9), BW_METHOD(kv_cache_write, 9),
                         BW_METHOD(kv_cache_read, 9), BW_METHOD(gqa_decode_paged_fp8, 10), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_front", "Checked calls of the rotary and cache entry points.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

// BW_FRONT_TORCH: the torch version of the build (its C++ types are not another version's).
extern "C" __attribute__((visibility("default"))) PyObject* PyInit__front() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_with_torch", BW_FRONT_TORCH) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
