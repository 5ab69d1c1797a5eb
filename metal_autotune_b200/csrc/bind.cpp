// Native binding of the paged-serving entry points (include/mt.h): argument
// checks, output allocation and the call, without a detour through ctypes.
//
// These operators run once per layer of every decode step, where the call
// itself is what a small batch waits for: on the host that measured it the
// ctypes wrapper of mt_paged_sdpa_decode took 19.3 us a call (3.3 us of it
// torch.cuda.current_stream(), 2.5 us each output allocation, 2.9 us the
// conversion of 26 arguments), the launch itself 4.2 us.
//
// Each function takes positional arguments from its wrapper in lib.py and
// returns its outputs, or the entry point's error code as an int, which the
// wrapper turns into MTError. Argument errors are ValueError / TypeError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <initializer_list>

#include "../../include/mt.h"

namespace {

struct Raised {};  // a Python exception is set

[[noreturn]] void raise(PyObject* type, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  PyErr_FormatV(type, fmt, ap);
  va_end(ap);
  throw Raised();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) raise(PyExc_TypeError, "%s must be a tensor", name);
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* name) {
  return o == Py_None ? nullptr : &tensor(o, name);
}
int64_t integer(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    raise(PyExc_TypeError, "%s must be an integer", name);
  }
  return v;
}
float number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return static_cast<float>(v);
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised();
  return v != 0;
}

const char* type_name(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kFloat: return "torch.float32";
    case at::kInt: return "torch.int32";
    case at::kLong: return "torch.int64";
    default: return c10::toString(t);
  }
}
int code_of(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MT_BF16;
    case at::kHalf: return MT_F16;
    case at::kFloat: return MT_F32;
    default: raise(PyExc_TypeError, "dtype %s is not built for this operator", type_name(t));
  }
}

std::string shape_text(at::IntArrayRef s) {
  std::string out = "(";
  for (size_t i = 0; i < s.size(); ++i) out += (i ? ", " : "") + std::to_string(s[i]);
  return out + ")";
}

// dense, of this type and shape
void want(const at::Tensor& t, const char* name, at::ScalarType dt, at::IntArrayRef shape) {
  if (t.scalar_type() != dt) raise(PyExc_TypeError, "%s must be %s, got %s", name, type_name(dt), type_name(t.scalar_type()));
  if (t.sizes() != shape)
    raise(PyExc_ValueError, "%s must have shape %s, got %s", name, shape_text(shape).c_str(), shape_text(t.sizes()).c_str());
  if (!t.is_contiguous()) raise(PyExc_ValueError, "%s must be row-contiguous", name);
}

// every tensor on the current CUDA device
int on_device(std::initializer_list<const at::Tensor*> ts) {
  for (const at::Tensor* t : ts)
    if (t && !t->is_cuda())
      raise(PyExc_ValueError, "libmt kernels take CUDA tensors; got a tensor on %s", t->device().str().c_str());
  const int dev = c10::cuda::current_device();
  for (const at::Tensor* t : ts)
    if (t && t->get_device() != dev)
      raise(PyExc_ValueError, "a tensor is on cuda:%d, the current device is cuda:%d", (int)t->get_device(), dev);
  return dev;
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType dt, int dev) {
  return at::detail::empty_cuda(shape, dt, c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(dev)), std::nullopt);
}

// Several outputs in one allocation, each at a multiple of 16 bytes: an
// allocation of its own costs each of them about a microsecond.
struct Outputs {
  at::Tensor base;
  int64_t at = 0;
  static int64_t room(int64_t n, size_t size) { return (n * static_cast<int64_t>(size) + 15) & ~int64_t{15}; }
  Outputs(int64_t bytes, int dev) : base(empty({bytes}, at::kByte, dev)) {}
  at::Tensor take(at::IntArrayRef shape, at::ScalarType dt) {
    const size_t size = c10::elementSize(dt);
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(),
                                                            c10::scalarTypeToTypeMeta(dt));
    t.unsafeGetTensorImpl()->set_storage_offset(at / static_cast<int64_t>(size));
    t.unsafeGetTensorImpl()->set_sizes_contiguous(shape);
    at += room(t.numel(), size);
    return t;
  }
};

template <typename T = void>
T* ptr(const at::Tensor* t) {
  return t ? static_cast<T*>(t->data_ptr()) : nullptr;
}
template <typename T = void>
T* ptr(const at::Tensor& t) {
  return static_cast<T*>(t.data_ptr());
}
mt_stream_t stream(int dev) {
  return reinterpret_cast<mt_stream_t>(c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream());
}

// the step of a dimension, 0 where it has one entry (its stride then says nothing)
int64_t step(const at::Tensor& t, int d) { return t.size(d) > 1 ? t.stride(d) : 0; }

struct Table {
  int64_t stride, width;
};
Table block_table(const at::Tensor& t, int64_t B) {
  if (t.scalar_type() != at::kInt || t.dim() != 2 || t.size(0) != B || (t.size(1) > 1 && t.stride(1) != 1))
    raise(PyExc_ValueError, "block_table must be int32 [%lld, max_pages] with contiguous rows", (long long)B);
  return {t.size(0) > 1 ? t.stride(0) : t.size(1), t.size(1)};
}

struct Cache {
  int64_t pages, heads, page_size, D, page_stride, head_stride, slot_stride;
};
Cache cache(const at::Tensor& k, const at::Tensor& v, at::ScalarType dt) {
  if (k.dim() != 4 || k.sizes() != v.sizes() || k.strides() != v.strides())
    raise(PyExc_ValueError, "k_cache and v_cache must be [pages, Hkv, page_size, D] of one shape and strides");
  if (k.scalar_type() != dt || v.scalar_type() != dt)
    raise(PyExc_TypeError, "the caches must be %s, as q", type_name(dt));
  if (k.stride(3) != 1 && k.size(3) > 1) raise(PyExc_ValueError, "the caches' rows (D) must be contiguous");
  return {k.size(0), k.size(1), k.size(2), k.size(3), step(k, 0), step(k, 1), step(k, 2)};
}

PyObject* tuple(std::initializer_list<const at::Tensor*> ts) {
  PyObject* out = PyTuple_New(static_cast<Py_ssize_t>(ts.size()));
  if (!out) throw Raised();
  Py_ssize_t i = 0;
  for (const at::Tensor* t : ts) {
    PyObject* o = t ? THPVariable_Wrap(*t) : Py_NewRef(Py_None);
    if (!o) {
      Py_DECREF(out);
      throw Raised();
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

// entries of an `out` tuple
PyObject* item(PyObject* out, Py_ssize_t i) {
  if (!PyTuple_Check(out) || PyTuple_GET_SIZE(out) <= i) raise(PyExc_TypeError, "out must be the operator's result tuple");
  return PyTuple_GET_ITEM(out, i);
}

// ctx_lens, new_lens, block_table, free_pages, page_size, token_cap, free_head, out
PyObject* paged_plan(PyObject* const* a) {
  const at::Tensor &ctx = tensor(a[0], "ctx_lens"), &fresh = tensor(a[1], "new_lens"), &table = tensor(a[2], "block_table"),
                   &pages = tensor(a[3], "free_pages");
  const int64_t page_size = integer(a[4], "page_size"), cap = integer(a[5], "token_cap");
  const at::Tensor* head = maybe(a[6], "free_head");
  if (ctx.dim() != 1) raise(PyExc_ValueError, "ctx_lens must be [B]");
  const int64_t B = ctx.size(0);
  want(ctx, "ctx_lens", at::kInt, {B});
  want(fresh, "new_lens", at::kInt, {B});
  want(pages, "free_pages", at::kInt, {pages.numel()});
  if (head) want(*head, "free_head", at::kInt, {1});
  const Table tb = block_table(table, B);
  if (cap < 0) raise(PyExc_ValueError, "token_cap must not be negative");
  at::Tensor o[6];
  static const char* names[6] = {"out.seq_lens", "out.query_start", "out.positions", "out.token_seq", "out.slots", "out.counts"};
  const int64_t sizes[6] = {B, B + 1, cap, cap, cap, 5};
  if (a[7] != Py_None)
    for (int i = 0; i < 6; ++i) {
      o[i] = tensor(item(a[7], i), names[i]);
      want(o[i], names[i], i == 4 ? at::kLong : at::kInt, {sizes[i]});
    }
  const int dev = on_device({&ctx, &fresh, &table, &pages, head});
  if (a[7] == Py_None) {
    int64_t bytes = 0;
    for (int i = 0; i < 6; ++i) bytes += Outputs::room(sizes[i], i == 4 ? 8 : 4);
    Outputs out(bytes, dev);
    for (int i = 0; i < 6; ++i) o[i] = out.take({sizes[i]}, i == 4 ? at::kLong : at::kInt);
  } else
    on_device({&o[0], &o[1], &o[2], &o[3], &o[4], &o[5]});
  const int rc = mt_paged_plan(ptr<int32_t>(ctx), ptr<int32_t>(fresh), B, ptr<int32_t>(table), tb.stride, tb.width,
                               ptr<int32_t>(pages), pages.numel(), ptr<int32_t>(head), page_size, cap, ptr<int32_t>(o[0]),
                               ptr<int32_t>(o[1]), ptr<int32_t>(o[2]), ptr<int32_t>(o[3]), ptr<int64_t>(o[4]),
                               ptr<int32_t>(o[5]), stream(dev));
  if (rc) return PyLong_FromLong(rc);
  if (a[7] != Py_None) return Py_NewRef(a[7]);
  return tuple({&o[0], &o[1], &o[2], &o[3], &o[4], &o[5]});
}

// q, k, v, positions, slots, k_cache, v_cache, inv_freq, traditional, mscale, q_norm_w, k_norm_w, eps, out, k_out
PyObject* rope_paged_append(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v"), &pos = tensor(a[3], "positions"),
                   &slots = tensor(a[4], "slots"), &kc = tensor(a[5], "k_cache"), &vc = tensor(a[6], "v_cache"),
                   &inv = tensor(a[7], "inv_freq");
  const at::Tensor *qw = maybe(a[10], "q_norm_w"), *kw = maybe(a[11], "k_norm_w"), *out = maybe(a[13], "out"),
                   *k_out = maybe(a[14], "k_out");
  if (q.dim() != 3 || k.dim() != 3) raise(PyExc_ValueError, "q must be [T, Hq, D], k and v [T, Hkv, D]");
  const int64_t T = q.size(0), Hq = q.size(1), D = q.size(2), Hkv = k.size(1);
  const at::ScalarType dt = q.scalar_type();
  if (k.size(0) != T || k.size(2) != D || v.sizes() != k.sizes() || k.scalar_type() != dt || v.scalar_type() != dt)
    raise(PyExc_ValueError, "k and v must be %s [%lld, Hkv, %lld]", type_name(dt), (long long)T, (long long)D);
  if (D > 1 && (q.stride(2) != 1 || k.stride(2) != 1 || v.stride(2) != 1))
    raise(PyExc_ValueError, "q, k and v must have D contiguous");
  const Cache c = cache(kc, vc, dt);
  if (c.heads != Hkv || c.D != D)
    raise(PyExc_ValueError, "the caches must be [pages, %lld, page_size, %lld]", (long long)Hkv, (long long)D);
  want(pos, "positions", at::kInt, {T});
  want(slots, "slots", at::kLong, {T});
  want(inv, "inv_freq", at::kFloat, {inv.numel()});
  if (qw) want(*qw, "q_norm_w", dt, {D});
  if (kw) want(*kw, "k_norm_w", dt, {D});
  if (out && (out->sizes() != q.sizes() || out->scalar_type() != dt || (D > 1 && out->stride(2) != 1)))
    raise(PyExc_ValueError, "out must have q's shape and dtype with D contiguous");
  if (k_out) want(*k_out, "k_out", dt, {T, Hkv, D});
  const int dtype = code_of(dt);
  const int dev = on_device({&q, &k, &v, &pos, &slots, &kc, &vc, &inv, qw, kw, out, k_out});
  const at::Tensor y = out ? *out : empty({T, Hq, D}, dt, dev);
  const int rc = mt_rope_paged_append(
      ptr(q), ptr(k), ptr(v), step(q, 0), step(q, 1), step(k, 0), step(k, 1), step(v, 0), step(v, 1), ptr(qw), ptr(kw),
      number(a[12]), ptr<int32_t>(pos), ptr<int64_t>(slots), ptr<float>(inv), static_cast<int>(2 * inv.numel()),
      truth(a[8]), number(a[9]), ptr(y), step(y, 0), step(y, 1), ptr(k_out), ptr(kc), ptr(vc), c.pages, c.page_size,
      c.page_stride, c.head_stride, c.slot_stride, T, Hq, Hkv, D, dtype, stream(dev));
  if (rc) return PyLong_FromLong(rc);
  return out ? Py_NewRef(a[13]) : THPVariable_Wrap(y);
}

// q, k_cache, v_cache, block_table, seq_lens, scale, out, workspace buffer
PyObject* paged_sdpa_decode(PyObject* const* a) {
  const at::Tensor &q = tensor(a[0], "q"), &kc = tensor(a[1], "k_cache"), &vc = tensor(a[2], "v_cache"),
                   &table = tensor(a[3], "block_table"), &lens = tensor(a[4], "seq_lens"), &ws = tensor(a[7], "workspace");
  const at::Tensor* out = maybe(a[6], "out");
  if (q.dim() != 3) raise(PyExc_ValueError, "q must be [B, Hq, D]");
  const int64_t B = q.size(0), Hq = q.size(1), D = q.size(2);
  const at::ScalarType dt = q.scalar_type();
  const Cache c = cache(kc, vc, dt);
  if (c.D != D) raise(PyExc_ValueError, "the caches must be [pages, Hkv, page_size, %lld]", (long long)D);
  if (D > 1 && q.stride(2) != 1) raise(PyExc_ValueError, "q must have D contiguous");
  const Table tb = block_table(table, B);
  want(lens, "seq_lens", at::kInt, {B});
  if (out && (out->sizes() != q.sizes() || out->scalar_type() != dt || (D > 1 && out->stride(2) != 1)))
    raise(PyExc_ValueError, "out must have q's shape and dtype with D contiguous");
  const int dtype = code_of(dt);
  const int dev = on_device({&q, &kc, &vc, &table, &lens, out, &ws});
  const at::Tensor o = out ? *out : empty({B, Hq, D}, dt, dev);
  const int rc = mt_paged_sdpa_decode(ptr(q), step(q, 0), step(q, 1), ptr(kc), ptr(vc), c.pages, c.page_size, c.page_stride,
                                      c.head_stride, c.slot_stride, ptr<int32_t>(table), tb.stride, tb.width,
                                      ptr<int32_t>(lens), ptr(o), step(o, 0), step(o, 1), B, Hq, c.heads, D, number(a[5]),
                                      dtype, ptr(ws), static_cast<size_t>(ws.nbytes()), stream(dev));
  if (rc) return PyLong_FromLong(rc);
  return out ? Py_NewRef(a[6]) : THPVariable_Wrap(o);
}

// logits, tokens, top_k, out
PyObject* token_logprobs(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "logits");
  const at::Tensor* tokens = maybe(a[1], "tokens");
  const int64_t k = integer(a[2], "top_k");
  if (x.dim() != 2 || (x.size(1) > 1 && x.stride(1) != 1)) raise(PyExc_ValueError, "logits must be [R, V] with contiguous rows");
  const int64_t R = x.size(0), V = x.size(1);
  if (tokens) want(*tokens, "tokens", at::kInt, {R});
  if (k < 0) raise(PyExc_ValueError, "top_k must not be negative");
  const int dtype = code_of(x.scalar_type());
  at::Tensor lp, entropy, lse, ids, top;
  if (a[3] != Py_None) {
    if (tokens) {
      lp = tensor(item(a[3], 0), "out.logprob");
      want(lp, "out.logprob", at::kFloat, {R});
    }
    entropy = tensor(item(a[3], 1), "out.entropy");
    want(entropy, "out.entropy", at::kFloat, {R});
    lse = tensor(item(a[3], 2), "out.lse");
    want(lse, "out.lse", at::kFloat, {R});
    ids = tensor(item(a[3], 3), "out.top_ids");
    want(ids, "out.top_ids", at::kInt, {R, k});
    top = tensor(item(a[3], 4), "out.top_logprobs");
    want(top, "out.top_logprobs", at::kFloat, {R, k});
  }
  const int dev = on_device({&x, tokens});
  if (a[3] != Py_None) {
    on_device({tokens ? &lp : nullptr, &entropy, &lse, &ids, &top});
  } else {
    Outputs out((tokens ? 3 : 2) * Outputs::room(R, 4) + 2 * Outputs::room(R * k, 4), dev);
    if (tokens) lp = out.take({R}, at::kFloat);
    entropy = out.take({R}, at::kFloat);
    lse = out.take({R}, at::kFloat);
    ids = out.take({R, k}, at::kInt);
    top = out.take({R, k}, at::kFloat);
  }
  const int rc = mt_token_logprobs(ptr(x), R > 1 ? x.stride(0) : V, ptr<int32_t>(tokens), R, V,
                                   static_cast<int>(k < 1000 ? k : 1000), tokens ? ptr<float>(lp) : nullptr,
                                   ptr<float>(entropy), ptr<float>(lse), ptr<int32_t>(ids), ptr<float>(top), dtype,
                                   stream(dev));
  if (rc) return PyLong_FromLong(rc);
  if (a[3] != Py_None) return Py_NewRef(a[3]);
  return tuple({tokens ? &lp : nullptr, &entropy, &lse, &ids, &top});
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != N) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", N, n);
    return nullptr;
  }
  try {
    return F(args);
  } catch (const Raised&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

template <PyObject* (*F)(PyObject* const*), Py_ssize_t N>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<F, N>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<paged_plan, 8>("paged_plan"), method<rope_paged_append, 15>("rope_paged_append"),
                         method<paged_sdpa_decode, 8>("paged_sdpa_decode"), method<token_logprobs, 4>("token_logprobs"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "mt_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_mt_bind() { return PyModule_Create(&module); }
