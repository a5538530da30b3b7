// Python entry points of the 8-bit serving operators: a step's kernels run for a few
// microseconds, so the argument checks, output and workspace allocation and the launch
// happen in one C call each (through ctypes they took 15 to 25 us, here 4 to 7).  The
// work itself is libb200block.so's C ABI (include/b200_block.h).  A function returns
// its result, or the launcher's status (an int) if that is not B200_OK; arguments that
// do not fit raise ValueError, tensors off the current CUDA device RuntimeError.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>

#include "b200_block.h"

namespace {

constexpr int MAX_BATCH = 2048;
constexpr const char* CAPSULE = "b200.kv8";

struct Refused {  // a Python exception is set
};
[[noreturn]] void refuse(PyObject* type, const char* what) {
  PyErr_SetString(type, what);
  throw Refused{};
}
void need(bool ok, const char* what) {
  if (!ok) refuse(PyExc_ValueError, what);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) {
    PyErr_Format(PyExc_TypeError, "%s: a tensor expected", name);
    throw Refused{};
  }
  return THPVariable_Unpack(o);
}
const at::Tensor* maybe(PyObject* o, const char* name) { return o == Py_None ? nullptr : &tensor(o, name); }
long long whole(PyObject* o, const char* name) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Format(PyExc_TypeError, "%s: a whole number expected", name);
    throw Refused{};
  }
  if (v > 0x7fffffffLL || v < -0x7fffffffLL) refuse(PyExc_ValueError, "a size of 32 bits expected");
  return v;
}
bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Refused{};
  return v != 0;
}

void on_device(int device, const at::Tensor* t) {
  if (t && (!t->is_cuda() || t->get_device() != device))
    refuse(PyExc_RuntimeError, "libb200block kernels take CUDA tensors on one device only (no CPU fallback)");
}
void* stream_of(int device) {
  if (device < 0 || c10::cuda::current_device() != device)
    refuse(PyExc_RuntimeError, "the tensors' CUDA device is not the current one");
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}
int cuda_index(const at::Tensor& t) {
  if (!t.is_cuda())
    refuse(PyExc_RuntimeError, "libb200block kernels take CUDA tensors on one device only (no CPU fallback)");
  return t.get_device();
}
bool shaped(const at::Tensor& t, std::initializer_list<int64_t> sizes) { return t.sizes() == at::IntArrayRef(sizes); }
const int* index(const at::Tensor& t, int64_t n, const char* name) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) {
    PyErr_Format(PyExc_ValueError, "%s: contiguous int32 tensor with %lld entries expected", name, static_cast<long long>(n));
    throw Refused{};
  }
  return static_cast<const int*>(t.data_ptr());
}

struct Cache {
  B200KvCache8 c;
  int device;
  at::ScalarType type;
  at::Tensor hold[8];
};
Cache* cache_of(PyObject* o) {
  auto* c = static_cast<Cache*>(PyCapsule_GetPointer(o, CAPSULE));
  if (!c) throw Refused{};
  return c;
}

// runs f, turning refusals and C++ exceptions into Python ones
template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}
bool count(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", want, n);
  return false;
}

// cache(k_pages, v_pages, k_scale, v_scale, k_newest, v_newest, table, rows or None) -> capsule
PyObject* py_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &kp = tensor(a[0], "k_pages"), &vp = tensor(a[1], "v_pages"), &ks = tensor(a[2], "k_scale"),
                     &vs = tensor(a[3], "v_scale"), &kn = tensor(a[4], "k_newest"), &vn = tensor(a[5], "v_newest"),
                     &table = tensor(a[6], "table");
    const at::Tensor* rows = maybe(a[7], "rows");
    need(kp.dim() == 4 && kp.scalar_type() == at::kByte, "k_pages: uint8 [pages, kv_heads, P, D] expected");
    const int64_t N = kp.size(0), H = kp.size(1), P = kp.size(2), D = kp.size(3);
    need((P == 16 || P == 32 || P == 64 || P == 128) && (D == 32 || D == 64 || D == 128),
         "a page size of 16, 32, 64 or 128 and a head_dim of 32, 64 or 128 expected");
    need(vp.scalar_type() == at::kByte && shaped(vp, {N, H, P / 4, D, 4}), "v_pages: uint8 [pages, kv_heads, P/4, D, 4] expected");
    need(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && shaped(ks, {N, H}) && shaped(vs, {N, H}),
         "k_scale, v_scale: fp32 [pages, kv_heads] expected");
    need(kn.dim() == 5 && (kn.scalar_type() == at::kHalf || kn.scalar_type() == at::kBFloat16), "k_newest: fp16 or bf16 [rows, 2, kv_heads, P, D] expected");
    const int64_t M = kn.size(0);
    need(shaped(kn, {M, 2, H, P, D}), "k_newest: fp16 or bf16 [rows, 2, kv_heads, P, D] expected");
    need(vn.scalar_type() == kn.scalar_type() && shaped(vn, {M, 2, H, P / 4, D, 4}),
         "v_newest: k_newest's type, [rows, 2, kv_heads, P/4, D, 4] expected");
    need(table.dim() == 2 && table.scalar_type() == at::kInt, "table: int32 [batch, blocks] expected");
    const int64_t B = table.size(0), W = table.size(1);
    need(B >= 1 && B <= MAX_BATCH && W >= 1 && N >= 1 && M >= 1 && H >= 1,
         "a batch of 1 to 2048, at least one page, head, row and block expected");
    need(std::max({N, H, M, W}) <= 0x7fffffff, "sizes of 32 bits expected");
    need(rows || M >= B, "fewer rows of newest blocks than sequences");
    for (const at::Tensor* t : {&kp, &vp, &ks, &vs, &kn, &vn, &table}) need(t->is_contiguous(), "cache tensors must be contiguous");
    const int device = cuda_index(kp);
    for (const at::Tensor* t : {&vp, &ks, &vs, &kn, &vn, &table}) on_device(device, t);
    on_device(device, rows);
    auto* c = new Cache{{kp.data_ptr(), vp.data_ptr(), static_cast<float*>(ks.data_ptr()), static_cast<float*>(vs.data_ptr()),
                         kn.data_ptr(), vn.data_ptr(), static_cast<const int*>(table.data_ptr()), nullptr, static_cast<int>(N),
                         static_cast<int>(H), static_cast<int>(P), static_cast<int>(D), static_cast<int>(M),
                         static_cast<int>(W), static_cast<int>(B), kn.scalar_type() == at::kBFloat16},
                        device, kn.scalar_type(), {kp, vp, ks, vs, kn, vn, table, rows ? *rows : at::Tensor()}};
    PyObject* capsule = PyCapsule_New(c, CAPSULE, [](PyObject* o) { delete static_cast<Cache*>(PyCapsule_GetPointer(o, CAPSULE)); });
    if (!capsule) {
      delete c;
      return nullptr;
    }
    if (rows) {
      try {
        c->c.rows = index(*rows, B, "rows");
      } catch (const Refused&) {
        Py_DECREF(capsule);
        throw;
      }
    }
    return capsule;
  });
}

// append(cache, qkv, cu, start, heads, cos, sin, interleaved, out) -> q
PyObject* py_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 9)) return nullptr;
  return guarded([&]() -> PyObject* {
    Cache* c = cache_of(a[0]);
    const at::Tensor &qkv = tensor(a[1], "qkv"), &cu = tensor(a[2], "cu"), &start = tensor(a[3], "start");
    const long long heads = whole(a[4], "heads");
    const at::Tensor *cos = maybe(a[5], "cos"), *sin = maybe(a[6], "sin"), *given = maybe(a[8], "out");
    const bool interleaved = truth(a[7]);
    const int64_t D = c->c.head_dim;
    need(heads > 0 && heads % c->c.kv_heads == 0, "heads: a multiple of the cache's key heads expected");
    const int64_t width = (heads + 2 * c->c.kv_heads) * D;
    need(qkv.dim() == 2 && qkv.size(1) == width && qkv.scalar_type() == c->type,
         "qkv: the cache's 16-bit type, [tokens, (heads + 2 kv_heads) * D] expected");
    const int64_t tokens = qkv.size(0);
    int64_t ld = width;
    if (tokens > 1) ld = qkv.stride(0);
    need(tokens == 0 || (qkv.stride(1) == 1 && ld % 8 == 0 && ld >= width),
         "qkv: dense rows that start 16-byte aligned and do not overlap expected");
    need(tokens <= 0x7fffffff, "sizes of 32 bits expected");
    int64_t rot = 0, turns = 0;
    if (cos || sin) {
      need(cos && sin && cos->dim() == 2 && cos->sizes() == sin->sizes() && cos->scalar_type() == at::kFloat &&
               sin->scalar_type() == at::kFloat && cos->is_contiguous() && sin->is_contiguous(),
           "cos, sin: both or neither, contiguous fp32 [positions, rot / 2] expected");
      turns = cos->size(0);
      rot = 2 * cos->size(1);
      need(turns > 0 && turns <= 0x7fffffff && rot > 0 && rot % 16 == 0 && rot <= D,
           "rotated channels: a multiple of 16 up to head_dim expected");
    }
    for (const at::Tensor* t : {&qkv, &cu, &start, cos, sin, given}) on_device(c->device, t);
    const int *pc = index(cu, c->c.batch + 1, "cu"), *ps = index(start, c->c.batch, "start");
    void* st = stream_of(c->device);
    at::Tensor out;
    if (given) {
      need(shaped(*given, {tokens, heads, D}) && given->scalar_type() == c->type && given->is_contiguous(),
           "out: contiguous, qkv's type, [tokens, heads, D] expected");
      out = *given;
    } else {
      out = at::empty({tokens, heads, D}, qkv.options());
    }
    const int rc = b200_kv8_append(&c->c, qkv.data_ptr(), ld, out.data_ptr(), pc, ps,
                                   cos ? static_cast<const float*>(cos->data_ptr()) : nullptr,
                                   sin ? static_cast<const float*>(sin->data_ptr()) : nullptr, static_cast<int>(rot), interleaved,
                                   static_cast<int>(turns), static_cast<int>(tokens), static_cast<int>(heads), st);
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(out));
  });
}

// read(cache, cu, start, lens, total) -> (k, v)
PyObject* py_read(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 5)) return nullptr;
  return guarded([&]() -> PyObject* {
    Cache* c = cache_of(a[0]);
    const at::Tensor &cu = tensor(a[1], "cu"), &start = tensor(a[2], "start"), &lens = tensor(a[3], "lens");
    const long long total = whole(a[4], "total");
    need(total >= 0, "total: the number of rows expected");
    for (const at::Tensor* t : {&cu, &start, &lens}) on_device(c->device, t);
    const int *pc = index(cu, c->c.batch + 1, "cu"), *ps = index(start, c->c.batch, "start"), *pl = index(lens, c->c.batch, "lens");
    void* st = stream_of(c->device);
    at::Tensor k = at::empty({total, c->c.kv_heads, c->c.head_dim}, c->hold[4].options());
    at::Tensor v = at::empty({total, c->c.kv_heads, c->c.head_dim}, c->hold[4].options());
    const int rc = b200_kv8_read(&c->c, pc, ps, pl, k.data_ptr(), v.data_ptr(), static_cast<int>(total), st);
    if (rc) return PyLong_FromLong(rc);
    PyObject *x = THPVariable_Wrap(std::move(k)), *y = THPVariable_Wrap(std::move(v));
    PyObject* both = x && y ? PyTuple_Pack(2, x, y) : nullptr;
    Py_XDECREF(x);
    Py_XDECREF(y);
    return both;
  });
}

// the row stride of [tokens, heads, D], whose heads lie side by side
int64_t row_stride(const at::Tensor& t) {
  const int64_t n = t.size(0), h = t.size(1), d = t.size(2), ld = t.stride(0);
  need(t.stride(2) == 1 && (h == 1 || t.stride(1) == d) && (n <= 1 || (ld % 8 == 0 && ld >= h * d)),
       "q, out: the heads of a token must be dense, and rows start 16-byte aligned and not overlap");
  return n > 1 ? ld : h * d;
}

// attend(cache, q, cu, lens, max_q_len, scale or None, out or None) -> out
PyObject* py_attend(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 7)) return nullptr;
  return guarded([&]() -> PyObject* {
    Cache* c = cache_of(a[0]);
    const at::Tensor &q = tensor(a[1], "q"), &cu = tensor(a[2], "cu"), &lens = tensor(a[3], "lens");
    const long long most = whole(a[4], "max_q_len");
    const at::Tensor* given = maybe(a[6], "out");
    const int64_t D = c->c.head_dim;
    need(q.dim() == 3 && q.size(2) == D && q.scalar_type() == c->type, "q: the cache's 16-bit type, [tokens, heads, D] expected");
    const int64_t tokens = q.size(0), heads = q.size(1);
    need(heads > 0 && heads % c->c.kv_heads == 0, "heads: a multiple of the cache's key heads expected");
    need(most >= 1 || tokens == 0, "max_q_len: at least 1 expected");
    need(tokens <= 0x7fffffff && heads <= 0x7fffffff, "sizes of 32 bits expected");
    double scale = 1 / std::sqrt(static_cast<double>(D));
    if (a[5] != Py_None) {
      scale = PyFloat_AsDouble(a[5]);
      if (scale == -1.0 && PyErr_Occurred()) throw Refused{};
    }
    const int64_t ld_q = row_stride(q);
    for (const at::Tensor* t : {&q, &cu, &lens, given}) on_device(c->device, t);
    const int *pc = index(cu, c->c.batch + 1, "cu"), *pl = index(lens, c->c.batch, "lens");
    void* st = stream_of(c->device);
    at::Tensor out;
    int64_t ld_out = heads * D;
    if (given) {
      need(given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type(), "out: q's shape and type expected");
      out = *given;
      ld_out = row_stride(out);
    } else {
      out = at::empty({tokens, heads, D}, q.options());
    }
    const size_t bytes = b200_kv8_attention_workspace_bytes(c->c.batch, static_cast<int>(heads), c->c.kv_heads, static_cast<int>(D),
                                                            static_cast<int>(most));
    const at::Tensor ws = at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte));
    const int rc = b200_kv8_attention(&c->c, q.data_ptr(), ld_q, out.data_ptr(), ld_out, pc, pl, static_cast<int>(tokens),
                                      static_cast<int>(heads), static_cast<int>(most), static_cast<float>(scale), ws.data_ptr(),
                                      bytes, st);
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(out));
  });
}

int type_code(at::ScalarType t) { return t == at::kHalf ? 0 : t == at::kBFloat16 ? 1 : t == at::kFloat ? 2 : -1; }

// linear_i8(x, w, w_scale, bias, gelu, resid, out_dtype or None, out or None) -> out
PyObject* py_linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count(n, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor &x = tensor(a[0], "x"), &w = tensor(a[1], "w"), &ws = tensor(a[2], "w_scale");
    const at::Tensor *bias = maybe(a[3], "bias"), *resid = maybe(a[5], "resid"), *given = maybe(a[7], "out");
    const bool gelu = truth(a[4]);
    const int xt = type_code(x.scalar_type());
    need(x.dim() == 2 && xt >= 0, "x: fp16, bf16 or fp32 [m, k] expected");
    const int64_t m = x.size(0), k = x.size(1);
    need(k >= 1 && (x.stride(1) == 1 || k == 1) && (x.stride(0) >= k || m <= 1), "x: dense rows that do not overlap expected");
    need(w.dim() == 2 && w.scalar_type() == at::kChar && w.size(1) >= k && w.size(1) < k + 16 && w.stride(1) == 1 &&
             w.stride(0) % 16 == 0,
         "w: int8 [n, k rounded up to 16] with a row pitch that is a multiple of 16 expected");
    const int64_t N = w.size(0);
    need(m <= 0x7fffffff && k <= 0x7fffffff && N <= 0x7fffffff, "sizes of 32 bits expected");
    need(ws.scalar_type() == at::kFloat && shaped(ws, {N}) && ws.is_contiguous(), "w_scale: contiguous fp32 [n] expected");
    need(!bias || (bias->scalar_type() == at::kFloat && shaped(*bias, {N}) && bias->is_contiguous()),
         "bias: contiguous fp32 [n] expected");
    at::ScalarType type = x.scalar_type();
    if (a[6] != Py_None) {
      if (!THPDtype_Check(a[6])) refuse(PyExc_TypeError, "out_dtype: a torch.dtype expected");
      type = reinterpret_cast<THPDtype*>(a[6])->scalar_type;
    }
    int64_t ld_r = N;
    if (resid) {
      need(!gelu && (a[6] == Py_None || type == at::kFloat), "with resid the result is fp32, and there is no GELU");
      need(resid->scalar_type() == at::kFloat && shaped(*resid, {m, N}) && (resid->stride(1) == 1 || N == 1) &&
               (resid->stride(0) >= N || m <= 1),
           "resid: fp32 [m, n] with dense rows expected");
      type = at::kFloat;
      ld_r = std::max(resid->stride(0), N);
    }
    const int ot = type_code(type);
    need(ot >= 0, "out_dtype: fp16, bf16 or fp32 expected");
    const int device = cuda_index(x);
    for (const at::Tensor* t : {&w, &ws, bias, resid, given}) on_device(device, t);
    void* st = stream_of(device);
    at::Tensor out;
    int64_t ld_out = N;
    if (given) {
      need(shaped(*given, {m, N}) && given->scalar_type() == type && (given->stride(1) == 1 || N == 1) &&
               (given->stride(0) >= N || m <= 1),
           "out: the result's type, [m, n] with dense rows expected");
      out = *given;
      ld_out = std::max(out.stride(0), N);
    } else {
      out = at::empty({m, N}, x.options().dtype(type));
    }
    const size_t bytes = b200_linear_i8_workspace_bytes(static_cast<int>(m), static_cast<int>(k));
    at::Tensor space;
    if (bytes) space = at::empty({static_cast<int64_t>(bytes)}, x.options().dtype(at::kByte));
    B200LinearI8Args p{};
    p.x = x.data_ptr();
    p.w = w.data_ptr();
    p.w_scale = static_cast<const float*>(ws.data_ptr());
    p.bias = bias ? static_cast<const float*>(bias->data_ptr()) : nullptr;
    p.resid = resid ? static_cast<const float*>(resid->data_ptr()) : nullptr;
    p.out = out.data_ptr();
    p.ld_x = std::max(x.stride(0), k);
    p.ld_w = w.stride(0);
    p.ld_resid = ld_r;
    p.ld_out = ld_out;
    p.m = static_cast<int>(m);
    p.n = static_cast<int>(N);
    p.k = static_cast<int>(k);
    p.x_type = xt;
    p.out_type = ot;
    p.gelu = gelu;
    p.workspace = bytes ? space.data_ptr() : nullptr;
    p.workspace_bytes = bytes;
    const int rc = b200_linear_i8(&p, st);
    return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(std::move(out));
  });
}

#define FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"cache", FAST(py_cache), nullptr},   {"append", FAST(py_append), nullptr},
                         {"read", FAST(py_read), nullptr},     {"attend", FAST(py_attend), nullptr},
                         {"linear_i8", FAST(py_linear), nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b200serving", "8-bit serving operators", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b200serving() { return PyModule_Create(&module); }
