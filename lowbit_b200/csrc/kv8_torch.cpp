// The torch side of the paged 8-bit KV cache's Python calls: argument checks,
// allocation of outputs and workspace, stream, and the C ABI call
// (include/lowbit_b200.h: lbc_kv8_*). A decode step calls these once a layer;
// the same in Python costs as much host time as the kernels take.
//
// The library's entry points are handed over as addresses (init), so that the
// module uses the one copy of the library that the process has loaded.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/lowbit_b200.h"

namespace {

decltype(&lbc_kv8_append) f_append;
decltype(&lbc_kv8_attention) f_attention;
decltype(&lbc_kv8_attention_workspace) f_workspace;
decltype(&lbc_kv8_read) f_read;
decltype(&lbc_last_error) f_error;

struct Refused {
  std::string why;
};
[[noreturn]] void refuse(const char *why) { throw Refused{why}; }
inline void need(bool ok, const char *why) {
  if (!ok) refuse(why);
}

// a tensor argument; None gives nullptr where `optional`
const at::Tensor *tensor(PyObject *o, const char *why, bool optional = false) {
  if (optional && o == Py_None) return nullptr;
  need(THPVariable_Check(o), why);
  return &THPVariable_Unpack(o);
}

int dtype_id(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return LBC_F32;
    case at::kBFloat16: return LBC_BF16;
    case at::kHalf: return LBC_F16;
    default: return -1;
  }
}

inline bool aligned(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

struct Rows {
  const int32_t *table, *pos, *starts;
  int width, B, N, most;
};

long as_long(PyObject *o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{""};
  return v;
}

Rows rows_of(const c10::Device &dev, int64_t n, PyObject *o_table, PyObject *o_pos, PyObject *o_starts, PyObject *o_most) {
  const char *w_table = "table must be a contiguous int32 [B, pages] tensor on the cache's device";
  const char *w_pos = "pos must be a contiguous int32 [B] tensor on the cache's device";
  const char *w_starts = "starts must be a contiguous int32 [B + 1] tensor on the cache's device";
  const at::Tensor &t = *tensor(o_table, w_table), &p = *tensor(o_pos, w_pos);
  need(t.dim() == 2 && t.scalar_type() == at::kInt && t.is_contiguous() && t.device() == dev, w_table);
  const int64_t b = t.size(0), width = t.size(1);
  need(p.dim() == 1 && p.size(0) == b && p.scalar_type() == at::kInt && p.is_contiguous() && p.device() == dev, w_pos);
  need(b > 0 && width > 0 && b <= 65535 && width <= 0x7fffffff, "table must hold at least one sequence and one page");
  need(n <= 0x7fffffff, "too many rows");
  Rows r{t.const_data_ptr<int32_t>(), p.const_data_ptr<int32_t>(), nullptr, (int)width, (int)b, (int)n, 0};
  const at::Tensor *s = tensor(o_starts, w_starts, true);
  const long given = o_most == Py_None ? -1 : as_long(o_most);
  need(o_most == Py_None || given >= 0, "max_tokens must not be negative");
  if (!s) {
    need(n % b == 0, "the rows do not divide over the sequences; give starts");
    r.most = (int)(n / b);
    need(o_most == Py_None || given >= r.most, "max_tokens is below the rows of a sequence");
  } else {
    need(s->dim() == 1 && s->size(0) == b + 1 && s->scalar_type() == at::kInt && s->is_contiguous() && s->device() == dev, w_starts);
    r.starts = s->const_data_ptr<int32_t>();
    r.most = o_most == Py_None ? (int)n : (int)std::min<int64_t>(given, n);
  }
  return r;
}

const lbc_kv8 *pool(PyObject *o) { return static_cast<const lbc_kv8 *>(PyLong_AsVoidPtr(o)); }

c10::Device device(PyObject *o) { return c10::Device(c10::kCUDA, (c10::DeviceIndex)as_long(o)); }

void *stream(const c10::Device &d) { return c10::cuda::getCurrentCUDAStream(d.index()).stream(); }

PyObject *status_error(int rc, const char *what) {
  PyErr_Format(rc == LBC_ERR_SHAPE || rc == LBC_ERR_PARAMS ? PyExc_ValueError : PyExc_RuntimeError, "%s failed (rc=%d): %s", what, rc,
               f_error());
  return nullptr;
}

template <typename F>
PyObject *guarded(F &&f) {
  try {
    return f();
  } catch (const Refused &e) {
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, e.why.c_str());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

PyObject *init(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 5) return PyErr_Format(PyExc_TypeError, "init takes 5 addresses");
  f_append = reinterpret_cast<decltype(f_append)>(PyLong_AsVoidPtr(a[0]));
  f_attention = reinterpret_cast<decltype(f_attention)>(PyLong_AsVoidPtr(a[1]));
  f_workspace = reinterpret_cast<decltype(f_workspace)>(PyLong_AsVoidPtr(a[2]));
  f_read = reinterpret_cast<decltype(f_read)>(PyLong_AsVoidPtr(a[3]));
  f_error = reinterpret_cast<decltype(f_error)>(PyLong_AsVoidPtr(a[4]));
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

// append(pool, device, qkv, table, pos, cos, sin, bias, starts, max_tokens, out)
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 11) return PyErr_Format(PyExc_TypeError, "append takes 11 arguments");
  return guarded([&]() -> PyObject * {
    const lbc_kv8 *c = pool(a[0]);
    const c10::Device dev = device(a[1]);
    const int kv = c->kv_heads, d = c->head_dim;
    const char *w_qkv = "qkv must be an fp32, bf16 or fp16 [N, (H + 2*KV)*D] tensor on the cache's device";
    const at::Tensor &x = *tensor(a[2], w_qkv);
    const int dt = dtype_id(x);
    need(x.dim() == 2 && dt >= 0 && x.device() == dev, w_qkv);
    const int64_t rows = x.size(0), w = x.size(1), heads = w / d - 2 * kv;
    need(w % d == 0 && heads > 0 && heads % kv == 0, "qkv's columns are not (H + 2*KV)*D with H a multiple of the KV heads");
    const char *w_tab = "cos and sin must be contiguous fp32 [positions, head_dim/2] tensors on the cache's device";
    const at::Tensor &cos = *tensor(a[5], w_tab), &sin = *tensor(a[6], w_tab);
    need(cos.dim() == 2 && cos.size(1) * 2 == d && cos.scalar_type() == at::kFloat && cos.is_contiguous() && cos.device() == dev, w_tab);
    need(sin.sizes() == cos.sizes() && sin.scalar_type() == at::kFloat && sin.is_contiguous() && sin.device() == dev, w_tab);
    need(aligned(cos.const_data_ptr()) && aligned(sin.const_data_ptr()), "cos and sin must be 16-byte aligned");
    const char *w_bias = "bias must be a contiguous fp32 tensor of qkv's width";
    const at::Tensor *bias = tensor(a[7], w_bias, true);
    need(!bias || (bias->dim() == 1 && bias->size(0) == w && bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->device() == dev),
         w_bias);
    const Rows r = rows_of(dev, rows, a[3], a[4], a[8], a[9]);
    const at::Tensor *given = tensor(a[10], "out must be a tensor", true);
    const int64_t shape[3] = {rows, heads, d};
    need(!given || (given->sizes() == c10::IntArrayRef(shape, 3) && given->scalar_type() == x.scalar_type() && given->device() == dev &&
                    given->is_contiguous() && aligned(given->const_data_ptr())),
         "out must be a contiguous, 16-byte aligned [N, H, D] tensor of qkv's type");
    const c10::cuda::OptionalCUDAGuard guard(dev);
    at::Tensor y = given ? *given : at::empty(c10::IntArrayRef(shape, 3), x.options());
    if (rows == 0) return THPVariable_Wrap(y);
    const bool fits = x.stride(1) == 1 && x.stride(0) >= w && aligned(x.const_data_ptr()) && x.stride(0) * x.element_size() % 16 == 0;
    const at::Tensor src = fits ? x : x.clone(at::MemoryFormat::Contiguous);
    const int rc = f_append(c, dt, src.const_data_ptr(), src.stride(0), bias ? bias->const_data_ptr<float>() : nullptr,
                            cos.const_data_ptr<float>(), sin.const_data_ptr<float>(), (int)std::min<int64_t>(cos.size(0), 0x7fffffff), r.table, r.width,
                            r.pos, r.starts, r.B, r.N, r.most, (int)heads, y.mutable_data_ptr(), stream(dev));
    return rc < 0 ? status_error(rc, "lbc_kv8_append") : THPVariable_Wrap(std::move(y));
  });
}

// attention(pool, device, q, table, pos, starts, max_tokens, window, scale, out); scale None: 1/sqrt(D)
PyObject *attention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 10) return PyErr_Format(PyExc_TypeError, "attention takes 10 arguments");
  return guarded([&]() -> PyObject * {
    const lbc_kv8 *c = pool(a[0]);
    const c10::Device dev = device(a[1]);
    const int kv = c->kv_heads, d = c->head_dim;
    const char *w_q = "q must be an fp32, bf16 or fp16 [N, H, D] tensor of the cache's head_dim on its device";
    const at::Tensor &q = *tensor(a[2], w_q);
    const int dt = dtype_id(q);
    need(q.dim() == 3 && dt >= 0 && q.size(2) == d && q.device() == dev, w_q);
    const int64_t rows = q.size(0), heads = q.size(1);
    need(heads > 0 && heads % kv == 0, "the query heads are not a multiple of the KV heads");
    const long window = as_long(a[7]);
    need(window >= 0, "window must not be negative");
    double scale = 1.0 / std::sqrt((double)d);
    if (a[8] != Py_None) {
      scale = PyFloat_AsDouble(a[8]);
      if (PyErr_Occurred()) return nullptr;
    }
    const Rows r = rows_of(dev, rows, a[3], a[4], a[5], a[6]);
    const at::Tensor *given = tensor(a[9], "out must be a tensor", true);
    need(!given || (given->sizes() == q.sizes() && given->scalar_type() == q.scalar_type() && given->device() == dev &&
                    given->is_contiguous() && aligned(given->const_data_ptr())),
         "out must be a contiguous, 16-byte aligned tensor of q's shape and type");
    const c10::cuda::OptionalCUDAGuard guard(dev);
    at::Tensor y = given ? *given : at::empty(q.sizes(), q.options());
    if (rows == 0) return THPVariable_Wrap(y);
    const bool fits = q.stride(2) == 1 && q.stride(1) == d && q.stride(0) >= heads * d && aligned(q.const_data_ptr()) &&
                      q.stride(0) * q.element_size() % 16 == 0;
    const at::Tensor src = fits ? q : q.clone(at::MemoryFormat::Contiguous);
    const int win = (int)std::min<long>(window, 0x7fffffff);
    const size_t bytes = f_workspace(c, dt, r.width, r.B, r.N, r.most, (int)heads, win);
    // from torch's allocator: private to this call in stream order, and to a graph when captured
    at::Tensor ws;
    if (bytes) ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
    const int rc = f_attention(c, dt, src.const_data_ptr(), src.stride(0), r.table, r.width, r.pos, r.starts, r.B, r.N, r.most, (int)heads, win,
                               (float)scale, y.mutable_data_ptr(), bytes ? ws.mutable_data_ptr() : nullptr, bytes, stream(dev));
    return rc < 0 ? status_error(rc, "lbc_kv8_attention") : THPVariable_Wrap(std::move(y));
  });
}

// read(pool, device, pages, dtype id) -> (k, v)
PyObject *read(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 4) return PyErr_Format(PyExc_TypeError, "read takes 4 arguments");
  return guarded([&]() -> PyObject * {
    const lbc_kv8 *c = pool(a[0]);
    const c10::Device dev = device(a[1]);
    const char *w_ids = "pages must be a contiguous int32 tensor of ids on the cache's device";
    const at::Tensor &ids = *tensor(a[2], w_ids);
    need(ids.dim() == 1 && ids.scalar_type() == at::kInt && ids.is_contiguous() && ids.device() == dev, w_ids);
    const long dt = as_long(a[3]);
    const at::ScalarType type = dt == LBC_F32 ? at::kFloat : dt == LBC_BF16 ? at::kBFloat16 : at::kHalf;
    const c10::cuda::OptionalCUDAGuard guard(dev);
    const auto opts = ids.options().dtype(type);
    at::Tensor k = at::empty({ids.size(0), c->kv_heads, c->page, c->head_dim}, opts), v = at::empty(k.sizes(), opts);
    if (ids.size(0)) {
      need(ids.size(0) <= 0x7fffffff, "too many pages");
      const int rc = f_read(c, (int)dt, ids.const_data_ptr<int32_t>(), (int)ids.size(0), k.mutable_data_ptr(), v.mutable_data_ptr(), stream(dev));
      if (rc < 0) return status_error(rc, "lbc_kv8_read");
    }
    PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v)), *both = PyTuple_New(2);
    PyTuple_SET_ITEM(both, 0, pk);
    PyTuple_SET_ITEM(both, 1, pv);
    return both;
  });
}

PyMethodDef methods[] = {{"init", (PyCFunction)(void (*)())init, METH_FASTCALL, nullptr},
                         {"append", (PyCFunction)(void (*)())append, METH_FASTCALL, nullptr},
                         {"attention", (PyCFunction)(void (*)())attention, METH_FASTCALL, nullptr},
                         {"read", (PyCFunction)(void (*)())read, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "_kv8_torch", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv8_torch() { return PyModule_Create(&module_def); }
