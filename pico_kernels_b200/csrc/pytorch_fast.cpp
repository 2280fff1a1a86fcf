// Torch-aware fast-call entry points (module pico_kernels_b200._pktorch).
//
// gemm_int4.int4_gemm and int4_gemm_host (and the W8A8 calls of gemm_w8a8 and
// norm) check a dozen tensor attributes before their C-ABI call; on a slow host
// CPU each attribute read from Python costs 0.1-0.3 us, together more than the
// decode GEMM's kernel. These
// functions make the same checks on the tensors in C++ and call
// libpico_b200.so directly (linked by its soname, so the library instance is
// the one ctypes loaded). Each returns the output tensor, or the C ABI's
// status when the call failed, or -1 when the call is not one it serves
// (inputs that need a copy or a cast, a workspace not yet allocated, a host
// output not given, anything unexpected): the caller then takes the Python
// path, which raises the documented errors or allocates. Calls run with the
// GIL held (the shape cache below relies on it). The
// workspaces are the ones pico_kernels_b200._lib keeps (its dict is bound
// once with bind()), so reset_workspaces() covers both paths.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <initializer_list>
#include <utility>

#include "pico_b200.h"

namespace {

constexpr long kNotServed = -1;

PyObject* g_workspaces = nullptr;  // _lib._workspaces: {(device, stream, tag): uint8 tensor}
PyObject* g_tag_splitk = nullptr;
PyObject* g_tag_a = nullptr;
PyObject* g_tag_y = nullptr;

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return PK_F16;
    case at::kBFloat16: return PK_BF16;
    case at::kFloat: return PK_F32;
    default: return -1;
  }
}

// Pointer of the cached workspace (device, stream, tag) when it holds at
// least `nbytes`; nullptr otherwise (the Python path allocates it).
void* workspace(int device, uint64_t stream, PyObject* tag, size_t nbytes) {
  if (g_workspaces == nullptr) return nullptr;
  PyObject* key = Py_BuildValue("(iKO)", device, static_cast<unsigned long long>(stream), tag);
  if (key == nullptr) {
    PyErr_Clear();
    return nullptr;
  }
  PyObject* buf = PyDict_GetItemWithError(g_workspaces, key);  // borrowed
  Py_DECREF(key);
  if (buf == nullptr) {
    PyErr_Clear();
    return nullptr;
  }
  if (!THPVariable_Check(buf)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(buf);
  if (static_cast<size_t>(t.numel()) < nbytes || t.scalar_type() != at::kByte) return nullptr;
  return t.data_ptr();
}

// pk_w4a16_workspace_size per (M, N, K, split_k): a pure function of the shape.
size_t workspace_bytes(int64_t M, int64_t N, int64_t K, int split_k) {
  struct Entry {
    int64_t M, N, K;
    int split;
    size_t bytes;
  };
  static Entry cache[16];
  static int used = 0, next = 0;
  for (int i = 0; i < used; ++i)
    if (cache[i].M == M && cache[i].N == N && cache[i].K == K && cache[i].split == split_k)
      return cache[i].bytes;
  const size_t b = pk_w4a16_workspace_size(M, N, K, split_k);
  cache[next] = Entry{M, N, K, split_k, b};
  next = (next + 1) % 16;
  if (used < 16) ++used;
  return b;
}

// The weights and scales of a W4A16 call: w_packed [K, N/2] uint8 on `device`
// (contiguous), scale a [G, N] tensor of a's dtype (contiguous, same device)
// or a Python number. False when the Python path must handle them.
struct Weights {
  const void* wp;
  const void* scales;
  float scalar;
  int group;
  int64_t N;
};
bool weights(PyObject* w_obj, PyObject* scale_obj, PyObject* group_obj, int64_t K,
             at::ScalarType a_type, int device, Weights* w) {
  if (!THPVariable_Check(w_obj)) return false;
  const at::Tensor& wp = THPVariable_Unpack(w_obj);
  if (!wp.is_cuda() || wp.get_device() != device || wp.scalar_type() != at::kByte ||
      wp.dim() != 2 || wp.size(0) != K || !wp.is_contiguous())
    return false;
  w->wp = wp.data_ptr();
  w->N = 2 * wp.size(1);
  if (THPVariable_Check(scale_obj)) {
    const at::Tensor& s = THPVariable_Unpack(scale_obj);
    if (s.numel() <= 1) return false;  // a one-element tensor: the Python path reads it
    if (!s.is_cuda() || s.get_device() != device || s.dim() != 2 || s.size(1) != w->N ||
        s.scalar_type() != a_type || !s.is_contiguous())
      return false;
    const int64_t G = s.size(0);
    int64_t group = 0;
    if (group_obj == Py_None) {  // prefer 128 when several sizes give G groups
      for (int64_t g : {static_cast<int64_t>(128), K / G})
        if (g > 0 && (K + g - 1) / g == G) {
          group = g;
          break;
        }
    } else {
      group = PyLong_AsLongLong(group_obj);
      if (group == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
      }
    }
    if (group <= 0 || (K + group - 1) / group != G || group > (1ll << 30)) return false;
    w->scales = s.data_ptr();
    w->scalar = 1.0f;
    w->group = static_cast<int>(group);
    return true;
  }
  if (!PyFloat_Check(scale_obj) && !PyLong_Check(scale_obj)) return false;
  const double v = PyFloat_AsDouble(scale_obj);
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  w->scales = nullptr;
  w->scalar = static_cast<float>(v);
  w->group = 0;
  return true;
}

// out_dtype (a torch.dtype) and out: a contiguous [M, N] tensor of that
// dtype (fp32 or bf16), on CUDA `device` (device >= 0) or on the host (-1).
bool output(PyObject* out_obj, PyObject* dtype_obj, int64_t M, int64_t N, int device, void** ptr,
            int* code, int64_t* elt) {
  if (!THPVariable_Check(out_obj) || !THPDtype_Check(dtype_obj)) return false;
  const at::ScalarType want = reinterpret_cast<THPDtype*>(dtype_obj)->scalar_type;
  const at::Tensor& out = THPVariable_Unpack(out_obj);
  if (out.scalar_type() != want || (want != at::kFloat && want != at::kBFloat16)) return false;
  if (device >= 0 ? (!out.is_cuda() || out.get_device() != device) : out.is_cuda()) return false;
  if (out.dim() != 2 || out.size(0) != M || out.size(1) != N || !out.is_contiguous())
    return false;
  *ptr = out.data_ptr();
  *code = code_of(want);
  *elt = out.element_size();
  return true;
}

// int4_gemm(a, w_packed, scale, group_size, out, out_dtype, split_k)
//   -> out (allocated here when None), or the status, or -1
PyObject* int4_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) {
    PyErr_Format(PyExc_TypeError, "int4_gemm takes 7 arguments (%zd given)", n);
    return nullptr;
  }
  try {
    if (!THPVariable_Check(args[0])) return PyLong_FromLong(kNotServed);
    const at::Tensor& a = THPVariable_Unpack(args[0]);
    const int a_code = code_of(a.scalar_type());
    if (!a.is_cuda() || (a_code != PK_F16 && a_code != PK_BF16) || a.dim() != 2)
      return PyLong_FromLong(kNotServed);
    const int64_t M = a.size(0), K = a.size(1);
    if (a.stride(1) != 1 || a.stride(0) < K) return PyLong_FromLong(kNotServed);
    const int device = a.get_device();
    Weights w;
    if (!weights(args[1], args[2], args[3], K, a.scalar_type(), device, &w))
      return PyLong_FromLong(kNotServed);
    void* out = nullptr;
    int out_code = 0;
    int64_t elt = 0;
    const bool alloc = args[4] == Py_None;
    if (alloc) {
      if (!THPDtype_Check(args[5])) return PyLong_FromLong(kNotServed);
      const at::ScalarType want = reinterpret_cast<THPDtype*>(args[5])->scalar_type;
      if (want != at::kFloat && want != at::kBFloat16) return PyLong_FromLong(kNotServed);
      out_code = code_of(want);
    } else if (!output(args[4], args[5], M, w.N, device, &out, &out_code, &elt)) {
      return PyLong_FromLong(kNotServed);
    }
    const long split = PyLong_AsLong(args[6]);
    if (split == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return PyLong_FromLong(kNotServed);
    }
    const uint64_t stream =
        reinterpret_cast<uint64_t>(c10::cuda::getCurrentCUDAStream(device).stream());
    const size_t ws_bytes = workspace_bytes(M, w.N, K, static_cast<int>(split));
    void* ws = nullptr;
    if (ws_bytes > 0) {
      ws = workspace(device, stream, g_tag_splitk, ws_bytes);
      if (ws == nullptr) return PyLong_FromLong(kNotServed);
    }
    at::Tensor y;
    if (alloc) {
      y = at::empty({M, w.N}, at::TensorOptions()
                                  .dtype(out_code == PK_F32 ? at::kFloat : at::kBFloat16)
                                  .device(at::Device(at::kCUDA, static_cast<int8_t>(device))));
      out = y.data_ptr();
    }
    const int st = pk_w4a16_gemm(a.data_ptr(), a_code, a.stride(0),
                                 static_cast<const uint8_t*>(w.wp), w.scales, w.scalar, w.group,
                                 M, w.N, K, out, out_code, w.N, static_cast<int>(split), ws,
                                 ws_bytes, reinterpret_cast<void*>(stream));
    if (st != PK_OK) return PyLong_FromLong(st);
    if (alloc) return THPVariable_Wrap(std::move(y));
    Py_INCREF(args[4]);
    return args[4];
  } catch (...) {
    PyErr_Clear();
    return PyLong_FromLong(kNotServed);
  }
}

// int4_gemm_host(a, w_packed, scale, group_size, out, out_dtype) -> out, or the status, or -1
// (a and out: host tensors; the staging buffers "stage_a" / "stage_y" and the
// workspace are the cached ones of the weights' device and current stream)
PyObject* int4_gemm_host(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6) {
    PyErr_Format(PyExc_TypeError, "int4_gemm_host takes 6 arguments (%zd given)", n);
    return nullptr;
  }
  try {
    if (!THPVariable_Check(args[0]) || !THPVariable_Check(args[1]))
      return PyLong_FromLong(kNotServed);
    const at::Tensor& a = THPVariable_Unpack(args[0]);
    const int a_code = code_of(a.scalar_type());
    if (a.is_cuda() || (a_code != PK_F16 && a_code != PK_BF16) || a.dim() != 2)
      return PyLong_FromLong(kNotServed);
    const int64_t M = a.size(0), K = a.size(1);
    if (a.stride(1) != 1 || a.stride(0) < K) return PyLong_FromLong(kNotServed);
    const at::Tensor& wp = THPVariable_Unpack(args[1]);
    if (!wp.is_cuda()) return PyLong_FromLong(kNotServed);
    const int device = wp.get_device();
    Weights w;
    if (!weights(args[1], args[2], args[3], K, a.scalar_type(), device, &w))
      return PyLong_FromLong(kNotServed);
    void* out;
    int out_code;
    int64_t elt;
    if (!output(args[4], args[5], M, w.N, -1, &out, &out_code, &elt))
      return PyLong_FromLong(kNotServed);
    const uint64_t stream =
        reinterpret_cast<uint64_t>(c10::cuda::getCurrentCUDAStream(device).stream());
    const size_t ws_bytes = workspace_bytes(M, w.N, K, 0);
    void* ws = nullptr;
    if (ws_bytes > 0) {
      ws = workspace(device, stream, g_tag_splitk, ws_bytes);
      if (ws == nullptr) return PyLong_FromLong(kNotServed);
    }
    void* a_dev = workspace(device, stream, g_tag_a, static_cast<size_t>(M * K * 2));
    void* y_dev = workspace(device, stream, g_tag_y, static_cast<size_t>(M * w.N * elt));
    if (a_dev == nullptr || y_dev == nullptr) return PyLong_FromLong(kNotServed);
    const int st = pk_w4a16_gemm_host(a.data_ptr(), a_code, a.stride(0),
                                      static_cast<const uint8_t*>(w.wp), w.scales, w.scalar,
                                      w.group, M, w.N, K, out, out_code, a_dev, y_dev, ws,
                                      ws_bytes, reinterpret_cast<void*>(stream));
    if (st != PK_OK) return PyLong_FromLong(st);
    Py_INCREF(args[4]);
    return args[4];
  } catch (...) {
    PyErr_Clear();
    return PyLong_FromLong(kNotServed);
  }
}

// ---------------------------------------------------------------------------
// W8A8 (gemm_w8a8, norm). Served: CUDA tensors on the current device whose
// strides the kernels read as they are. Outputs are allocated here.
// ---------------------------------------------------------------------------
int code8_of(at::ScalarType t) {
  return t == at::kChar ? PK_I8 : t == at::kFloat8_e4m3fn ? PK_E4M3 : -1;
}

bool dtype_arg(PyObject* o, at::ScalarType* t) {
  if (!THPDtype_Check(o)) return false;
  *t = reinterpret_cast<THPDtype*>(o)->scalar_type;
  return true;
}

// A tensor on the current device, or nullptr.
const at::Tensor* device_tensor(PyObject* o) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.is_cuda() && t.get_device() == c10::cuda::current_device() ? &t : nullptr;
}

at::TensorOptions on_device(const at::Tensor& like, at::ScalarType t) {
  return at::TensorOptions().dtype(t).device(like.device());
}

void* stream_of(const at::Tensor& t) {
  return reinterpret_cast<void*>(c10::cuda::getCurrentCUDAStream(t.get_device()).stream());
}

int64_t pitch16(int64_t K) { return (K + 15) / 16 * 16; }

// Contiguous rows of fp16 / bf16 / fp32 values, at least one row and column.
bool value_rows(const at::Tensor& x, int64_t* rows, int64_t* K) {
  if (code_of(x.scalar_type()) < 0 || x.dim() < 1 || !x.is_contiguous() || x.numel() == 0)
    return false;
  *K = x.size(-1);
  *rows = x.numel() / *K;
  return true;
}

// Storage of x's shape in 8-bit codes (rows 16 bytes' multiples apart) and one
// scale per row.
void empty_codes(const at::Tensor& x, int64_t K, at::ScalarType t, at::Tensor* q,
                 at::Tensor* scale) {
  const int64_t pitch = pitch16(K);
  if (pitch == K) {
    *q = at::empty(x.sizes(), on_device(x, t));
  } else {
    auto sizes = x.sizes().vec();
    sizes.back() = pitch;
    *q = at::empty(sizes, on_device(x, t)).narrow(-1, 0, K);
  }
  *scale = at::empty(x.sizes().slice(0, x.dim() - 1), on_device(x, at::kFloat));
}

PyObject* tuple_of(at::Tensor&& q, at::Tensor&& scale, PyObject* h) {
  PyObject* a = THPVariable_Wrap(std::move(q));
  PyObject* b = THPVariable_Wrap(std::move(scale));
  PyObject* t = nullptr;
  if (a != nullptr && b != nullptr)
    t = h == nullptr ? PyTuple_Pack(2, a, b) : PyTuple_Pack(3, a, b, h);
  Py_XDECREF(a);
  Py_XDECREF(b);
  Py_XDECREF(h);
  return t;
}

// quantize_rows(x, dtype) -> (codes, scale), or the status, or -1
PyObject* quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 2) {
    PyErr_Format(PyExc_TypeError, "quantize_rows takes 2 arguments (%zd given)", n);
    return nullptr;
  }
  try {
    const at::Tensor* x = device_tensor(args[0]);
    at::ScalarType t;
    int64_t rows, K;
    if (x == nullptr || !dtype_arg(args[1], &t) || code8_of(t) < 0 || !value_rows(*x, &rows, &K))
      return PyLong_FromLong(kNotServed);
    at::Tensor q, scale;
    empty_codes(*x, K, t, &q, &scale);
    const int st = pk_quantize_rows(x->data_ptr(), code_of(x->scalar_type()), rows, K, K,
                                    q.data_ptr(), code8_of(t), pitch16(K),
                                    scale.data_ptr<float>(), stream_of(*x));
    if (st != PK_OK) return PyLong_FromLong(st);
    return tuple_of(std::move(q), std::move(scale), nullptr);
  } catch (...) {
    PyErr_Clear();
    return PyLong_FromLong(kNotServed);
  }
}

// One fp32 value per row, contiguous: `shape`, or `shape` with a trailing 1.
const float* row_values(PyObject* o, int64_t rows) {
  const at::Tensor* s = device_tensor(o);
  if (s == nullptr || s->scalar_type() != at::kFloat || !s->is_contiguous() ||
      s->numel() != rows || s->dim() < 1 || s->dim() > 2 || s->size(0) != rows)
    return nullptr;
  return s->data_ptr<float>();
}

// A 2-D 8-bit operand with rows the kernels can load, at least one of them.
struct Codes {
  const at::Tensor* t;
  int64_t rows, K, pitch;
  int code;
};
bool codes(PyObject* o, Codes* c) {
  c->t = device_tensor(o);
  if (c->t == nullptr) return false;
  const at::Tensor& t = *c->t;
  c->code = code8_of(t.scalar_type());
  if (c->code < 0 || t.dim() != 2) return false;
  c->rows = t.size(0);
  c->K = t.size(1);
  if (c->rows < 1 || c->K < 1) return false;
  c->pitch = c->rows > 1 ? t.stride(0) : pitch16(c->K);
  return (c->K == 1 || t.stride(1) == 1) && c->pitch % 16 == 0 && c->pitch >= c->K &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

// Tells autograd that a caller's tensor has new contents (a backward pass that saved
// the old ones then fails; inference tensors are not counted).
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// Whether two ranges of addresses meet.
struct Range {
  uintptr_t at;
  int64_t bytes;
};
bool meet(Range a, Range b) { return a.at < b.at + b.bytes && b.at < a.at + a.bytes; }
Range range_of(const at::Tensor& t) {  // contiguous
  return {reinterpret_cast<uintptr_t>(t.data_ptr()), static_cast<int64_t>(t.nbytes())};
}
Range range_of(const Codes& c) {
  return {reinterpret_cast<uintptr_t>(c.t->data_ptr()), (c.rows - 1) * c.pitch + c.K};
}
Range range_of(const float* p, int64_t n) {
  return {reinterpret_cast<uintptr_t>(p), p != nullptr ? 4 * n : 0};
}

// dequantize_rows(codes, scale, dtype) -> values, or the status, or -1
PyObject* dequantize_rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) {
    PyErr_Format(PyExc_TypeError, "dequantize_rows takes 3 arguments (%zd given)", n);
    return nullptr;
  }
  try {
    Codes c;
    at::ScalarType t;
    if (!codes(args[0], &c) || !dtype_arg(args[2], &t) || code_of(t) < 0)
      return PyLong_FromLong(kNotServed);
    const float* scale = row_values(args[1], c.rows);
    if (scale == nullptr) return PyLong_FromLong(kNotServed);
    at::Tensor out = at::empty({c.rows, c.K}, on_device(*c.t, t));
    const int st = pk_dequantize_rows(c.t->data_ptr(), c.code, c.rows, c.K, c.pitch, scale,
                                      out.data_ptr(), code_of(t), c.K, stream_of(*c.t));
    if (st != PK_OK) return PyLong_FromLong(st);
    return THPVariable_Wrap(std::move(out));
  } catch (...) {
    PyErr_Clear();
    return PyLong_FromLong(kNotServed);
  }
}

// rms_norm_quant(x, weight, eps, residual, dtype, residual_out)
//   -> (codes, scale[, h]), or the status, or -1
PyObject* rms_norm_quant(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 6) {
    PyErr_Format(PyExc_TypeError, "rms_norm_quant takes 6 arguments (%zd given)", n);
    return nullptr;
  }
  try {
    const at::Tensor* x = device_tensor(args[0]);
    const at::Tensor* w = device_tensor(args[1]);
    at::ScalarType t;
    int64_t rows, K;
    if (x == nullptr || w == nullptr || !PyFloat_Check(args[2]) || !dtype_arg(args[4], &t) ||
        code8_of(t) < 0 || !value_rows(*x, &rows, &K))
      return PyLong_FromLong(kNotServed);
    if (w->dim() != 1 || w->size(0) != K || !w->is_contiguous() ||
        (w->scalar_type() != x->scalar_type() && w->scalar_type() != at::kFloat))
      return PyLong_FromLong(kNotServed);
    const at::Tensor* r = nullptr;
    if (args[3] != Py_None) {
      r = device_tensor(args[3]);
      if (r == nullptr || r->scalar_type() != x->scalar_type() || r->sizes() != x->sizes() ||
          !r->is_contiguous())
        return PyLong_FromLong(kNotServed);
    }
    at::Tensor h;
    if (args[5] != Py_None) {
      const at::Tensor* o = device_tensor(args[5]);
      if (r == nullptr || o == nullptr || o->scalar_type() != x->scalar_type() ||
          o->sizes() != x->sizes() || !o->is_contiguous())
        return PyLong_FromLong(kNotServed);
      // x, residual or memory of its own: another overlap is refused in Python
      for (const at::Tensor* in : {x, r, w})
        if (meet(range_of(*o), range_of(*in)) && (in == w || o->data_ptr() != in->data_ptr()))
          return PyLong_FromLong(kNotServed);
      h = *o;
    } else if (r != nullptr) {
      h = at::empty(x->sizes(), on_device(*x, x->scalar_type()));
    }
    at::Tensor q, scale;
    empty_codes(*x, K, t, &q, &scale);
    const int st = pk_rms_norm_quant(
        x->data_ptr(), code_of(x->scalar_type()), rows, K, K, r ? r->data_ptr() : nullptr, K,
        w->data_ptr(), code_of(w->scalar_type()), static_cast<float>(PyFloat_AS_DOUBLE(args[2])),
        r ? h.data_ptr() : nullptr, K, q.data_ptr(), code8_of(t), pitch16(K),
        scale.data_ptr<float>(), stream_of(*x));
    if (st != PK_OK) return PyLong_FromLong(st);
    PyObject* ho = nullptr;
    if (args[5] != Py_None) {
      written(h);
      Py_INCREF(args[5]);
      ho = args[5];
    } else if (r != nullptr) {
      ho = THPVariable_Wrap(std::move(h));
      if (ho == nullptr) return nullptr;
    }
    return tuple_of(std::move(q), std::move(scale), ho);
  } catch (...) {
    PyErr_Clear();
    return PyLong_FromLong(kNotServed);
  }
}

// The output of a product: allocated, or `out_obj` (contiguous [M, N]), which meets
// none of the operands.
bool product_out(PyObject* dtype_obj, PyObject* out_obj, int64_t M, int64_t N,
                 const at::Tensor& like, std::initializer_list<Range> operands, at::Tensor* y) {
  at::ScalarType t;
  if (!dtype_arg(dtype_obj, &t) || code_of(t) < 0) return false;
  if (out_obj == Py_None) {
    *y = at::empty({M, N}, on_device(like, t));
    return true;
  }
  const at::Tensor* o = device_tensor(out_obj);
  if (o == nullptr || o->scalar_type() != t || o->dim() != 2 || o->size(0) != M ||
      o->size(1) != N || !o->is_contiguous())
    return false;
  for (const Range& r : operands)
    if (meet(range_of(*o), r)) return false;
  *y = *o;
  return true;
}

PyObject* product_result(int st, PyObject* out_obj, at::Tensor&& y) {
  if (st != PK_OK) return PyLong_FromLong(st);
  if (out_obj == Py_None) return THPVariable_Wrap(std::move(y));
  written(y);
  Py_INCREF(out_obj);
  return out_obj;
}

// w8a8_gemm(a8, a_scale, w8, w_scale, bias, out_dtype, out) -> y, or the status, or -1
PyObject* w8a8_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) {
    PyErr_Format(PyExc_TypeError, "w8a8_gemm takes 7 arguments (%zd given)", n);
    return nullptr;
  }
  try {
    Codes a, w;
    if (!codes(args[0], &a) || !codes(args[2], &w) || a.code != w.code || a.K != w.K)
      return PyLong_FromLong(kNotServed);
    const float* sa = row_values(args[1], a.rows);
    const float* sw = row_values(args[3], w.rows);
    const float* bias = args[4] == Py_None ? nullptr : row_values(args[4], w.rows);
    at::Tensor y;
    if (sa == nullptr || sw == nullptr || (args[4] != Py_None && bias == nullptr) ||
        !product_out(args[5], args[6], a.rows, w.rows, *a.t,
                     {range_of(a), range_of(sa, a.rows), range_of(w), range_of(sw, w.rows),
                      range_of(bias, w.rows)},
                     &y))
      return PyLong_FromLong(kNotServed);
    const int st = pk_w8a8_gemm(a.t->data_ptr(), a.code, a.pitch, sa, w.t->data_ptr(), w.pitch, sw,
                                bias, a.rows, w.rows, a.K, y.data_ptr(), code_of(y.scalar_type()),
                                w.rows, stream_of(*a.t));
    return product_result(st, args[6], std::move(y));
  } catch (...) {
    PyErr_Clear();
    return PyLong_FromLong(kNotServed);
  }
}

// w8a8_gated_gemm(a8, a_scale, w_gate, gate_scale, w_up, up_scale, activation,
//                 out_dtype, out) -> y, or the status, or -1
PyObject* w8a8_gated_gemm(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 9) {
    PyErr_Format(PyExc_TypeError, "w8a8_gated_gemm takes 9 arguments (%zd given)", n);
    return nullptr;
  }
  try {
    Codes a, g, u;
    if (!codes(args[0], &a) || !codes(args[2], &g) || !codes(args[4], &u) || a.code != g.code ||
        a.code != u.code || a.K != g.K || a.K != u.K || g.rows != u.rows)
      return PyLong_FromLong(kNotServed);
    const float* sa = row_values(args[1], a.rows);
    const float* sg = row_values(args[3], g.rows);
    const float* su = row_values(args[5], u.rows);
    const long act = PyLong_Check(args[6]) ? PyLong_AsLong(args[6]) : -1;
    at::Tensor y;
    if (sa == nullptr || sg == nullptr || su == nullptr ||
        (act != PK_ACT_SILU && act != PK_ACT_GELU_TANH) ||
        !product_out(args[7], args[8], a.rows, g.rows, *a.t,
                     {range_of(a), range_of(sa, a.rows), range_of(g), range_of(sg, g.rows),
                      range_of(u), range_of(su, g.rows)},
                     &y))
      return PyLong_FromLong(kNotServed);
    const int st = pk_w8a8_gated_gemm(a.t->data_ptr(), a.code, a.pitch, sa, g.t->data_ptr(),
                                      g.pitch, sg, u.t->data_ptr(), u.pitch, su,
                                      static_cast<int>(act), a.rows, g.rows, a.K, y.data_ptr(),
                                      code_of(y.scalar_type()), g.rows, stream_of(*a.t));
    return product_result(st, args[8], std::move(y));
  } catch (...) {
    PyErr_Clear();
    return PyLong_FromLong(kNotServed);
  }
}

// bind(workspaces): the dict of cached workspaces the Python path fills.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 1 || !PyDict_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "bind takes the workspace dict");
    return nullptr;
  }
  Py_INCREF(args[0]);
  Py_XDECREF(g_workspaces);
  g_workspaces = args[0];
  Py_RETURN_NONE;
}

PyMethodDef kMethods[] = {
    {"int4_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(int4_gemm)),
     METH_FASTCALL,
     "int4_gemm(a, w_packed, scale, group_size, out, out_dtype, split_k): the output tensor, "
     "the C ABI's status on failure, or -1 when the Python path must take the call."},
    {"int4_gemm_host",
     reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(int4_gemm_host)), METH_FASTCALL,
     "int4_gemm_host(a, w_packed, scale, group_size, out, out_dtype): out, the C ABI's status "
     "on failure, or -1 when the Python path must take the call."},
    {"quantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(quantize_rows)),
     METH_FASTCALL,
     "quantize_rows(x, dtype): (codes, scale), the C ABI's "
     "status on failure, or -1 when the Python path must take the call."},
    {"dequantize_rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(dequantize_rows)),
     METH_FASTCALL,
     "dequantize_rows(codes, scale, dtype): the values, the C ABI's "
     "status on failure, or -1 when the Python path must take the call."},
    {"rms_norm_quant", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rms_norm_quant)),
     METH_FASTCALL,
     "rms_norm_quant(x, weight, eps, residual, dtype, residual_out): (codes, scale[, h]), the C ABI's "
     "status on failure, or -1 when the Python path must take the call."},
    {"w8a8_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(w8a8_gemm)),
     METH_FASTCALL,
     "w8a8_gemm(a8, a_scale, w8, w_scale, bias, out_dtype, out): the output, the C ABI's "
     "status on failure, or -1 when the Python path must take the call."},
    {"w8a8_gated_gemm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(w8a8_gated_gemm)),
     METH_FASTCALL,
     "w8a8_gated_gemm(a8, a_scale, w_gate, gate_scale, w_up, up_scale, activation, out_dtype, out): the output, the C ABI's "
     "status on failure, or -1 when the Python path must take the call."},
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL,
     "bind(workspaces): the workspace dict of pico_kernels_b200._lib."},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_pktorch",
                       "Torch-aware fast-call entry points of libpico_b200.so.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__pktorch() {
  g_tag_splitk = PyUnicode_InternFromString("splitk");
  g_tag_a = PyUnicode_InternFromString("stage_a");
  g_tag_y = PyUnicode_InternFromString("stage_y");
  if (!g_tag_splitk || !g_tag_a || !g_tag_y) return nullptr;
  return PyModule_Create(&kModule);
}
