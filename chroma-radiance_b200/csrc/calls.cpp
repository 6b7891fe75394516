// calls.cpp — b2g_calls, the Python side of the packed operators: checks of arguments, outputs and
// workspaces from torch's allocator, the descriptor, the call of libb2g.so.
//
// The work of a small call takes the GPU 2 to 7 us, so that the host's share counts: us per call, launches
// included, here and as the same steps in Python around ctypes: gemm_s8 of one token 4.5, 9.0; qk_norm_rope 5.8, 12.0;
// attention_packed of 64 short sequences 10.8, 16.4 (the GPU's time).  Nothing is kept between calls.  The entry
// points' addresses come from b2g.py (bind), so this module links nothing of the engine.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <string>
#include "b2g.h"

namespace {

using at::ScalarType;
using at::Tensor;

decltype(&b2g_gemm_s8) call_gemm_s8 = nullptr;
decltype(&b2g_gemm_s8_workspace) call_gemm_s8_workspace = nullptr;
decltype(&b2g_qk_norm_rope) call_qk_norm_rope = nullptr;
decltype(&b2g_attention_packed) call_attention_packed = nullptr;
decltype(&b2g_attention_packed_workspace) call_attention_packed_workspace = nullptr;
decltype(&b2g_last_error) call_last_error = nullptr;
PyObject* error_type = nullptr;

struct Refused {
  std::string why;
};
struct PythonError {};  // the interpreter's error is set
[[noreturn]] void refuse(std::string why) { throw Refused{std::move(why)}; }

void check(b2g_status s) {
  if (s != B2G_OK) refuse("b2g status " + std::to_string(static_cast<int>(s)) + ": " + call_last_error());
}

const Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) refuse(std::string(what) + ": a tensor expected");
  return THPVariable_Unpack(o);
}
const Tensor* maybe(PyObject* o, const char* what) { return o == Py_None ? nullptr : &tensor(o, what); }

int dtype_of(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return B2G_F32;
    case ScalarType::Half: return B2G_F16;
    case ScalarType::BFloat16: return B2G_BF16;
    default: return -1;
  }
}
ScalarType scalar_type(PyObject* o, const char* what) {
  if (!THPDtype_Check(o)) refuse(std::string(what) + ": out_dtype must be a torch.dtype");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

const char* name_of(ScalarType t) {
  switch (t) {
    case ScalarType::Float: return "F32";
    case ScalarType::Half: return "F16";
    case ScalarType::BFloat16: return "BF16";
    default: return "int32";
  }
}

// The address of a contiguous vector of n values.
const void* vector(const Tensor& t, ScalarType type, int64_t n, const char* what) {
  if (t.scalar_type() != type || t.numel() != n || !t.is_contiguous())
    refuse(std::string(what) + " must be contiguous " + name_of(type) + " [" + std::to_string(n) + "]");
  return t.data_ptr();
}

// The raw stream of a call on these tensors (NULL: absent), all of the current device.
void* stream_of(std::initializer_list<const Tensor*> ts) {
  int dev = -1;
  for (const Tensor* t : ts) {
    if (!t) continue;
    if (t->is_cuda() && dev < 0) dev = c10::cuda::current_device();
    if (!t->is_cuda() || t->get_device() != dev) refuse("all tensors must be CUDA tensors of the current device");
  }
  return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(dev)).stream();
}

// Memory of torch's allocator, for use on the current stream.
Tensor make(at::IntArrayRef shape, ScalarType type, const Tensor& like) {
  return at::empty(shape, at::TensorOptions().dtype(type).device(like.device()));
}

// Token and head stride of a [tokens, heads, d] tensor whose heads are contiguous.
struct Heads {
  int64_t ld, hs;
};
Heads heads(const Tensor& t, const char* what) {
  if (t.dim() != 3 || (t.stride(2) != 1 && t.size(2) > 1))
    refuse(std::string(what) + ": [tokens, heads, d] with unit stride along d expected");
  return {t.stride(0), t.stride(1)};
}

// An output of t's shape: the given one, checked, or a new one.
Tensor output_like(const Tensor& t, const Tensor* out, ScalarType type, const char* what) {
  if (!out) return make(t.sizes(), type, t);
  if (out->sizes() != t.sizes() || out->scalar_type() != type)
    refuse(std::string(what) + " must be " + name_of(type) + " of the input's shape");
  return *out;
}

// The given object, or a new one for a new tensor.
PyObject* result(PyObject* given, const Tensor& t) {
  if (given == Py_None) return THPVariable_Wrap(t);
  Py_INCREF(given);
  return given;
}

template <typename F>
PyObject* guarded(F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused& e) {
    PyErr_SetString(error_type, e.why.c_str());
  } catch (const PythonError&) {
  }
  return nullptr;
  END_HANDLE_TH_ERRORS
}

void expect(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) refuse("b2g_calls: wrong number of arguments");
}

// (x, wq, w_scale, bias, out, out_dtype, epilogue, gate, x_scale) -> out
PyObject* gemm_s8(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 9);
    const Tensor &x = tensor(a[0], "gemm_s8: x"), &w = tensor(a[1], "gemm_s8: wq"), &ws = tensor(a[2], "gemm_s8: w_scale");
    const Tensor *bias = maybe(a[3], "gemm_s8: bias"), *gate = maybe(a[7], "gemm_s8: gate"),
                 *xs = maybe(a[8], "gemm_s8: x_scale"), *given = maybe(a[4], "gemm_s8: out");
    if (x.dim() != 2 || w.dim() != 2 || w.scalar_type() != ScalarType::Char) refuse("gemm_s8: 2-D x and int8 wq expected");
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    if (w.size(1) != K)
      refuse("gemm_s8: K mismatch (" + std::to_string(M) + ", " + std::to_string(K) + ") vs (" + std::to_string(N) + ", " +
             std::to_string(w.size(1)) + ")");
    if (K > 1 && (x.stride(1) != 1 || w.stride(1) != 1)) refuse("gemm_s8: x and wq need unit stride along K");
    const bool codes = x.scalar_type() == ScalarType::Char;
    const int a_dtype = codes ? B2G_S8 : dtype_of(x.scalar_type());
    if (a_dtype < 0) refuse("gemm_s8: x must be int8, F32, BF16 or F16");
    int epi = -1;
    static const struct { const char* name; int value; } kEpilogues[] = {
        {"none", B2G_EPI_NONE}, {"gelu", B2G_EPI_GELU}, {"gated_residual", B2G_EPI_GATED_RESIDUAL}, {"silu", B2G_EPI_SILU}};
    if (PyUnicode_Check(a[6]))
      for (const auto& e : kEpilogues)
        if (PyUnicode_CompareWithASCIIString(a[6], e.name) == 0) epi = e.value;
    if (epi < 0) refuse("gemm_s8: unknown epilogue");
    if (!given && epi == B2G_EPI_GATED_RESIDUAL) refuse("gemm_s8: gated_residual needs `out` (the residual)");
    if (given && (given->dim() != 2 || given->size(0) != M || given->size(1) != N || (N > 1 && given->stride(1) != 1)))
      refuse("gemm_s8: out must be [M, N] with unit column stride");
    const ScalarType o_type = given ? given->scalar_type() : a[5] == Py_None ? ScalarType::Float : scalar_type(a[5], "gemm_s8");
    if (dtype_of(o_type) < 0) refuse("gemm_s8: out must be F32, BF16 or F16");
    const int64_t pad = (K + 15) / 16 * 16;
    b2g_gemm_desc d{};
    d.M = M; d.N = N; d.K = K;
    d.a = x.data_ptr();
    d.a_dtype = static_cast<b2g_dtype>(a_dtype);
    d.lda = M > 1 ? x.stride(0) : codes ? pad : K;
    d.b = w.data_ptr();
    d.b_dtype = B2G_S8;
    d.ldb = N > 1 ? w.stride(0) : pad;
    const float* w_ptr = static_cast<const float*>(vector(ws, ScalarType::Float, N, "gemm_s8: w_scale"));
    if (bias) {
      if (bias->scalar_type() != ScalarType::Float && bias->scalar_type() != ScalarType::BFloat16)
        refuse("gemm_s8: bias must be F32 or BF16");
      d.bias = vector(*bias, bias->scalar_type(), N, "gemm_s8: bias");
      d.bias_dtype = static_cast<b2g_dtype>(dtype_of(bias->scalar_type()));
    }
    d.epilogue = static_cast<b2g_epilogue>(epi);
    if (epi != B2G_EPI_GATED_RESIDUAL) gate = nullptr;
    if (gate) d.gate = static_cast<const float*>(vector(*gate, ScalarType::Float, N, "gemm_s8: gate"));
    if (!codes) xs = nullptr;
    const float* x_ptr = xs ? static_cast<const float*>(vector(*xs, ScalarType::Float, M, "gemm_s8: x_scale")) : nullptr;
    void* stream = stream_of({&x, &w, &ws, given, bias, gate, xs});
    const Tensor out = given ? *given : make({M, N}, o_type, x);
    d.d = out.data_ptr();
    d.d_dtype = static_cast<b2g_dtype>(dtype_of(o_type));
    d.ldd = M > 1 ? out.stride(0) : N;
    Tensor space;
    const bool needs_none = M == 1 && K <= 16384;  // (one launch; the library would take its own if it did need one)
    const size_t n = needs_none ? 0 : call_gemm_s8_workspace(M, K, d.a_dtype);
    if (n) space = make({static_cast<int64_t>(n)}, ScalarType::Char, x);
    check(call_gemm_s8(&d, x_ptr, w_ptr, n ? space.data_ptr() : nullptr, n, stream));
    return result(a[4], out);
  });
}

// (q, k, positions, axes_dim, q_norm, k_norm, eps, theta, interleaved, q_out, k_out, out_dtype) -> (q', k')
PyObject* qk_norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 12);
    const Tensor &q = tensor(a[0], "qk_norm_rope: q"), &k = tensor(a[1], "qk_norm_rope: k"),
                 &pos = tensor(a[2], "qk_norm_rope: positions");
    const Tensor *qn = maybe(a[4], "qk_norm_rope: q_norm"), *kn = maybe(a[5], "qk_norm_rope: k_norm"),
                 *q_given = maybe(a[9], "qk_norm_rope: q_out"), *k_given = maybe(a[10], "qk_norm_rope: k_out");
    const Heads hq = heads(q, "qk_norm_rope: q"), hk = heads(k, "qk_norm_rope: k");
    const int64_t T = q.size(0), D = q.size(2);
    const int dt = dtype_of(q.scalar_type());
    if (k.size(0) != T || k.size(2) != D || k.scalar_type() != q.scalar_type() || dt < 0)
      refuse("qk_norm_rope: q and k must have the same tokens, head width and F32/BF16/F16 type");
    b2g_qk_norm_rope_desc d{};
    if (!PyList_Check(a[3]) && !PyTuple_Check(a[3])) refuse("qk_norm_rope: axes_dim must be a list");
    const Py_ssize_t n_axes = PySequence_Fast_GET_SIZE(a[3]);
    if (n_axes > 4) refuse("qk_norm_rope: at most 4 axes");
    for (Py_ssize_t i = 0; i < n_axes; ++i) {
      const long v = PyLong_AsLong(PySequence_Fast_GET_ITEM(a[3], i));
      if (v == -1 && PyErr_Occurred()) throw PythonError{};
      if (v < 0 || v > 1 << 20) refuse("qk_norm_rope: axes_dim out of range");
      d.axis_dim[i] = static_cast<int>(v);
    }
    if (pos.dim() != 2 || pos.size(0) != T || pos.size(1) != n_axes || pos.scalar_type() != ScalarType::Float ||
        (n_axes > 1 && pos.stride(1) != 1))
      refuse("qk_norm_rope: positions must be F32 [tokens, len(axes_dim)]");
    const ScalarType o_type = a[11] != Py_None ? scalar_type(a[11], "qk_norm_rope")
                              : q_given        ? q_given->scalar_type()
                              : k_given        ? k_given->scalar_type()
                                               : q.scalar_type();
    if (dtype_of(o_type) < 0) refuse("qk_norm_rope: outputs must be F32, BF16 or F16");
    if (qn) d.q_norm = static_cast<const float*>(vector(*qn, ScalarType::Float, D, "qk_norm_rope: q_norm"));
    if (kn) d.k_norm = static_cast<const float*>(vector(*kn, ScalarType::Float, D, "qk_norm_rope: k_norm"));
    void* stream = stream_of({&q, &k, &pos, qn, kn, q_given, k_given});
    const Tensor qo = output_like(q, q_given, o_type, "qk_norm_rope: q_out"), ko = output_like(k, k_given, o_type, "qk_norm_rope: k_out");
    const Heads hqo = heads(qo, "qk_norm_rope: q_out"), hko = heads(ko, "qk_norm_rope: k_out");
    d.q = q.data_ptr(); d.k = k.data_ptr();
    d.dtype = static_cast<b2g_dtype>(dt);
    d.q_out = qo.data_ptr(); d.k_out = ko.data_ptr();
    d.out_dtype = static_cast<b2g_dtype>(dtype_of(o_type));
    d.ldq = hq.ld; d.hsq = hq.hs; d.ldk = hk.ld; d.hsk = hk.hs;
    d.ldq_out = hqo.ld; d.hsq_out = hqo.hs; d.ldk_out = hko.ld; d.hsk_out = hko.hs;
    d.tokens = T;
    d.n_head = static_cast<int>(q.size(1)); d.n_kv_head = static_cast<int>(k.size(1)); d.d_head = static_cast<int>(D);
    d.eps = static_cast<float>(PyFloat_AsDouble(a[6]));
    d.theta = PyFloat_AsDouble(a[7]);
    d.positions = static_cast<const float*>(pos.data_ptr());
    d.ldp = T > 1 ? pos.stride(0) : n_axes;
    d.n_axes = static_cast<int>(n_axes);
    d.interleaved = PyObject_IsTrue(a[8]);
    if (PyErr_Occurred()) throw PythonError{};
    check(call_qk_norm_rope(&d, stream));
    PyObject *ro = result(a[9], qo), *rk = result(a[10], ko);
    PyObject* both = ro && rk ? PyTuple_Pack(2, ro, rk) : nullptr;
    Py_XDECREF(ro);
    Py_XDECREF(rk);
    return both;
  });
}

// (q, k, v, cu_q, cu_k, k_lens, causal, scale, out) -> out
PyObject* attention_packed(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 9);
    const Tensor &q = tensor(a[0], "attention_packed: q"), &k = tensor(a[1], "attention_packed: k"),
                 &v = tensor(a[2], "attention_packed: v"), &cu_q = tensor(a[3], "attention_packed: cu_q");
    const Tensor *cu_k = maybe(a[4], "attention_packed: cu_k"), *lens = maybe(a[5], "attention_packed: k_lens"),
                 *given = maybe(a[8], "attention_packed: out");
    const Heads hq = heads(q, "attention_packed: q"), hk = heads(k, "attention_packed: k"), hv = heads(v, "attention_packed: v");
    const int64_t D = q.size(2);
    const ScalarType type = q.scalar_type();
    if (v.sizes() != k.sizes() || k.size(2) != D || k.scalar_type() != type || v.scalar_type() != type ||
        (type != ScalarType::BFloat16 && type != ScalarType::Half))
      refuse("attention_packed: q, k, v must be BF16 or F16 of one head width, k and v of one shape");
    if (!cu_k) cu_k = &cu_q;
    const int64_t B = cu_q.numel() - 1;
    if (B < 0) refuse("attention_packed: cu_q must hold batch + 1 offsets");
    b2g_attention_packed_desc d{};
    d.cu_q = static_cast<const int32_t*>(vector(cu_q, ScalarType::Int, B + 1, "attention_packed: cu_q"));
    d.cu_k = static_cast<const int32_t*>(vector(*cu_k, ScalarType::Int, B + 1, "attention_packed: cu_k"));
    if (lens) d.k_lens = static_cast<const int32_t*>(vector(*lens, ScalarType::Int, B, "attention_packed: k_lens"));
    void* stream = stream_of({&q, &k, &v, &cu_q, cu_k, lens, given});
    const Tensor out = output_like(q, given, type, "attention_packed: out");
    const Heads ho = heads(out, "attention_packed: out");
    d.q = q.data_ptr(); d.k = k.data_ptr(); d.v = v.data_ptr(); d.out = out.data_ptr();
    d.dtype = static_cast<b2g_dtype>(dtype_of(type));
    d.ldq = hq.ld; d.hsq = hq.hs; d.ldk = hk.ld; d.hsk = hk.hs;
    d.ldv = hv.ld; d.hsv = hv.hs; d.ldo = ho.ld; d.hso = ho.hs;
    d.total_q = q.size(0); d.total_k = k.size(0); d.batch = B;
    d.n_head = static_cast<int>(q.size(1)); d.n_kv_head = static_cast<int>(k.size(1)); d.d_head = static_cast<int>(D);
    d.causal = PyObject_IsTrue(a[6]);
    d.scale = a[7] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(D)))
                              : static_cast<float>(PyFloat_AsDouble(a[7]));
    if (PyErr_Occurred()) throw PythonError{};
    Tensor space;
    const size_t n = call_attention_packed_workspace(&d);
    if (n) space = make({static_cast<int64_t>(n)}, ScalarType::Char, q);
    check(call_attention_packed(&d, n ? space.data_ptr() : nullptr, n, stream));
    return result(a[8], out);
  });
}

// (library: a ctypes-like callable that gives a symbol's address, error type)
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 2);
    auto address = [&](const char* name) {
      PyObject* o = PyObject_CallFunction(a[0], "s", name);
      void* p = o ? PyLong_AsVoidPtr(o) : nullptr;
      Py_XDECREF(o);
      if (!p) {
        if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "b2g_calls: no address for %s", name);
        throw PythonError{};
      }
      return p;
    };
    call_gemm_s8 = reinterpret_cast<decltype(call_gemm_s8)>(address("b2g_gemm_s8"));
    call_gemm_s8_workspace = reinterpret_cast<decltype(call_gemm_s8_workspace)>(address("b2g_gemm_s8_workspace"));
    call_qk_norm_rope = reinterpret_cast<decltype(call_qk_norm_rope)>(address("b2g_qk_norm_rope"));
    call_attention_packed = reinterpret_cast<decltype(call_attention_packed)>(address("b2g_attention_packed"));
    call_attention_packed_workspace =
        reinterpret_cast<decltype(call_attention_packed_workspace)>(address("b2g_attention_packed_workspace"));
    call_last_error = reinterpret_cast<decltype(call_last_error)>(address("b2g_last_error"));
    Py_INCREF(a[1]);
    Py_XDECREF(error_type);
    error_type = a[1];
    Py_RETURN_NONE;
  });
}

#define B2G_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {B2G_METHOD(gemm_s8), B2G_METHOD(qk_norm_rope), B2G_METHOD(attention_packed), B2G_METHOD(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b2g_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b2g_calls() {
  error_type = PyExc_RuntimeError;
  Py_INCREF(error_type);
  return PyModule_Create(&module);
}
