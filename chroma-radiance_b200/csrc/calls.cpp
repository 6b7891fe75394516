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
decltype(&b2g_block_means) call_block_means = nullptr;
decltype(&b2g_select_blocks) call_select_blocks = nullptr;
decltype(&b2g_attention_blocks) call_attention_blocks = nullptr;
decltype(&b2g_attention_blocks_workspace) call_attention_blocks_workspace = nullptr;
decltype(&b2g_lora_down) call_lora_down = nullptr;
decltype(&b2g_lora_up) call_lora_up = nullptr;
decltype(&b2g_lora) call_lora = nullptr;
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

int64_t whole(PyObject* o, const char* what) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PythonError{};
  if (v < 0) refuse(std::string(what) + " must not be negative");
  return v;
}

// The keys' side of a descriptor: offsets, lengths, sizes.
void key_side(b2g_attention_packed_desc& d, const Tensor& cu_k, const Tensor* lens, int64_t B, const std::string& who) {
  d.cu_k = static_cast<const int32_t*>(vector(cu_k, ScalarType::Int, B + 1, (who + ": cu_k").c_str()));
  if (lens) d.k_lens = static_cast<const int32_t*>(vector(*lens, ScalarType::Int, B, (who + ": k_lens").c_str()));
  d.batch = B;
}
bool is_half(ScalarType t) { return t == ScalarType::BFloat16 || t == ScalarType::Half; }

// (k, cu_k, k_lens, since, out) -> means
PyObject* block_means(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 5);
    const Tensor &k = tensor(a[0], "block_means: k"), &cu_k = tensor(a[1], "block_means: cu_k");
    const Tensor *lens = maybe(a[2], "block_means: k_lens"), *since = maybe(a[3], "block_means: since"),
                 *given = maybe(a[4], "block_means: out");
    const Heads hk = heads(k, "block_means: k");
    if (!is_half(k.scalar_type())) refuse("block_means: k must be BF16 or F16");
    const int64_t B = cu_k.numel() - 1, D = k.size(2);
    if (B < 0) refuse("block_means: cu_k must hold batch + 1 offsets");
    if (since && !given) refuse("block_means: since needs `out` (the means kept so far)");
    if (given && (given->dim() != 3 || given->size(1) != k.size(1) || given->size(2) != D || !given->is_contiguous() ||
                  given->scalar_type() != ScalarType::Float))
      refuse("block_means: out must be contiguous F32 [blocks, n_kv_head, d]");
    b2g_attention_packed_desc d{};
    key_side(d, cu_k, lens, B, "block_means");
    const int32_t* from = since ? static_cast<const int32_t*>(vector(*since, ScalarType::Int, B, "block_means: since")) : nullptr;
    void* stream = stream_of({&k, &cu_k, lens, since, given});
    const Tensor out = given ? *given : make({k.size(0) / 128 + B, k.size(1), D}, ScalarType::Float, k);
    d.k = k.data_ptr();
    d.dtype = static_cast<b2g_dtype>(dtype_of(k.scalar_type()));
    d.ldk = hk.ld; d.hsk = hk.hs;
    d.total_k = k.size(0);
    d.n_kv_head = static_cast<int>(k.size(1)); d.d_head = static_cast<int>(D);
    check(call_block_means(&d, from, static_cast<float*>(out.data_ptr()), out.size(0), stream));
    return result(a[4], out);
  });
}

// (q, means, cu_q, top, cu_k, k_lens, first, last, causal, max_k, out) -> chosen
PyObject* select_blocks(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 11);
    const Tensor &q = tensor(a[0], "select_blocks: q"), &means = tensor(a[1], "select_blocks: means"),
                 &cu_q = tensor(a[2], "select_blocks: cu_q");
    const Tensor *cu_k = maybe(a[4], "select_blocks: cu_k"), *lens = maybe(a[5], "select_blocks: k_lens"),
                 *given = maybe(a[10], "select_blocks: out");
    const Heads hq = heads(q, "select_blocks: q");
    const int64_t D = q.size(2);
    if (!is_half(q.scalar_type())) refuse("select_blocks: q must be BF16 or F16");
    if (means.dim() != 3 || means.size(2) != D || means.scalar_type() != ScalarType::Float || !means.is_contiguous())
      refuse("select_blocks: means must be contiguous F32 [blocks, n_kv_head, d]");
    if (!cu_k) cu_k = &cu_q;
    const int64_t B = cu_q.numel() - 1, blocks = means.size(0);
    if (B < 0) refuse("select_blocks: cu_q must hold batch + 1 offsets");
    b2g_attention_packed_desc d{};
    d.cu_q = static_cast<const int32_t*>(vector(cu_q, ScalarType::Int, B + 1, "select_blocks: cu_q"));
    key_side(d, *cu_k, lens, B, "select_blocks");
    const int64_t top = whole(a[3], "select_blocks: top"), first = whole(a[6], "select_blocks: first"),
                  last = whole(a[7], "select_blocks: last");
    int64_t most = blocks;  // blocks of a sequence
    if (a[9] != Py_None) {
      const int64_t keys = whole(a[9], "select_blocks: max_k");
      most = keys / 128 + (keys % 128 != 0);
    } else if (!given && blocks > 32 * 256) {  // (no one sequence need have so many)
      refuse("select_blocks: max_k, the keys of the longest sequence or more, is needed where means has more than 8192 rows");
    }
    if (given && (given->dim() != 3 || given->size(1) != means.size(1) || !given->is_contiguous() ||
                  given->scalar_type() != ScalarType::Int))
      refuse("select_blocks: out must be contiguous int32 [tiles, n_kv_head, words]");
    void* stream = stream_of({&q, &means, &cu_q, cu_k, lens, given});
    const Tensor out = given ? *given : make({q.size(0) / 128 + B, means.size(1), (most + 31) / 32}, ScalarType::Int, q);
    d.q = q.data_ptr();
    d.dtype = static_cast<b2g_dtype>(dtype_of(q.scalar_type()));
    d.ldq = hq.ld; d.hsq = hq.hs;
    d.total_q = q.size(0);
    d.total_k = blocks < (1 << 23) ? 128 * blocks : 1 << 30;  // (no key is read: a bound for the offsets)
    d.n_head = static_cast<int>(q.size(1)); d.n_kv_head = static_cast<int>(means.size(1)); d.d_head = static_cast<int>(D);
    d.causal = PyObject_IsTrue(a[8]);
    if (PyErr_Occurred()) throw PythonError{};
    check(call_select_blocks(&d, static_cast<const float*>(means.data_ptr()), blocks, top, first, last,
                             static_cast<int32_t*>(out.data_ptr()), out.size(0), out.size(2), stream));
    return result(a[10], out);
  });
}

// (q, k, v, chosen, cu_q, cu_k, k_lens, causal, scale, out) -> out
PyObject* attention_blocks(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 10);
    const Tensor &q = tensor(a[0], "attention_blocks: q"), &k = tensor(a[1], "attention_blocks: k"),
                 &v = tensor(a[2], "attention_blocks: v"), &chosen = tensor(a[3], "attention_blocks: chosen"),
                 &cu_q = tensor(a[4], "attention_blocks: cu_q");
    const Tensor *cu_k = maybe(a[5], "attention_blocks: cu_k"), *lens = maybe(a[6], "attention_blocks: k_lens"),
                 *given = maybe(a[9], "attention_blocks: out");
    const Heads hq = heads(q, "attention_blocks: q"), hk = heads(k, "attention_blocks: k"), hv = heads(v, "attention_blocks: v");
    const int64_t D = q.size(2);
    const ScalarType type = q.scalar_type();
    if (v.sizes() != k.sizes() || k.size(2) != D || k.scalar_type() != type || v.scalar_type() != type || !is_half(type))
      refuse("attention_blocks: q, k, v must be BF16 or F16 of one head width, k and v of one shape");
    if (chosen.dim() != 3 || chosen.size(1) != k.size(1) || chosen.scalar_type() != ScalarType::Int || !chosen.is_contiguous())
      refuse("attention_blocks: chosen must be contiguous int32 [tiles, n_kv_head, words]");
    if (!cu_k) cu_k = &cu_q;
    const int64_t B = cu_q.numel() - 1;
    if (B < 0) refuse("attention_blocks: cu_q must hold batch + 1 offsets");
    b2g_attention_packed_desc d{};
    d.cu_q = static_cast<const int32_t*>(vector(cu_q, ScalarType::Int, B + 1, "attention_blocks: cu_q"));
    key_side(d, *cu_k, lens, B, "attention_blocks");
    void* stream = stream_of({&q, &k, &v, &chosen, &cu_q, cu_k, lens, given});
    const Tensor out = output_like(q, given, type, "attention_blocks: out");
    const Heads ho = heads(out, "attention_blocks: out");
    d.q = q.data_ptr(); d.k = k.data_ptr(); d.v = v.data_ptr(); d.out = out.data_ptr();
    d.dtype = static_cast<b2g_dtype>(dtype_of(type));
    d.ldq = hq.ld; d.hsq = hq.hs; d.ldk = hk.ld; d.hsk = hk.hs;
    d.ldv = hv.ld; d.hsv = hv.hs; d.ldo = ho.ld; d.hso = ho.hs;
    d.total_q = q.size(0); d.total_k = k.size(0);
    d.n_head = static_cast<int>(q.size(1)); d.n_kv_head = static_cast<int>(k.size(1)); d.d_head = static_cast<int>(D);
    d.causal = PyObject_IsTrue(a[7]);
    d.scale = a[8] == Py_None ? static_cast<float>(1.0 / std::sqrt(static_cast<double>(D)))
                              : static_cast<float>(PyFloat_AsDouble(a[8]));
    if (PyErr_Occurred()) throw PythonError{};
    Tensor space;
    const size_t n = call_attention_blocks_workspace(&d, chosen.size(2));
    if (n) space = make({static_cast<int64_t>(n)}, ScalarType::Char, q);
    check(call_attention_blocks(&d, static_cast<const int32_t*>(chosen.data_ptr()), chosen.size(0), chosen.size(2),
                                n ? space.data_ptr() : nullptr, n, stream));
    return result(a[9], out);
  });
}

// The parts of lora's descriptor: requests; x and A; t; B, y and what is done with them.
void lora_requests(b2g_lora_desc& d, const Tensor& cu, const Tensor* ids, const std::string& who) {
  d.batch = cu.numel() - 1;
  if (d.batch < 0) refuse(who + ": cu must hold batch + 1 offsets");
  d.cu = static_cast<const int32_t*>(vector(cu, ScalarType::Int, d.batch + 1, (who + ": cu").c_str()));
  if (ids) d.ids = static_cast<const int32_t*>(vector(*ids, ScalarType::Int, d.batch, (who + ": ids").c_str()));
}
void lora_first(b2g_lora_desc& d, const Tensor& x, const Tensor& a, const std::string& who) {
  if (x.dim() != 2 || a.dim() != 3 || !is_half(x.scalar_type()) || a.scalar_type() != x.scalar_type())
    refuse(who + ": x [rows, K] and a [adapters, R, K] must be BF16 or F16, of one type");
  if (x.size(1) != a.size(2))
    refuse(who + ": K mismatch (" + std::to_string(x.size(1)) + " and " + std::to_string(a.size(2)) + ")");
  if (x.size(1) > 1 && (x.stride(1) != 1 || a.stride(2) != 1)) refuse(who + ": x and a need unit stride along K");
  d.rows = x.size(0); d.K = x.size(1); d.R = a.size(1); d.adapters = a.size(0);
  d.x = x.data_ptr(); d.a = a.data_ptr();
  d.dtype = static_cast<b2g_dtype>(dtype_of(x.scalar_type()));
  d.ldx = x.stride(0); d.lda = a.stride(1); d.a_stride = a.stride(0);
}
void lora_second(b2g_lora_desc& d, const Tensor& b, const Tensor& y, const Tensor* scale, PyObject* epilogue, const Tensor* gate,
                 const Tensor* given, const std::string& who) {
  if (b.dim() != 3 || !is_half(b.scalar_type()) || b.size(2) != d.R || (b.size(2) > 1 && b.stride(2) != 1))
    refuse(who + ": b must be BF16 or F16 [adapters, N, R] with unit stride along R");
  d.N = b.size(1);
  if (y.dim() != 2 || y.size(0) != d.rows || y.size(1) != d.N || (d.N > 1 && y.stride(1) != 1))
    refuse(who + ": y must be [rows, N] with unit column stride");
  if (given && (given->sizes() != y.sizes() || given->scalar_type() != y.scalar_type() || (d.N > 1 && given->stride(1) != 1)))
    refuse(who + ": out must be of y's shape and type with unit column stride");
  if (y.scalar_type() != ScalarType::Float && y.scalar_type() != b.scalar_type()) refuse(who + ": y must be F32 or of b's type");
  int epi = -1;
  static const struct { const char* name; int value; } kEpilogues[] = {
      {"none", B2G_EPI_NONE}, {"gelu", B2G_EPI_GELU}, {"gated_residual", B2G_EPI_GATED_RESIDUAL}, {"silu", B2G_EPI_SILU}};
  if (PyUnicode_Check(epilogue))
    for (const auto& e : kEpilogues)
      if (PyUnicode_CompareWithASCIIString(epilogue, e.name) == 0) epi = e.value;
  if (epi < 0) refuse(who + ": unknown epilogue");
  d.epilogue = static_cast<b2g_epilogue>(epi);
  if (epi == B2G_EPI_GATED_RESIDUAL) {
    if (!gate) refuse(who + ": gated_residual needs a gate");
    d.gate = static_cast<const float*>(vector(*gate, ScalarType::Float, d.N, (who + ": gate").c_str()));
  }
  if (scale) d.scale = static_cast<const float*>(vector(*scale, ScalarType::Float, b.size(0), (who + ": scale").c_str()));
  d.dtype = static_cast<b2g_dtype>(dtype_of(b.scalar_type()));
  d.adapters = b.size(0);
  d.b = b.data_ptr();
  d.ldb = b.stride(1); d.b_stride = b.stride(0);
  d.y = y.data_ptr();
  d.y_dtype = static_cast<b2g_dtype>(dtype_of(y.scalar_type()));
  d.ldy = y.stride(0);
}
void lora_out(b2g_lora_desc& d, const Tensor& out) {
  d.out = out.data_ptr();
  d.ldo = out.stride(0);
}
void lora_t(b2g_lora_desc& d, const Tensor& t, const std::string& who) {
  if (t.dim() != 2 || t.scalar_type() != ScalarType::Float || (t.size(1) > 1 && t.stride(1) != 1))
    refuse(who + ": t must be F32 [rows, R] with unit column stride");
  d.rows = t.size(0); d.R = t.size(1);
  d.t = static_cast<float*>(t.data_ptr());
  d.ldt = t.size(0) > 1 ? t.stride(0) : t.size(1);
}

// (x, a, cu, ids, out) -> t
PyObject* lora_down(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 5);
    const Tensor &x = tensor(a[0], "lora_down: x"), &w = tensor(a[1], "lora_down: a"), &cu = tensor(a[2], "lora_down: cu");
    const Tensor *ids = maybe(a[3], "lora_down: ids"), *given = maybe(a[4], "lora_down: out");
    b2g_lora_desc d{};
    lora_first(d, x, w, "lora_down");
    if (given && (given->dim() != 2 || given->size(0) != d.rows || given->size(1) != d.R)) refuse("lora_down: out must be F32 [rows, R]");
    lora_requests(d, cu, ids, "lora_down");
    void* stream = stream_of({&x, &w, &cu, ids, given});
    const Tensor out = given ? *given : make({d.rows, d.R}, ScalarType::Float, x);
    lora_t(d, out, "lora_down");
    check(call_lora_down(&d, stream));
    return result(a[4], out);
  });
}

// (t, b, y, cu, ids, scale, epilogue, gate, out) -> out
PyObject* lora_up(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 9);
    const Tensor &t = tensor(a[0], "lora_up: t"), &w = tensor(a[1], "lora_up: b"), &y = tensor(a[2], "lora_up: y"),
                 &cu = tensor(a[3], "lora_up: cu");
    const Tensor *ids = maybe(a[4], "lora_up: ids"), *scale = maybe(a[5], "lora_up: scale"), *gate = maybe(a[7], "lora_up: gate"),
                 *given = maybe(a[8], "lora_up: out");
    b2g_lora_desc d{};
    lora_t(d, t, "lora_up");
    lora_second(d, w, y, scale, a[6], gate, given, "lora_up");
    if (!d.gate) gate = nullptr;
    lora_requests(d, cu, ids, "lora_up");
    void* stream = stream_of({&t, &w, &y, &cu, ids, scale, gate, given});
    const Tensor out = given ? *given : make(y.sizes(), y.scalar_type(), y);
    lora_out(d, out);
    check(call_lora_up(&d, stream));
    return result(a[8], out);
  });
}

// (x, a, b, y, cu, ids, scale, epilogue, gate, out) -> out
PyObject* lora(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded([&]() -> PyObject* {
    expect(n_args, 10);
    const Tensor &x = tensor(a[0], "lora: x"), &down = tensor(a[1], "lora: a"), &up = tensor(a[2], "lora: b"),
                 &y = tensor(a[3], "lora: y"), &cu = tensor(a[4], "lora: cu");
    const Tensor *ids = maybe(a[5], "lora: ids"), *scale = maybe(a[6], "lora: scale"), *gate = maybe(a[8], "lora: gate"),
                 *given = maybe(a[9], "lora: out");
    b2g_lora_desc d{};
    lora_first(d, x, down, "lora");
    if (up.dim() != 3 || up.size(0) != down.size(0) || up.scalar_type() != down.scalar_type())
      refuse("lora: a and b must hold as many adapters, of one type");
    lora_second(d, up, y, scale, a[7], gate, given, "lora");
    if (!d.gate) gate = nullptr;
    lora_requests(d, cu, ids, "lora");
    void* stream = stream_of({&x, &down, &up, &y, &cu, ids, scale, gate, given});
    const Tensor t = make({d.rows, d.R}, ScalarType::Float, x);
    lora_t(d, t, "lora");
    const Tensor out = given ? *given : make(y.sizes(), y.scalar_type(), y);
    lora_out(d, out);
    check(call_lora(&d, stream));
    return result(a[9], out);
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
    call_block_means = reinterpret_cast<decltype(call_block_means)>(address("b2g_block_means"));
    call_select_blocks = reinterpret_cast<decltype(call_select_blocks)>(address("b2g_select_blocks"));
    call_attention_blocks = reinterpret_cast<decltype(call_attention_blocks)>(address("b2g_attention_blocks"));
    call_attention_blocks_workspace =
        reinterpret_cast<decltype(call_attention_blocks_workspace)>(address("b2g_attention_blocks_workspace"));
    call_lora_down = reinterpret_cast<decltype(call_lora_down)>(address("b2g_lora_down"));
    call_lora = reinterpret_cast<decltype(call_lora)>(address("b2g_lora"));
    call_lora_up = reinterpret_cast<decltype(call_lora_up)>(address("b2g_lora_up"));
    call_last_error = reinterpret_cast<decltype(call_last_error)>(address("b2g_last_error"));
    Py_INCREF(a[1]);
    Py_XDECREF(error_type);
    error_type = a[1];
    Py_RETURN_NONE;
  });
}

#define B2G_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {B2G_METHOD(gemm_s8), B2G_METHOD(qk_norm_rope), B2G_METHOD(attention_packed), B2G_METHOD(block_means),
                         B2G_METHOD(select_blocks), B2G_METHOD(attention_blocks), B2G_METHOD(lora_down), B2G_METHOD(lora_up),
                         B2G_METHOD(lora), B2G_METHOD(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "b2g_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_b2g_calls() {
  error_type = PyExc_RuntimeError;
  Py_INCREF(error_type);
  return PyModule_Create(&module);
}
