// s8.cu — 8-bit integer linear layers: per-row quantisation and the product for few tokens.
//
//   s[m] = max_k |x[m, k]| / 127          (1 for an all-zero row)
//   q[m, k] = round(x[m, k] * 127 / max)  (ties to even, |q| <= 127)
//   y[m, n] = act((sum_k q[m, k] w[n, k]) * s[m] * t[n] + bias[n])
//
// The sums are exact 32-bit integers (K <= 131071, so |sum| < 2^31 even for codes of -128 that a
// caller may give).  Products of many tokens run on tcgen05.mma kind::i8
// (gemm_tc.cu, KIND 3); those of up to kS8RowsMaxM tokens here, see s8_rows_kernel.  The reference's
// quantised path has the same form per channel (cublas_ops.cuh:294-352, quantize_activations
// kernels.cu:1988-2125), with the product in cuBLASLt.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>
#include "activations.cuh"
#include "engine.cuh"
#include "ptx_sm100.cuh"

namespace b2g {

namespace {

// ---------------------------------------------------------------------------- quantisation
//
// Bound by memory: each value is read once and kept in registers between the row's maximum and its
// codes.  kWarps warps share a row of up to 32 * kWarps * 8 * NV values (a block is 8 warps, so
// short rows go 8 to a block); longer rows are read twice.

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Eight consecutive values of a row (`vec`: 16-byte aligned and all of them inside it).
template <typename T>
__device__ __forceinline__ void load8(const T* p, int left, bool vec, float (&v)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = to_f32(h[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? to_f32(p[i]) : 0.f;
  }
}

// |v| as ordered integers: every finite value below every infinity below every NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }

// The code of v in a row whose largest magnitude is amax: the correctly rounded quotient
// v * 127 / amax, so that the exact halves (v = amax / 2 gives 63.5) round to even as the
// definition has them.  v * 127 is exact for 16-bit inputs.  live: a finite, nonzero amax.
__device__ __forceinline__ uint32_t code_s8(float v, float amax, bool live) {
  return live ? static_cast<uint32_t>(__float2int_rn(__fdiv_rn(v * 127.0f, amax))) & 0xFFu : 0u;
}

// Codes of one group of 8 values at column c.
__device__ __forceinline__ void store8(int8_t* row, int c, int cols, bool vec, const float (&v)[8], float amax, bool live) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    w[i] = code_s8(v[4 * i], amax, live) | code_s8(v[4 * i + 1], amax, live) << 8 |
           code_s8(v[4 * i + 2], amax, live) << 16 | code_s8(v[4 * i + 3], amax, live) << 24;
  if (vec) {
    *reinterpret_cast<uint2*>(row + c) = make_uint2(w[0], w[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (c + i < cols) row[c + i] = static_cast<int8_t>(w[i >> 2] >> (8 * (i & 3)));
  }
}

// A row's scale: max / 127, 1 for a row of zeros, NaN for a row with an infinity or a NaN (its
// codes are 0, and the NaN reaches every output of the row).
__device__ __forceinline__ float row_scale(uint32_t bits) {
  if (bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  return bits ? __fdiv_rn(__uint_as_float(bits), 127.0f) : 1.0f;
}

struct QuantArgs {
  const void* src;
  long long ld;
  int rows, cols;
  int src_vec, dst_vec; // 16-byte source rows, 8-byte destination rows
  int8_t* dst;
  long long dst_ld;
  float* scales;
};

template <int kWarps>
__device__ __forceinline__ uint32_t row_max(uint32_t m, uint32_t* red) {
  m = __reduce_max_sync(0xffffffffu, m);
  if constexpr (kWarps > 1) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = max(m, red[w]);
  }
  return m;
}

template <typename T, int kWarps, int NV>
__global__ void __launch_bounds__(256) quantize_rows_s8_kernel(const QuantArgs a) {
  static_assert(kWarps == 1 || kWarps == 8, "a block is 8 warps: 8 rows or one");
  __shared__ uint32_t red[8];
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kThreads = 32 * kWarps;
  const int t = static_cast<int>(threadIdx.x) % kThreads;
  const long long row = static_cast<long long>(blockIdx.x) * (8 / kWarps) + threadIdx.x / kThreads;
  if (row >= a.rows) return;  // (whole warps; one row per block otherwise)
  const T* s = static_cast<const T*>(a.src) + row * a.ld;
  float v[NV][8];
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * kThreads + t) * 8;
    if (c < a.cols) load8<T>(s + c, a.cols - c, a.src_vec && c + 8 <= a.cols, v[k]);
    else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[k][i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[k][i]));
  }
  m = row_max<kWarps>(m, red);
  const float amax = __uint_as_float(m);
  const bool live = m != 0 && m < 0x7F800000u;
  if (t == 0) a.scales[row] = row_scale(m);
  int8_t* d = a.dst + row * a.dst_ld;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * kThreads + t) * 8;
    if (c < a.cols) store8(d, c, a.cols, a.dst_vec && c + 8 <= a.cols, v[k], amax, live);
  }
}

// Rows of more than 16384 values: read twice (the second time from L2).
template <typename T>
__global__ void __launch_bounds__(256) quantize_long_rows_s8_kernel(const QuantArgs a) {
  __shared__ uint32_t red[8];
  griddep_wait();
  griddep_launch_dependents();
  const long long row = blockIdx.x;
  const T* s = static_cast<const T*>(a.src) + row * a.ld;
  uint32_t m = 0;
  for (int c = static_cast<int>(threadIdx.x) * 8; c < a.cols; c += 2048) {
    float v[8];
    load8<T>(s + c, a.cols - c, a.src_vec && c + 8 <= a.cols, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(v[i]));
  }
  m = row_max<8>(m, red);
  const float amax = __uint_as_float(m);
  const bool live = m != 0 && m < 0x7F800000u;
  if (threadIdx.x == 0) a.scales[row] = row_scale(m);
  int8_t* d = a.dst + row * a.dst_ld;
  for (int c = static_cast<int>(threadIdx.x) * 8; c < a.cols; c += 2048) {
    float v[8];
    load8<T>(s + c, a.cols - c, a.src_vec && c + 8 <= a.cols, v);
    store8(d, c, a.cols, a.dst_vec && c + 8 <= a.cols, v, amax, live);
  }
}

template <typename T>
b2g_status launch_quantize_s8(const QuantArgs& a, cudaStream_t st) {
  const char* what = "quantize_s8 launch";
  const dim3 one(static_cast<unsigned>(a.rows)), eight(static_cast<unsigned>((a.rows + 7) / 8)), block(256);
  if (a.cols <= 1024) return launch_pdl(quantize_rows_s8_kernel<T, 1, 4>, eight, block, 0, st, what, a);
  if (a.cols <= 4096) return launch_pdl(quantize_rows_s8_kernel<T, 8, 2>, one, block, 0, st, what, a);
  if (a.cols <= 8192) return launch_pdl(quantize_rows_s8_kernel<T, 8, 4>, one, block, 0, st, what, a);
  if (a.cols <= 16384) return launch_pdl(quantize_rows_s8_kernel<T, 8, 8>, one, block, 0, st, what, a);
  return launch_pdl(quantize_long_rows_s8_kernel<T>, one, block, 0, st, what, a);
}

// ---------------------------------------------------------------------------- few tokens
//
// Up to 8 * MT tokens: the weight [N, K] is read once and nothing else matters (one token at
// N = K = 5120: 26 MB).  A block owns 16 weight rows; its 8 warps take the 64-byte chunks of K in
// turn, so that together they read 512 consecutive bytes of each row.  Lane (g, t) of a warp
// loads 16 bytes of rows g and g + 8 and of token g at offset 16 t of the chunk: words (0, 1) and
// (2, 3) of these are the operands of two m16n8k32 products, whose K order is permuted in the
// same way for both operands and so does not matter.  The 8 warps' sums meet in shared memory.
constexpr int kRowsWarps = 8;
constexpr int kRowsUnroll = 4;  // chunks in flight per warp

struct RowsArgs {
  const int8_t* x;
  const int8_t* w;
  long long ldx, ldw;
  int M, N, K;
  const float* xs;
  const float* ws;
  const void* bias;
  int bias_kind;  // 0 none, 1 f32, 2 bf16
  void* d;
  int out;        // b2g_dtype
  long long ldd;
  int epi;
  const float* gate;
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes of a row at column k; the bytes at and past K are zero and are not read.
__device__ __forceinline__ uint4 load16(const int8_t* row, int k, int K, bool stream) {
  if (k + 16 <= K) {
    const uint4* p = reinterpret_cast<const uint4*>(row + k);
    return stream ? __ldcs(p) : __ldg(p);
  }
  uint32_t w[4] = {0, 0, 0, 0};
  for (int i = 0; i < 16; ++i)
    if (k + i < K) w[i >> 2] |= static_cast<uint32_t>(static_cast<uint8_t>(row[k + i])) << (8 * (i & 3));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int MT>
__global__ void __launch_bounds__(32 * kRowsWarps) s8_rows_kernel(const RowsArgs a) {
  __shared__ int sums[kRowsWarps][MT][16][8 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  griddep_wait();
  griddep_launch_dependents();
  // (rows past N and tokens past M repeat the last one; their sums are dropped)
  const int8_t* w0 = a.w + static_cast<long long>(min(n0 + g, a.N - 1)) * a.ldw + t * 16;
  const int8_t* w1 = a.w + static_cast<long long>(min(n0 + g + 8, a.N - 1)) * a.ldw + t * 16;
  const int8_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = a.x + static_cast<long long>(min(i * 8 + g, a.M - 1)) * a.ldx + t * 16;
  int acc[MT][4];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0;
  const int chunks = (a.K + 63) / 64, K = a.K - t * 16;
  for (int c0 = warp; c0 < chunks; c0 += kRowsWarps * kRowsUnroll) {
    uint4 u0[kRowsUnroll], u1[kRowsUnroll];
#pragma unroll
    for (int u = 0; u < kRowsUnroll; ++u) {
      const int k = (c0 + u * kRowsWarps) * 64;
      u0[u] = u1[u] = make_uint4(0, 0, 0, 0);
      if (k < a.K) {
        u0[u] = load16(w0, k, K, true);
        u1[u] = load16(w1, k, K, true);
      }
    }
#pragma unroll
    for (int u = 0; u < kRowsUnroll; ++u) {
      const int k = (c0 + u * kRowsWarps) * 64;
      if (k >= a.K) break;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint4 x = load16(xr[i], k, K, false);
        mma_s8(acc[i], u0[u].x, u1[u].x, u0[u].y, u1[u].y, x.x, x.y);
        mma_s8(acc[i], u0[u].z, u1[u].z, u0[u].w, u1[u].w, x.z, x.w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    sums[warp][i][g][2 * t] = acc[i][0];
    sums[warp][i][g][2 * t + 1] = acc[i][1];
    sums[warp][i][g + 8][2 * t] = acc[i][2];
    sums[warp][i][g + 8][2 * t + 1] = acc[i][3];
  }
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 128; o += 32 * kRowsWarps) {
    const int r = o & 15, m = o >> 4, n = n0 + r;
    if (n >= a.N || m >= a.M) continue;
    int sum = 0;
#pragma unroll
    for (int w = 0; w < kRowsWarps; ++w) sum += sums[w][m >> 3][r][m & 7];
    float y = __int2float_rn(sum) * a.xs[m] * a.ws[n];
    if (a.bias_kind == 1) y += static_cast<const float*>(a.bias)[n];
    if (a.bias_kind == 2) y += __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
    if (a.epi == B2G_EPI_GELU) y = gelu_tanh(y);
    if (a.epi == B2G_EPI_SILU) y = silu_fast(y);
    const long long at = m * a.ldd + n;
    if (a.epi == B2G_EPI_GATED_RESIDUAL) static_cast<float*>(a.d)[at] += a.gate[n] * y;
    else if (a.out == B2G_F32) static_cast<float*>(a.d)[at] = y;
    else if (a.out == B2G_BF16) static_cast<__nv_bfloat16*>(a.d)[at] = __float2bfloat16_rn(y);
    else static_cast<__half*>(a.d)[at] = __float2half_rn(y);
  }
}

// Most tokens that take s8_rows_kernel.
constexpr int64_t kS8RowsMaxM = 16;

b2g_status launch_rows(const GemmProblem& p, cudaStream_t st) {
  RowsArgs a{};
  a.x = static_cast<const int8_t*>(p.a); a.ldx = p.lda;
  a.w = static_cast<const int8_t*>(p.b); a.ldw = p.ldb;
  a.M = static_cast<int>(p.M); a.N = static_cast<int>(p.N); a.K = static_cast<int>(p.K);
  a.xs = p.a_scale; a.ws = p.b_scale;
  a.bias = p.bias; a.bias_kind = p.bias ? (p.bias_dtype == B2G_F32 ? 1 : 2) : 0;
  a.d = p.d; a.out = p.d_dtype; a.ldd = p.ldd;
  a.epi = p.epilogue; a.gate = p.gate;
  const dim3 grid(static_cast<unsigned>((p.N + 15) / 16)), block(32 * kRowsWarps);
  if (p.M <= 8) return launch_pdl(s8_rows_kernel<1>, grid, block, 0, st, "s8_rows launch", a);
  return launch_pdl(s8_rows_kernel<2>, grid, block, 0, st, "s8_rows launch", a);
}

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

// quantize_rows_s8 without its checks.
b2g_status run_quantize(const void* src, b2g_dtype src_dtype, int64_t rows, int64_t cols, int64_t ld,
                        int8_t* dst, int64_t dst_ld, float* scales, cudaStream_t st) {
  const int64_t esz = src_dtype == B2G_F32 ? 4 : 2;
  QuantArgs a{};
  a.src = src; a.ld = ld;
  a.rows = static_cast<int>(rows); a.cols = static_cast<int>(cols);
  a.src_vec = (reinterpret_cast<uintptr_t>(src) & 15u) == 0 && (ld * esz) % 16 == 0;
  a.dst_vec = (reinterpret_cast<uintptr_t>(dst) & 7u) == 0 && dst_ld % 8 == 0;
  a.dst = dst; a.dst_ld = dst_ld;
  a.scales = scales;
  if (src_dtype == B2G_BF16) return launch_quantize_s8<__nv_bfloat16>(a, st);
  if (src_dtype == B2G_F16) return launch_quantize_s8<__half>(a, st);
  return launch_quantize_s8<float>(a, st);
}

constexpr int64_t kS8MaxK = 131071;  // 128 * 128 * K < 2^31

}  // namespace

b2g_status quantize_rows_s8(const void* src, b2g_dtype src_dtype, int64_t rows, int64_t cols, int64_t ld, int8_t* dst,
                            int64_t dst_ld, float* scales, cudaStream_t st) {
  if (rows < 0 || cols < 0) return set_error(B2G_ERR_INVALID, "b2g_quantize_s8: negative size");
  if (rows == 0 || cols == 0) return B2G_OK;
  if (!src || !dst || !scales) return set_error(B2G_ERR_INVALID, "b2g_quantize_s8: null pointer");
  if (ld < cols || dst_ld < cols) return set_error(B2G_ERR_INVALID, "b2g_quantize_s8: ld < cols");
  if (rows > 0x7fffffff || cols > 0x7ffffff0)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_quantize_s8: too many rows or columns");
  if (src_dtype != B2G_F32 && src_dtype != B2G_BF16 && src_dtype != B2G_F16)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_quantize_s8: source must be F32, BF16 or F16");
  DeviceInfo* dev = nullptr;
  b2g_status s = device_info(&dev);
  if (s != B2G_OK) return s;
  return run_quantize(src, src_dtype, rows, cols, ld, dst, dst_ld, scales, st);
}

// Workspace of float activations: codes [M, round_up(K, 16)], then M scales.
size_t gemm_s8_workspace(int64_t M, int64_t K, b2g_dtype a_dtype) {
  if (a_dtype == B2G_S8 || M <= 0 || K <= 0) return 0;
  return static_cast<size_t>(round_up(M * round_up(K, 16), 256) + 4 * M);
}

b2g_status gemm_s8(const b2g_gemm_desc* d, const float* a_scale, const float* b_scale, void* workspace,
                   size_t workspace_bytes, cudaStream_t st) {
  if (!d) return set_error(B2G_ERR_INVALID, "b2g_gemm_s8: null descriptor");
  if (d->b_dtype != B2G_S8) return set_error(B2G_ERR_UNSUPPORTED, "b2g_gemm_s8: weights must be S8");
  if (d->a_dtype != B2G_S8 && d->a_dtype != B2G_F32 && d->a_dtype != B2G_BF16 && d->a_dtype != B2G_F16)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_gemm_s8: activations must be S8, F32, BF16 or F16");
  b2g_gemm_desc dd = *d;  // the checks of the 16-bit path, on a descriptor with bf16 operand tags
  dd.a_dtype = dd.b_dtype = B2G_BF16;
  GemmProblem p;
  bool empty = false;
  b2g_status s = desc_to_problem(&dd, "b2g_gemm_s8", &p, &empty);
  if (s != B2G_OK || empty) return s;
  if (p.K == 0 || p.K > kS8MaxK) return set_error(B2G_ERR_UNSUPPORTED, "b2g_gemm_s8: K must be in [1, 131071]");
  if (!b_scale || (d->a_dtype == B2G_S8 && !a_scale))
    return set_error(B2G_ERR_INVALID, "b2g_gemm_s8: S8 operands need their scales");
  if (p.M > 0x7fffffff - 256) return set_error(B2G_ERR_UNSUPPORTED, "b2g_gemm_s8: too many rows");
  p.a_dtype = p.b_dtype = B2G_S8;
  p.a_scale = a_scale;
  p.b_scale = b_scale;
  p.allow_split = false;
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  int8_t* q = nullptr;
  if (d->a_dtype != B2G_S8) {
    const size_t need = gemm_s8_workspace(p.M, p.K, d->a_dtype);
    void* ws = workspace;
    if (!ws && (s = workspace_get(need, &ws)) != B2G_OK) return s;
    if (workspace && (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
      return set_error(B2G_ERR_INVALID, "b2g_gemm_s8: the workspace is too small or not 256-byte aligned");
    q = static_cast<int8_t*>(ws);
    const int64_t kp = round_up(p.K, 16);
    p.a = q;
    p.lda = kp;
    p.a_scale = reinterpret_cast<float*>(q + round_up(p.M * kp, 256));
  }
  std::string why;
  if (!tc_gemm_supported(p, &why)) return set_error(B2G_ERR_UNSUPPORTED, "b2g_gemm_s8: " + why);
  if (q && (s = run_quantize(d->a, d->a_dtype, p.M, p.K, d->lda, q, p.lda, const_cast<float*>(p.a_scale), st)) !=
               B2G_OK)
    return s;
  if (p.M <= kS8RowsMaxM) return launch_rows(p, st);
  return tc_gemm_launch(p, st);
}

}  // namespace b2g
