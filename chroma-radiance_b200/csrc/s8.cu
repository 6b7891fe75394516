// s8.cu — 8-bit integer linear layers: per-row quantisation and the product for few tokens.
//
//   s[m] = max_k |x[m, k]| / 127          (1 for an all-zero row)
//   q[m, k] = round(x[m, k] * 127 / max)  (ties to even, |q| <= 127)
//   y[m, n] = act((sum_k q[m, k] w[n, k]) * t[n] * s[m] + bias[n])
//
// The sums are exact 32-bit integers (K <= 131071, so |sum| < 2^31 even for codes of -128 that a
// caller may give).  Products of many tokens run on tcgen05.mma kind::i8
// (gemm_tc.cu, KIND 3); the others here, see s8_one_kernel and s8_split_kernel.  The reference's
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
// Each value is read once and kept in registers between the row's maximum and its
// codes.  kWarps warps share a row of up to 32 * kWarps * 8 * NV values (a block is 8 warps, so rows of up to
// 1024 go 8 to a block; a warp for rows of 3072 took 21.6 us where a block takes 14.5); longer rows are
// read twice.  4608 x 3072 of bf16: 14.5 us (2.9 TB/s), of f32: 15.3 us (4.6 TB/s): not the bytes count but a block's chain
// of load, barrier and store, with no next row on its way.  128 x 5120 of bf16: 3.0 us, most of it
// one round trip to memory, one through the block and the launch.

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

// Eight consecutive values of a row, as they are in memory.
template <typename T>
struct Raw8 {
  uint32_t w[2 * sizeof(T)];
};
template <typename T>
__device__ __forceinline__ Raw8<T> zero8() {
  Raw8<T> r;
#pragma unroll
  for (uint32_t i = 0; i < 2 * sizeof(T); ++i) r.w[i] = 0u;
  return r;
}
// `vec`: 16-byte aligned and all of them inside the row.
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p, int left, bool vec) {
  Raw8<T> r;
  if (vec) {
#pragma unroll
    for (uint32_t i = 0; i < sizeof(T) / 2; ++i) {
      const uint4 u = reinterpret_cast<const uint4*>(p)[i];
      r.w[4 * i] = u.x; r.w[4 * i + 1] = u.y; r.w[4 * i + 2] = u.z; r.w[4 * i + 3] = u.w;
    }
  } else {
    r = zero8<T>();
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (i >= left) continue;
      if constexpr (sizeof(T) == 4) r.w[i] = reinterpret_cast<const uint32_t*>(p)[i];
      else r.w[i >> 1] |= static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(p)[i]) << (16 * (i & 1));
    }
  }
  return r;
}
template <typename T>
__device__ __forceinline__ float value8(const Raw8<T>& r, int i) {
  if constexpr (sizeof(T) == 4) {
    return __uint_as_float(r.w[i]);
  } else {
    const uint16_t h = static_cast<uint16_t>(r.w[i >> 1] >> (16 * (i & 1)));
    return to_f32(*reinterpret_cast<const T*>(&h));
  }
}

// The largest |v| as ordered integers: every finite value below every infinity below every NaN.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
template <typename T, int NV>
__device__ __forceinline__ uint32_t top8(const Raw8<T> (&r)[NV]) {
  uint32_t m = 0;
#pragma unroll
  for (int k = 0; k < NV; ++k)
#pragma unroll
    for (uint32_t i = 0; i < 2 * sizeof(T); ++i) {
      if constexpr (sizeof(T) == 4) m = max(m, r[k].w[i] & 0x7FFFFFFFu);
      else m = __vmaxu2(m, r[k].w[i] & 0x7FFF7FFFu);  // (the same order in 16 bits)
    }
  if constexpr (sizeof(T) == 2) {
    const uint16_t h = static_cast<uint16_t>(max(m & 0xFFFFu, m >> 16));
    m = abs_bits(to_f32(*reinterpret_cast<const T*>(&h)));
  }
  return m;
}

// A row's codes are v * 127 / amax rounded to integers, exact halves (v = amax / 2 gives 63.5: common in
// 16-bit rows) to even as the definition has them.  A division for every value costs more than the copy;
// v * (127 / amax) is within 2^-15 of the quotient (two roundings, 2^-24 each of at most 127) and rounds
// to the same integer unless it lies that close to a half h.  That is tested, with 2^-14, for 8 values at once,
// and then the sign of v * 127 - h * amax decides: one fma, exact for 16-bit inputs, whose v * 127 is.
struct RowCodes {
  float amax, inv, scale;  // amax and inv of values times scale, a power of two: 127 * amax and 127 / amax stay finite
  bool live;               // a finite, nonzero amax
};
__device__ __forceinline__ RowCodes row_codes(uint32_t top) {
  const float amax = __uint_as_float(top);
  RowCodes r{1.f, 0.f, amax > 1.0f ? 0x1p-8f : 0x1p64f, top != 0 && top < 0x7F800000u};
  if (r.live) {
    r.amax = amax * r.scale;
    r.inv = __fdiv_rn(127.0f, r.amax);
  }
  return r;
}

// Codes of one group of 8 values at column c.
template <typename T>
__device__ __forceinline__ void store8(int8_t* row, int c, int cols, bool vec, const Raw8<T>& v, const RowCodes& r) {
  uint32_t w[2] = {0u, 0u};
  if (r.live) {
    int q[8];
    bool sure = true;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float y = value8<T>(v, i) * r.scale * r.inv;
      q[i] = __float2int_rn(y);
      sure = sure && fabsf(y - static_cast<float>(q[i])) < 0.5f - 0x1p-14f;
    }
    if (!sure) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = value8<T>(v, i) * r.scale, y = x * r.inv;
        const int k = __float2int_rd(y);
        const float h = static_cast<float>(k) + 0.5f, over = fmaf(-h, r.amax, x * 127.0f);
        if (fabsf(y - h) <= 0x1p-14f) q[i] = over > 0.f ? k + 1 : over < 0.f ? k : k + (k & 1);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i >> 2] |= (static_cast<uint32_t>(q[i]) & 0xFFu) << (8 * (i & 3));
  }
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
  Raw8<T> v[NV];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * kThreads + t) * 8;
    v[k] = c < a.cols ? load8<T>(s + c, a.cols - c, a.src_vec && c + 8 <= a.cols) : zero8<T>();
  }
  uint32_t m = top8<T, NV>(v);
  m = row_max<kWarps>(m, red);
  const RowCodes rc = row_codes(m);
  if (t == 0) a.scales[row] = row_scale(m);
  int8_t* d = a.dst + row * a.dst_ld;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * kThreads + t) * 8;
    if (c < a.cols) store8<T>(d, c, a.cols, a.dst_vec && c + 8 <= a.cols, v[k], rc);
  }
}

// Rows of more than 16384 values: read twice (the second time from L2).  Columns are counted in 64 bits: a step past the
// longest row's end would not fit 32.
template <typename T>
__global__ void __launch_bounds__(256) quantize_long_rows_s8_kernel(const QuantArgs a) {
  __shared__ uint32_t red[8];
  griddep_wait();
  griddep_launch_dependents();
  const long long row = blockIdx.x;
  const T* s = static_cast<const T*>(a.src) + row * a.ld;
  uint32_t m = 0;
  for (int64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
    const Raw8<T> v[1] = {load8<T>(s + c, static_cast<int>(a.cols - c), a.src_vec && c + 8 <= a.cols)};
    m = max(m, top8<T, 1>(v));
  }
  m = row_max<8>(m, red);
  const RowCodes rc = row_codes(m);
  if (threadIdx.x == 0) a.scales[row] = row_scale(m);
  int8_t* d = a.dst + row * a.dst_ld;
  for (int64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
    const Raw8<T> v = load8<T>(s + c, static_cast<int>(a.cols - c), a.src_vec && c + 8 <= a.cols);
    store8<T>(d, static_cast<int>(c), a.cols, a.dst_vec && c + 8 <= a.cols, v, rc);
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

// ---------------------------------------------------------------------------- epilogue of the kernels below

struct S8Out {
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

// What a channel's outputs have in common.
struct Channel {
  float ws, bias, gate;
};
__device__ __forceinline__ Channel load_channel(const S8Out& o, int n) {
  Channel c{__ldg(o.ws + n), 0.f, 0.f};
  if (o.bias_kind == 1) c.bias = __ldg(static_cast<const float*>(o.bias) + n);
  if (o.bias_kind == 2) c.bias = __bfloat162float(static_cast<const __nv_bfloat16*>(o.bias)[n]);
  if (o.epi == B2G_EPI_GATED_RESIDUAL) c.gate = __ldg(o.gate + n);
  return c;
}
// Writes D[m, n] from the exact integer sum.
__device__ __forceinline__ void put_s8(const S8Out& o, const Channel& c, long long m, int n, int sum, float xs) {
  // (the channel's scale first: a token's may be near either end of the type's range)
  float y = fmaf(__int2float_rn(sum) * c.ws, xs, c.bias);
  if (o.epi == B2G_EPI_GELU) y = gelu_tanh<true>(y);
  if (o.epi == B2G_EPI_SILU) y = silu_fast<true>(y);
  const long long at = m * o.ldd + n;
  if (o.epi == B2G_EPI_GATED_RESIDUAL) static_cast<float*>(o.d)[at] += c.gate * y;
  else if (o.out == B2G_F32) static_cast<float*>(o.d)[at] = y;
  else if (o.out == B2G_BF16) static_cast<__nv_bfloat16*>(o.d)[at] = __float2bfloat16_rn(y);
  else static_cast<__half*>(o.d)[at] = __float2half_rn(y);
}

// ---------------------------------------------------------------------------- a token or a few
//
// Float activations of up to 8 tokens and kOneMax values in all: one launch that quantises and
// multiplies.  The weight [N, K] is read once and nothing else matters (one token at N = K = 5120:
// 26 MB, 8.4 us from HBM, 3.1 TB/s, 6.9 us with the weight in L2; N = 16 takes 4.2 us, a latency chain of token, maximum, codes,
// products), so the
// tokens are quantised by every block for itself, while its weights are on their way: a launch of its own before
// this one costs 3 to 4 us.  8 tokens of 2048: 9.6 us; past kOneMax quantising everywhere costs more than it saves.
// A block takes 16 weight rows at a time; its 8 warps take the
// 64-byte chunks of K in turn, so that together they read 512 consecutive bytes of each row.  Lane (g, t)
// of a warp has 16 bytes of rows g and g + 8 and of token g at offset 16 t of the chunk: words (0, 1) and
// (2, 3) of these are the operands of two m16n8k32 products, whose K order is permuted in the same way
// for both operands and so does not matter.  The weights go through the lane's own slots of shared
// memory (cp.async, across the block's row groups without a stop; nothing is shared between lanes).  The
// warps' sums meet in shared memory.
constexpr int kOneWarps = 8;
constexpr int kOneStages = 6;                                      // chunks on the way per warp
constexpr uint32_t kOneRing = kOneWarps * kOneStages * 1024u;      // bytes
constexpr int kOneMax = 16384;                                     // values of all tokens (their number a power of two)
constexpr uint32_t kOneSmem = kOneRing + kOneMax + 8 * 192;        // ring, codes

struct OneArgs {
  const void* x;
  long long ldx;
  int x_vec;      // 16-byte rows of x
  const int8_t* w;
  long long ldw;
  int M, N, K;
  int pitch;      // bytes of a token's codes in shared memory: past K, 64 modulo 128
  int row_warps;  // warps that quantise one token: 8 over M's power of two
  S8Out o;
};

__device__ __forceinline__ void mma_s8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint4 lds16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}
// 16 bytes of a row at column k into shared memory; those at and past K are zeros and are not read.
__device__ __forceinline__ void copy16(uint32_t dst, const int8_t* row, int k, int K) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(k < K ? row + k : row),
               "r"(min(max(K - k, 0), 16))
               : "memory");
}

// Blocks per SM: by the registers that hold a token's values.
template <typename T, int NV>
constexpr int kOneBlocks = NV * sizeof(T) <= 16 ? 3 : 2;

// NV groups of 8 values per lane.
template <typename T, int NV>
__global__ void __launch_bounds__(32 * kOneWarps, kOneBlocks<T, NV>) s8_one_kernel(const OneArgs a) {
  extern __shared__ __align__(16) uint8_t smem_one[];
  uint8_t* codes = smem_one + kOneRing;
  __shared__ uint32_t red[kOneWarps];
  __shared__ float scale[8];
  __shared__ int sums[kOneWarps][8][16 + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem_one) + warp * (kOneStages * 1024) + lane * 16;
  const int chunks = (a.K + 63) / 64, groups = (a.N + 15) / 16, stride = static_cast<int>(gridDim.x);
  griddep_wait();
  griddep_launch_dependents();
  // The next chunk to fetch: of row group fg (rows past N repeat the last one; their sums are dropped).
  int fg = blockIdx.x, fc = warp, fst = 0;
  const int8_t *w0 = nullptr, *w1 = nullptr;
  auto to_group = [&]() {
    w0 = a.w + static_cast<long long>(min(fg * 16 + g, a.N - 1)) * a.ldw;
    w1 = a.w + static_cast<long long>(min(fg * 16 + g + 8, a.N - 1)) * a.ldw;
  };
  to_group();
  auto fetch = [&]() {
    if (fg < groups && fc < chunks) {
      copy16(ring + fst * 1024, w0, fc * 64 + t * 16, a.K);
      copy16(ring + fst * 1024 + 512, w1, fc * 64 + t * 16, a.K);
      fst = fst + 1 == kOneStages ? 0 : fst + 1;
      fc += kOneWarps;
      if (fc >= chunks) {
        fc = warp;
        fg += stride;
        to_group();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kOneStages - 1; ++i) fetch();
  // The tokens' codes, zeros from K to the pitch: row_warps warps per token.
  {
    const int m = warp / a.row_warps, at = (warp - m * a.row_warps) * 32 + lane, step = a.row_warps * 32;
    const T* row = static_cast<const T*>(a.x) + m * a.ldx;
    Raw8<T> v[NV];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * step + at) * 8;
      v[k] = m < a.M && c < a.K ? load8<T>(row + c, a.K - c, a.x_vec && c + 8 <= a.K) : zero8<T>();
    }
    uint32_t top = top8<T, NV>(v);
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[warp] = top;
    __syncthreads();
    for (int i = 0; i < a.row_warps; ++i) top = max(top, red[m * a.row_warps + i]);
    const RowCodes rc = row_codes(top);
    if (m < a.M) {
      if (at == 0) scale[m] = row_scale(top);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * step + at) * 8;
        if (c < a.pitch) store8<T>(reinterpret_cast<int8_t*>(codes) + m * a.pitch, c, a.pitch, true, v[k], rc);
      }
      // (the values end before the pitch does where the lanes' groups do)
      for (int c = (NV * step + at) * 8; c < a.pitch; c += step * 8) *reinterpret_cast<uint2*>(codes + m * a.pitch + c) = make_uint2(0, 0);
    }
    __syncthreads();
  }
  const uint32_t x = smem_u32(codes) + min(g, a.M - 1) * a.pitch + t * 16;
  int st = 0;
  for (int group = blockIdx.x; group < groups; group += stride) {
    int acc[4] = {0, 0, 0, 0};
    for (int c = warp; c < chunks; c += kOneWarps) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kOneStages - 2) : "memory");
      fetch();  // (over the stage used up in the last round)
      const uint4 lo = lds16(ring + st * 1024), hi = lds16(ring + st * 1024 + 512), xv = lds16(x + c * 64);
      mma_s8(acc, lo.x, hi.x, lo.y, hi.y, xv.x, xv.y);
      mma_s8(acc, lo.z, hi.z, lo.w, hi.w, xv.z, xv.w);
      st = st + 1 == kOneStages ? 0 : st + 1;
    }
    sums[warp][2 * t][g] = acc[0];
    sums[warp][2 * t + 1][g] = acc[1];
    sums[warp][2 * t][g + 8] = acc[2];
    sums[warp][2 * t + 1][g + 8] = acc[3];
    __syncthreads();
    const int m = threadIdx.x >> 4, n = group * 16 + (threadIdx.x & 15);
    if (m < a.M && n < a.N) {
      const Channel ch = load_channel(a.o, n);
      int sum = 0;
#pragma unroll
      for (int v = 0; v < kOneWarps; ++v) sum += sums[v][m][threadIdx.x & 15];
      put_s8(a.o, ch, m, n, sum, scale[m]);
    }
    __syncthreads();
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
}

// ---------------------------------------------------------------------------- up to 128 tokens, or few channels
//
// With few tokens the tiles of gemm_tc.cu are few (N / 128), and each streams its 128 weight rows
// through one SM at the 90 bytes per ns that an SM takes in: its time grows with K alone.  Here the weights are
// the MMA's M side (128 rows) and the tokens its N side (16 to 128), and a cluster of up to 8 CTAs shares out the K
// axis of a tile: every SM streams, the tokens are read once per 128 weight rows, and the exact integer sums of
// the cluster meet through distributed shared memory, each CTA finishing its share of the tokens.  No
// workspace, no second launch, and the order of the sums does not matter.  After a quantising launch of the same call
// the weights set out before it is done.
// Time grows by 0.07 us per token (sums through shared memory, the tokens once more per CTA), so that it pays up to
// M = K / 48.  us with the quantiser, here against gemm_tc.cu's tiles, [N, K] and tokens:
//   [5120, 5120] 16: 12.2, 19.1; 64: 15.6, 19.3; 96: 19.1, 19.5; 128: 22, 18.7    [1024, 1024] 64: 13.9, 9.2
//   [21504, 3072] 16: 15.6, 22.4; 64: 20.3, 22.2; 128: 26.5, 22.5    [3072, 12288] 16: 17.7, 37.7; 128: 28.2, 38.6
// More tokens, in blocks of up to 128, where few channels leave a cluster of 3 or more to each block and tile
// (codes given): [512, 10944] 148: 10.8, 26.8; 600: 18.5, 27.1    [1024, 10944] 600: 22.3, 27.9    [256, 15360] 1000: 17, 36
//   warp 0 TMA, warp 1 MMA (kind::i8, sums in TMEM), warps 2-5 epilogue (a weight row per thread).
constexpr int kSplitThreads = 192;
constexpr uint32_t kSplitW = 128 * 128;  // bytes of a stage's weights: 128 rows x 128 of K
constexpr int kSplitMaxStages = 8;

struct SplitArgs {
  int M, N, nkb;     // nkb: blocks of 128 of K
  int tokens;        // per block of tokens: a multiple of 16, at most 128
  int stages;
  uint32_t tmem_cols;
  int early;         // the weights do not depend on the launch before this one
  int* err;
  S8Out o;
};

__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(r));
  return r;
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}

__global__ void __launch_bounds__(kSplitThreads, 1)
    s8_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX, const SplitArgs a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t full[kSplitMaxStages], empty[kSplitMaxStages], done, drain;
  __shared__ uint32_t tmem_slot;
  const uint32_t x_bytes = static_cast<uint32_t>(a.tokens) * 128u, stage_bytes = kSplitW + x_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = static_cast<int>(cluster_size()), rank = static_cast<int>(cluster_ctarank());
  const int n0 = static_cast<int>(blockIdx.x / S) * 128, m0 = static_cast<int>(blockIdx.y) * a.tokens;
  const int m_end = min(a.M, m0 + a.tokens);
  const int kb0 = static_cast<int>(static_cast<long long>(a.nkb) * rank / S);
  const int kb1 = static_cast<int>(static_cast<long long>(a.nkb) * (rank + 1) / S);
  if (warp == 0 && lane == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    mbar_init(&drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmW);
    tma_prefetch_desc(&tmX);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, a.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (!a.early) griddep_wait();
  if (warp == 0) {
    if (lane == 0) {
      const uint64_t once = policy_evict_first(), keep = policy_evict_last();
      auto load_w = [&](int kb, int st) {
        mbar_arrive_expect_tx(&full[st], stage_bytes);
        tma_load_3d(smem + st * stage_bytes, &tmW, &full[st], kb * 128, n0, 0, once);
      };
      auto load_x = [&](int kb, int st) {
        tma_load_3d(smem + st * stage_bytes + kSplitW, &tmX, &full[st], kb * 128, m0, 0, keep);
      };
      int issued = 0;
      for (; issued < a.stages && kb0 + issued < kb1; ++issued) load_w(kb0 + issued, issued);
      if (a.early) griddep_wait();
      for (int i = 0; i < issued; ++i) load_x(kb0 + i, i);
      int st = 0;
      uint32_t parity = 0;
      for (int kb = kb0 + issued; kb < kb1; ++kb) {
        if (!mbar_wait(&empty[st], parity, a.err, kErrWaitProducer)) break;
        load_w(kb, st);
        load_x(kb, st);
        ++issued;
        if (++st == a.stages) {
          st = 0;
          parity ^= 1u;
        }
      }
      // Copies land before the shared memory is used for the sums or goes away (they have, unless
      // another role gave up early).
      for (int i = max(0, issued - a.stages); i < issued; ++i)
        mbar_wait_drain(&full[i % a.stages], static_cast<uint32_t>(i / a.stages) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = idesc_make_s8(128, a.tokens);
      int st = 0;
      uint32_t parity = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(ok = mbar_wait(&full[st], parity, a.err, kErrWaitMma))) break;
        tc_fence_after();
        const uint32_t w0 = smem_u32(smem + st * stage_bytes), x0 = w0 + kSplitW;
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_i8(tmem, smem_desc_k_sw128(w0 + k * 32), smem_desc_k_sw128(x0 + k * 32), idesc, (kb != kb0 || k != 0) ? 1u : 0u);
        umma_commit(&empty[st]);
        if (++st == a.stages) {
          st = 0;
          parity ^= 1u;
        }
      }
      if (ok) umma_commit(&done);
      umma_commit(&drain);  // (all MMAs have retired before TMEM is released)
      mbar_wait_drain(&drain, 0);
    }
  }
  const int quarter = warp & 3, row = quarter * 32 + lane, n = n0 + row;  // (warps 2-5)
  const uint32_t lane_tmem = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
  int* part = reinterpret_cast<int*>(smem);  // [token][128] sums of this CTA, over the ring
  bool ok = true;
  if (warp >= 2) {
    if (a.early) griddep_wait();
    ok = __all_sync(0xffffffffu, mbar_wait(&done, 0, a.err, kErrWaitEpilogue));
    tc_fence_after();
  }
  griddep_launch_dependents();
  Channel ch{0.f, 0.f, 0.f};
  if (warp >= 2 && n < a.N) ch = load_channel(a.o, n);
  // 16 tokens' outputs of this thread's channel, from token m on.
  auto put = [&](const int (&sum)[16], int m, int count) {
    float xs[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) xs[i] = i < count ? __ldg(a.o.xs + m + i) : 0.f;
    if (n < a.N) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (i < count) put_s8(a.o, ch, m + i, n, sum[i], xs[i]);
    }
  };
  if (S == 1) {
    if (warp >= 2 && ok) {
      for (int c = 0; m0 + c < m_end; c += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(lane_tmem + c, r);
        tmem_wait_ld();
        int sum[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[i] = static_cast<int>(r[i]);
        put(sum, m0 + c, min(16, m_end - m0 - c));
      }
    }
  } else {
    if (warp >= 2 && ok) {
      for (int c = 0; c < a.tokens; c += 16) {
        uint32_t r[16];
        tmem_ld_32x32b_x16(lane_tmem + c, r);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) part[(c + i) * 128 + row] = static_cast<int>(r[i]);
      }
    }
    __syncwarp();
    cluster_sync_all();  // every CTA's sums are in its shared memory
    if (warp >= 2 && ok) {
      const int live = m_end - m0, c0 = live * rank / S, c1 = live * (rank + 1) / S;
      const uint32_t mine = smem_u32(part) + row * 4;
      for (int c = c0; c < c1; c += 16) {
        int sum[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) sum[i] = 0;
        const int count = min(16, c1 - c);
#pragma unroll 2
        for (int q = 0; q < S; ++q) {
          const uint32_t from = map_to_cta(mine, static_cast<uint32_t>(q)) + c * 512;
          int v[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = i < count ? ld_cluster(from + i * 512) : 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum[i] += v[i];
        }
        put(sum, m0 + c, count);
      }
    }
    __syncwarp();
    cluster_sync_all();  // nobody leaves while its sums are still read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, a.tmem_cols);
  }
}

// Most tokens that take s8_split_kernel.
constexpr int64_t kSplitTokens = 128;  // per block of tokens

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

S8Out out_args(const GemmProblem& p) {
  S8Out o{};
  o.xs = p.a_scale; o.ws = p.b_scale;
  o.bias = p.bias; o.bias_kind = p.bias ? (p.bias_dtype == B2G_F32 ? 1 : 2) : 0;
  o.d = p.d; o.out = p.d_dtype; o.ldd = p.ldd;
  o.epi = p.epilogue; o.gate = p.gate;
  return o;
}

template <typename T, int NV>
b2g_status launch_one_as(const OneArgs& a, const DeviceInfo* dev, cudaStream_t st) {
  b2g_status s = check_cuda(cudaFuncSetAttribute(s8_one_kernel<T, NV>, cudaFuncAttributeMaxDynamicSharedMemorySize, kOneSmem),
                            "cudaFuncSetAttribute(s8_one)");
  if (s != B2G_OK) return s;
  const int groups = (a.N + 15) / 16, most = kOneBlocks<T, NV> * dev->num_sms;
  return launch_pdl(s8_one_kernel<T, NV>, dim3(static_cast<unsigned>(groups < most ? groups : most)), dim3(32 * kOneWarps),
                    kOneSmem, st, "s8_one launch", a);
}

int64_t pow2_ceil(int64_t v) {
  int64_t r = 1;
  while (r < v) r *= 2;
  return r;
}

template <typename T>
b2g_status launch_one(const GemmProblem& p, const DeviceInfo* dev, cudaStream_t st) {
  OneArgs a{};
  a.x = p.a; a.ldx = p.lda;
  a.x_vec = (reinterpret_cast<uintptr_t>(p.a) & 15u) == 0 && (p.lda * static_cast<int64_t>(sizeof(T))) % 16 == 0;
  a.w = static_cast<const int8_t*>(p.b); a.ldw = p.ldb;
  a.M = static_cast<int>(p.M); a.N = static_cast<int>(p.N); a.K = static_cast<int>(p.K);
  a.pitch = static_cast<int>(round_up(p.K, 128) + 64);
  a.row_warps = static_cast<int>(kOneWarps / pow2_ceil(p.M));
  a.o = out_args(p);
  // 8 * NV values per lane, 256 lanes over all tokens.
  return pow2_ceil(p.M) * p.K <= 8192 ? launch_one_as<T, 4>(a, dev, st) : launch_one_as<T, 8>(a, dev, st);
}

b2g_status launch_split(const GemmProblem& p, bool early, const DeviceInfo* dev, cudaStream_t st) {
  SplitArgs a{};
  a.M = static_cast<int>(p.M); a.N = static_cast<int>(p.N);
  a.nkb = static_cast<int>((p.K + 127) / 128);
  const int64_t blocks = (p.M + kSplitTokens - 1) / kSplitTokens;
  a.tokens = static_cast<int>(round_up((p.M + blocks - 1) / blocks, 16));
  a.tmem_cols = 32;
  while (a.tmem_cols < static_cast<uint32_t>(a.tokens)) a.tmem_cols *= 2;
  const int64_t tiles = (p.N + 127) / 128;
  // As many CTAs per tile as find an SM, each of 4 blocks of K or more.
  int64_t S = dev->num_sms / (tiles * blocks);
  if (S > a.nkb / 4) S = a.nkb / 4;
  if (S > 8) S = 8;
  if (S < 1) S = 1;
  // Two CTAs per SM: clusters then find room everywhere, and N a little past 128 * the SMs takes one wave.
  const uint32_t stage = kSplitW + static_cast<uint32_t>(a.tokens) * 128u, sums = S > 1 ? static_cast<uint32_t>(a.tokens) * 512u : 0u;
  int stages = static_cast<int>(110 * 1024 / stage);
  if (stages > kSplitMaxStages) stages = kSplitMaxStages;
  a.stages = stages;
  a.early = early ? 1 : 0;
  a.err = dev->err_word;
  a.o = out_args(p);
  CUtensorMap tw, tx;
  b2g_status s;
  if ((s = make_operand_map(&tw, p.b, B2G_S8, p.K, p.N, p.ldb, 1, p.ldb * p.N, 128)) != B2G_OK) return s;
  if ((s = make_operand_map(&tx, p.a, B2G_S8, p.K, p.M, p.lda, 1, p.lda * p.M, static_cast<uint32_t>(a.tokens))) != B2G_OK)
    return s;
  const uint32_t used = static_cast<uint32_t>(stages) * stage, smem = 1024 + (used > sums ? used : sums);
  if ((s = check_cuda(cudaFuncSetAttribute(s8_split_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 111 * 1024),
                      "cudaFuncSetAttribute(s8_split)")) != B2G_OK)
    return s;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * S), static_cast<unsigned>(blocks));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(S);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  s = check_cuda(cudaLaunchKernelEx(&cfg, s8_split_kernel, tw, tx, a), "s8_split launch");
  if (s == B2G_OK) note_launch();
  return s;
}

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

// Tokens and channels that s8_split_kernel takes.
static bool takes_split(const GemmProblem& p, int num_sms) {
  const int64_t blocks = (p.M + kSplitTokens - 1) / kSplitTokens;
  if (blocks > 1 && 3 * blocks * ((p.N + 127) / 128) > num_sms) return false;
  return 48 * ((p.M + blocks - 1) / blocks) <= p.K;
}

constexpr int64_t kS8MaxK = 131071;  // 128 * 128 * K < 2^31

}  // namespace

b2g_status quantize_rows_s8(const void* src, b2g_dtype src_dtype, int64_t rows, int64_t cols, int64_t ld, int8_t* dst,
                            int64_t dst_ld, float* scales, cudaStream_t st) {
  if (rows < 0 || cols < 0) return set_error(B2G_ERR_INVALID, "b2g_quantize_s8: negative size");
  if (rows == 0) return B2G_OK;
  if ((cols > 0 && (!src || !dst)) || !scales) return set_error(B2G_ERR_INVALID, "b2g_quantize_s8: null pointer");
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

// Float activations that s8_one_kernel takes.
static bool takes_one_launch(int64_t M, int64_t K) { return M <= 8 && pow2_ceil(M) * K <= kOneMax; }

// Workspace of float activations: codes [M, round_up(K, 16)], then M scales.
size_t gemm_s8_workspace(int64_t M, int64_t K, b2g_dtype a_dtype) {
  if (a_dtype == B2G_S8 || M <= 0 || K <= 0 || M > 0x7fffffff || K > kS8MaxK) return 0;
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
  std::string why;
  if (d->a_dtype != B2G_S8) {
    // The weight's checks, before anything is launched, on activations as they will be.
    p.lda = round_up(p.K, 16);
    p.a = p.b;
    p.a_scale = b_scale;
  }
  if (!tc_gemm_supported(p, &why)) return set_error(B2G_ERR_UNSUPPORTED, "b2g_gemm_s8: " + why);
  if (p.N > 0x7fffffff - 256) return set_error(B2G_ERR_UNSUPPORTED, "b2g_gemm_s8: too many channels");
  if (d->a_dtype == B2G_S8) return takes_split(p, dev->num_sms) ? launch_split(p, false, dev, st) : tc_gemm_launch(p, st);
  if (takes_one_launch(p.M, p.K)) {
    p.a = d->a;
    p.lda = d->lda;
    if (d->a_dtype == B2G_BF16) return launch_one<__nv_bfloat16>(p, dev, st);
    if (d->a_dtype == B2G_F16) return launch_one<__half>(p, dev, st);
    return launch_one<float>(p, dev, st);
  }
  const size_t need = gemm_s8_workspace(p.M, p.K, d->a_dtype);
  void* ws = workspace;
  if (!ws && (s = workspace_get(need, &ws)) != B2G_OK) return s;
  if (workspace && (workspace_bytes < need || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
    return set_error(B2G_ERR_INVALID, "b2g_gemm_s8: the workspace is too small or not 256-byte aligned");
  int8_t* q = static_cast<int8_t*>(ws);
  float* scales = reinterpret_cast<float*>(q + round_up(p.M * p.lda, 256));
  p.a = q;
  p.a_scale = scales;
  if ((s = run_quantize(d->a, d->a_dtype, p.M, p.K, d->lda, q, p.lda, scales, st)) != B2G_OK) return s;
  p.b_early = true;
  return takes_split(p, dev->num_sms) ? launch_split(p, true, dev, st) : tc_gemm_launch(p, st);
}

}  // namespace b2g
