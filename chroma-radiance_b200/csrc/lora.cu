// lora.cu — low-rank adapters of many requests beside a shared projection.
//
//   t[m]   = x[m] A_r^T                                     R values a row, r the adapter of row m's request
//   out[m] = act(y[m] + s_r t[m] B_r^T)                     y the projection's result
//   out[m] = y[m] + gate * (s_r t[m] B_r^T)                 gated residual
//
// The rows of request b are [cu[b], cu[b+1]), its adapter is ids[b] (or b); a request without one has t = 0 and
// keeps act(y).  Offsets and adapters are read on the device and clamped: bad ones cannot make a kernel read or write
// outside its buffers.
//
// Both halves are bound by memory: down reads x (K values a row for R sums), up reads and writes y.  t is F32.
//
//   lora_down_tiles  128 rows of a request: tcgen05, x and A by TMA, K shared out over a cluster
//   lora_down_rows   few rows a request: m16n8k16 products from registers, K shared out over warps and a cluster
//   lora_up_tiles    128 rows of a request: tcgen05, y, B and out by TMA
//   lora_up_rows     few rows a request: m16n8k16 products, B through rings in shared memory
//   lora_up_any      many rows where TMA cannot take y or out: m16n8k16 products
//
// In the second product s t is the sum of two numbers of the operands' 16-bit type: bf16 keeps 2^-17 of a value, fp16, whose
// range is small, 2^-23 of its row's largest, as the row is brought to [1, 2) by a power of two.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cmath>
#include <cstdint>
#include "activations.cuh"
#include "attention_packed.cuh"

namespace b2g {

namespace {

struct LoraParams {
  const int* cu;
  const int* ids;          // [batch] or NULL: request b has adapter b
  const float* scale;      // [adapters] or NULL: 1
  const float* gate;
  int batch, rows, adapters;
  int K, N, R;
  const void *x, *a, *b;
  long long ldx, lda, as, ldb, bs;  // row and adapter strides, elements
  float* t;
  long long ldt;
  const void* y;
  void* out;
  long long ldy, ldo;
  int epilogue;
  int splits;              // CTAs of a cluster (lora_down)
  int stages;              // lora_down_tiles
  int slices;              // lora_up: parts of N
  int early;               // lora_up: all but t was ready before the launch in front of it
  int in_place;            // lora_up: out is y
  int* err;
};

// Tile `tile` of `span` rows: its first row, the end of its request's rows, its adapter (-1: none).  first < 0: no such tile.
struct LoraTile {
  int first, end, adapter;
};
// A whole warp looks, 32 requests at a time, whose offsets and adapters are loaded together: one round trip of memory.
__device__ __forceinline__ LoraTile lora_tile(const LoraParams& p, int tile, int span, int lane) {
  int base = 0;
  for (int b0 = 0; b0 < p.batch; b0 += 32) {
    const int b = b0 + lane;
    int lo = 0, end = 0, adapter = -1;
    if (b < p.batch) {
      lo = __ldg(p.cu + b);
      end = __ldg(p.cu + b + 1);
      adapter = p.ids ? __ldg(p.ids + b) : b;
    }
    lo = clampi(lo, 0, p.rows);
    end = clampi(end, lo, p.rows);
    const int n = (end - lo + span - 1) / span;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, base + sum > tile);
    if (past) {
      const int at = __ffs(past) - 1;
      LoraTile t;
      t.first = __shfl_sync(0xffffffffu, lo + (tile - base - sum + n) * span, at);
      t.end = __shfl_sync(0xffffffffu, end, at);
      t.adapter = __shfl_sync(0xffffffffu, adapter, at);
      if (t.adapter < 0 || t.adapter >= p.adapters) t.adapter = -1;
      return t;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  return {-1, 0, -1};
}

// ---------------------------------------------------------------------------- down, many rows
//
// Bound by memory (13938 rows of 3072, rank 16: 18.0 us, 4.8 TB/s).  128 rows x R sums in TMEM.  Warp 0 loads 64 values of K of x's rows and of A per stage, one thread of warp 1 issues
// the MMAs, all four warps read the sums out.  The CTAs of a cluster take a part of K each and meet in distributed
// shared memory, in rank order.  Two CTAs an SM, with 100 KB of stages each (18.4 to 23.6 us with fewer bytes in
// flight or more parts of K).
constexpr int kLdThreads = 128;
constexpr int kLdRows = 128;
constexpr int kLdMostStages = 6;
__host__ __device__ constexpr uint32_t ld_stage_bytes(int r_padded) { return (kLdRows + r_padded) * 128u; }

template <typename T>
__global__ void __launch_bounds__(kLdThreads)
    lora_down_tiles_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmA, const LoraParams p) {
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? kFmtF16 : kFmtBF16;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kLdMostStages], empty[kLdMostStages], done;
  __shared__ uint32_t tmem_slot;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.splits, rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int Rp = (p.R + 15) & ~15;
  const uint32_t stage_bytes = ld_stage_bytes(Rp);
  const uint32_t columns = Rp <= 32 ? 32 : Rp <= 64 ? 64 : 128;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&done, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmX);
    tma_prefetch_desc(&tmA);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_slot, columns);
    tmem_relinquish();
  }
  griddep_wait();
  griddep_launch_dependents();
  const LoraTile tile = lora_tile(p, static_cast<int>(blockIdx.x) / S, kLdRows, lane);
  const int rows = min(kLdRows, tile.end - tile.first);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const bool live = tile.first >= 0 && tile.adapter >= 0;  // (of the whole cluster)
  const int blocks = (p.K + 63) / 64;
  const int k0 = static_cast<int>(static_cast<long long>(blocks) * rank / S);
  const int n = live ? static_cast<int>(static_cast<long long>(blocks) * (rank + 1) / S) - k0 : 0;
  if (warp == 0 && lane == 0) {
    const uint64_t once = policy_evict_first(), shared = policy_evict_last();
    int stage = 0, used = 0;
    uint32_t parity = 0;
    for (int i = 0; i < n; ++i) {
      if (!mbar_wait_short(&empty[stage], parity ^ 1u, p.err, kErrWaitProducer)) break;
      uint8_t* at = ring + stage * stage_bytes;
      mbar_arrive_expect_tx(&full[stage], stage_bytes);
      tma_load_3d(at, &tmX, &full[stage], (k0 + i) * 64, tile.first, 0, once);
      tma_load_3d(at + kLdRows * 128, &tmA, &full[stage], (k0 + i) * 64, 0, p.as != 0 ? tile.adapter : 0, shared);
      ++used;
      if (++stage == p.stages) {
        stage = 0;
        parity ^= 1u;
      }
    }
    // This thread's copies land before the shared memory is used again or goes away.
    for (int i = min(used, p.stages); i > 0; --i) {
      if (stage-- == 0) {
        stage = p.stages - 1;
        parity ^= 1u;
      }
      mbar_wait_drain(&full[stage], parity);
    }
  } else if (warp == 1 && lane == 0) {
    const uint32_t idesc = idesc_make(kFmt, kLdRows, Rp);
    int stage = 0;
    uint32_t parity = 0;
    for (int i = 0; i < n; ++i) {
      if (!mbar_wait_short(&full[stage], parity, p.err, kErrWaitMma)) break;
      tc_fence_after();
      const uint32_t a0 = smem_u32(ring + stage * stage_bytes), b0 = a0 + kLdRows * 128;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        umma_f16(tmem, smem_desc_k_sw128(a0 + k * 32), smem_desc_k_sw128(b0 + k * 32), idesc, (i | k) != 0 ? 1u : 0u);
      umma_commit(&empty[stage]);
      if (++stage == p.stages) {
        stage = 0;
        parity ^= 1u;
      }
    }
    umma_commit(&done);
    mbar_wait_drain(&done, 0);
  }
  __syncthreads();  // all MMAs are complete, the ring is free
  tc_fence_after();
  const int row = warp * 32 + lane;
  float* sums = reinterpret_cast<float*>(ring);  // [128][Rp + 4]
  if (tile.first >= 0) {
    float* to = p.t + static_cast<long long>(tile.first + row) * p.ldt;
    for (int c = 0; c < Rp; c += 16) {
      uint32_t r[16];
      if (n > 0) {
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
        tmem_wait_ld();
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) r[i] = 0u;
      }
      if (S > 1) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<uint4*>(sums + row * (Rp + 4) + c + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
      } else if (row < rows) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          if (c + i < p.R) *reinterpret_cast<uint4*>(to + c + i) = make_uint4(r[i], r[i + 1], r[i + 2], r[i + 3]);
      }
    }
  }
  if (S > 1) {
    cluster_sync_all();  // every CTA's sums are in its shared memory
    const uint32_t from = smem_u32(sums);
    const int quads = p.R / 4;
    if (tile.first >= 0)
      for (int i = rank * kLdThreads + threadIdx.x; i < rows * quads; i += S * kLdThreads) {
        const int m = i / quads, c = (i - m * quads) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int s = 0; s < S; ++s) {
          const float4 v = ld_cluster_f4(map_to_cta(from + (m * (Rp + 4) + c) * 4, s));
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
        }
        *reinterpret_cast<float4*>(p.t + static_cast<long long>(tile.first + m) * p.ldt + c) = sum;
      }
    cluster_sync_all();  // nobody leaves while its sums are still read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, columns);
  }
}

// ---------------------------------------------------------------------------- down, few rows
//
// 16 rows of a request, of which often one is there: what has to be read is the adapter.  (Two round trips bound it: 48 single
// rows of 4096, rank 16: 5.5 us.)  A CTA takes 8 rows of A,
// its 16 warps 32 values of K in turn: lane (g, t) holds 16 bytes of row g (of x, of A) at k = 32 c + 8 t, words (0, 1) and
// (2, 3) of which are the operands of two products.  kLrAhead neighbouring chunks, 128 bytes of a row, are loaded
// together.  The warps' sums meet in shared memory in a fixed order; where there are few CTAs, those of a cluster
// share out K and meet in distributed shared memory.
constexpr int kLrWarps = 16;
constexpr int kLrAhead = 2;

template <typename T, int NT>
__global__ void __launch_bounds__(32 * kLrWarps) lora_down_rows_kernel(const LoraParams p) {
  constexpr int kCols = 8 * NT;
  __shared__ float sums[kLrWarps][16][kCols + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  griddep_wait();
  griddep_launch_dependents();
  const int S = p.splits, rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int item = static_cast<int>(blockIdx.x) / S, parts = (p.R + kCols - 1) / kCols;
  const int r0 = item % parts * kCols, width = min(kCols, p.R - r0);  // this CTA's rows of A
  const LoraTile tile = lora_tile(p, item / parts, 16, lane);
  if (tile.first < 0) return;  // (the whole cluster)
  const int rows = min(16, tile.end - tile.first);
  float acc[NT][4] = {};
  if (tile.adapter >= 0) {
    const int chunks = (p.K + 31) / 32;
    const int c0 = static_cast<int>(static_cast<long long>(chunks) * rank / S);
    const int c1 = static_cast<int>(static_cast<long long>(chunks) * (rank + 1) / S);
    const T* x = static_cast<const T*>(p.x) + static_cast<long long>(tile.first + g) * p.ldx + 8 * t;
    const T* a = static_cast<const T*>(p.a) + tile.adapter * p.as + (r0 + g) * p.lda + 8 * t;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c = c0 + warp * kLrAhead; c < c1; c += kLrWarps * kLrAhead) {
      uint4 xr[kLrAhead][2], ar[kLrAhead][NT];
#pragma unroll
      for (int u = 0; u < kLrAhead; ++u) {
        const bool in = c + u < c1 && 32 * (c + u) + 8 * t < p.K;
        const int k = 32 * (c + u);
#pragma unroll
        for (int i = 0; i < NT; ++i)
          ar[u][i] = in && 8 * i < width ? __ldg(reinterpret_cast<const uint4*>(a + 8 * i * p.lda + k)) : zero;
        xr[u][0] = in && g < rows ? __ldg(reinterpret_cast<const uint4*>(x + k)) : zero;
        xr[u][1] = in && g + 8 < rows ? __ldg(reinterpret_cast<const uint4*>(x + 8 * p.ldx + k)) : zero;
      }
#pragma unroll
      for (int u = 0; u < kLrAhead; ++u)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          mma_16816<T>(acc[i], xr[u][0].x, xr[u][1].x, xr[u][0].y, xr[u][1].y, ar[u][i].x, ar[u][i].y);
          mma_16816<T>(acc[i], xr[u][0].z, xr[u][1].z, xr[u][0].w, xr[u][1].w, ar[u][i].z, ar[u][i].w);
        }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[warp][g + 8 * (j >> 1)][8 * i + 2 * t + (j & 1)] = acc[i][j];
  __syncthreads();
  const int count = rows * width;
  float* to = p.t + r0;
  for (int i = threadIdx.x; i < count; i += 32 * kLrWarps) {
    const int m = i / width, c = i - m * width;
    float v[kLrWarps];
#pragma unroll
    for (int w = 0; w < kLrWarps; ++w) v[w] = sums[w][m][c];
#pragma unroll
    for (int o = 1; o < kLrWarps; o *= 2)
#pragma unroll
      for (int w = 0; w < kLrWarps; w += 2 * o) v[w] += v[w + o];
    const float sum = v[0];
    if (S == 1) to[static_cast<long long>(tile.first + m) * p.ldt + c] = sum;
    else sums[0][m][c] = sum;  // (read by this thread alone until here)
  }
  if (S == 1) return;
  cluster_sync_all();
  const uint32_t from = smem_u32(&sums[0][0][0]);
  for (int i = rank * 32 * kLrWarps + threadIdx.x; i < count; i += S * 32 * kLrWarps) {
    const int m = i / width, c = i - m * width;
    float v[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) v[s] = s < S ? ld_cluster_f1(map_to_cta(from + (m * (kCols + 1) + c) * 4, s)) : 0.f;
    to[static_cast<long long>(tile.first + m) * p.ldt + c] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  }
  cluster_sync_all();
}

// ---------------------------------------------------------------------------- up: values

// 8 values of type TY, as they lie in memory.
template <typename TY>
struct Eight {
  uint4 w[sizeof(TY) / 2];
  __device__ __forceinline__ void values(float (&v)[8]) const {
    if constexpr (sizeof(TY) == 4) {
      const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]);
    } else {
      const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 f;
        if constexpr (std::is_same<TY, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&v)[8]) {
    if constexpr (sizeof(TY) == 4) {
      w[0] = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      w[1] = make_uint4(__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
    } else {
      w[0] = make_uint4(pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3]), pack2<TY>(v[4], v[5]), pack2<TY>(v[6], v[7]));
    }
  }
};

// fp16: the power of two 2^e <= top < 2^(e + 1), e in [-126, 126], and its inverse.
__device__ __forceinline__ float row_unit(float top, float* down) {
  const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -126), 126);
  *down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}
// Two values as sums of two of type T: hi + lo.
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t* hi, uint32_t* lo) {
  const float ha = static_cast<float>(static_cast<T>(a)), hb = static_cast<float>(static_cast<T>(b));
  *hi = pack2<T>(a, b);
  *lo = pack2<T>(isfinite(ha) ? a - ha : 0.f, isfinite(hb) ? b - hb : 0.f);
}
// out of y and delta.
template <int EPI>
__device__ __forceinline__ float lora_out(float y, float delta, float gate) {
  if constexpr (EPI == B2G_EPI_GATED_RESIDUAL) return fmaf(gate, delta, y);
  y += delta;
  if constexpr (EPI == B2G_EPI_GELU) return gelu_tanh<true>(y);
  if constexpr (EPI == B2G_EPI_SILU) return silu_fast<true>(y);
  return y;
}
// The same of 8 values, the epilogue chosen once.
__device__ __forceinline__ void lora_out8(int epilogue, float (&v)[8], const float (&delta)[8], const float (&gate)[8]) {
  auto all = [&](auto f) {
#pragma unroll
    for (int x = 0; x < 8; ++x) v[x] = f(v[x], delta[x], gate[x]);
  };
  if (epilogue == B2G_EPI_GATED_RESIDUAL) all(lora_out<B2G_EPI_GATED_RESIDUAL>);
  else if (epilogue == B2G_EPI_GELU) all(lora_out<B2G_EPI_GELU>);
  else if (epilogue == B2G_EPI_SILU) all(lora_out<B2G_EPI_SILU>);
  else all(lora_out<B2G_EPI_NONE>);
}
// Whether a tile's rows are left as they are: no adapter, in place, and nothing else to do.
__device__ __forceinline__ bool lora_nothing(const LoraParams& p, const LoraTile& tile) {
  return tile.adapter < 0 && p.in_place && (p.epilogue == B2G_EPI_NONE || p.epilogue == B2G_EPI_GATED_RESIDUAL);
}

// ---------------------------------------------------------------------------- up, many rows
//
// Bound by memory (13938 rows of 9216, rank 16: 92.5 us, 5.6 TB/s; rank 128, whose A operand takes 64 KB of shared memory, 5 x 2000
// rows 152 us).  A CTA takes 128 rows and a part of N, 128 bytes of y's rows (kCols columns) at a time: y and the columns' rows of B
// come by TMA into a ring, one thread issues the products into one of four accumulators in TMEM, and the
// epilogue warps, a row per thread, add y in place in the ring's stage, which leaves by TMA.  Rows move in groups
// of 32: groups past the request's end are not loaded, and one that it ends in is stored row by row.
// A operand: hi and lo of s t, in one 128-byte row where they fit (R <= 32), else in tiles of 64 values of k.
constexpr int kUtThreads = 320;  // two sets of four epilogue warps, loads, products
constexpr int kUtRows = 128;
constexpr int kUtAcc = 4;
constexpr int kUtMostStages = 6;
struct UtLayout {
  int r16, atoms;            // k of one product, tiles of 64 values of it
  uint32_t a_bytes, stage;   // A operand; y and B of a stage
  uint32_t b_row;            // bytes of B's rows in shared memory
};
__host__ __device__ inline UtLayout ut_layout(int R, int cols) {
  UtLayout l;
  l.r16 = (R + 15) / 16 * 16;
  l.atoms = (R + 63) / 64;
  l.a_bytes = (l.r16 <= 32 ? 1 : 2 * l.atoms) * kUtRows * 128;
  l.b_row = l.r16 <= 16 ? 32 : l.r16 <= 32 ? 64 : 128;
  l.stage = kUtRows * 128 + l.atoms * cols * l.b_row;
  return l;
}

template <typename T, typename TY, int EPI>
__global__ void __launch_bounds__(kUtThreads)
    lora_up_tiles_kernel(const __grid_constant__ CUtensorMap tmY, const __grid_constant__ CUtensorMap tmO,
                         const __grid_constant__ CUtensorMap tmB, const LoraParams p) {
  constexpr int kCols = 128 / sizeof(TY);
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? kFmtF16 : kFmtBF16;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kUtMostStages], empty[kUtMostStages], acc_full[kUtAcc], acc_empty[kUtAcc], a_ready, drain;
  __shared__ uint32_t tmem_slot;
  __shared__ float units[kUtRows];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const UtLayout ly = ut_layout(p.R, kCols);
  uint8_t* ring = smem + ly.a_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int at_tile = static_cast<int>(blockIdx.x) / p.slices, slice = static_cast<int>(blockIdx.x) - at_tile * p.slices;
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 4);
    }
    for (int i = 0; i < kUtAcc; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    mbar_init(&a_ready, 8);
    mbar_init(&drain, 1);
    fence_mbar_init();
    tma_prefetch_desc(&tmY);
    tma_prefetch_desc(&tmO);
    tma_prefetch_desc(&tmB);
  }
  if (warp == 9) {
    tmem_alloc(&tmem_slot, kUtAcc * kCols);
    tmem_relinquish();
  }
  if (!p.early) griddep_wait();
  griddep_launch_dependents();
  const LoraTile tile = lora_tile(p, at_tile, kUtRows, lane);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  const bool has = tile.adapter >= 0;
  const int rows = tile.first < 0 || lora_nothing(p, tile) ? 0 : min(kUtRows, tile.end - tile.first);
  const int groups = (rows + 31) / 32;
  const int chunks = (p.N + kCols - 1) / kCols;
  // Its steps are slice, slice + slices, ..: CTAs side by side are at neighbouring columns.
  const int n = rows > 0 ? (chunks - slice + p.slices - 1) / p.slices : 0;
  if (warp == 8) {
    if (lane == 0) {
      const uint64_t once = policy_evict_first(), shared = policy_evict_last();
      const uint32_t bytes = groups * 4096u + (has ? ly.atoms * kCols * ly.b_row : 0u);
      int stage = 0, used = 0;
      uint32_t parity = 0;
      for (int i = 0; i < n; ++i) {
        if (!mbar_wait_short(&empty[stage], parity ^ 1u, p.err, kErrWaitProducer)) break;
        uint8_t* at = ring + stage * ly.stage;
        const int col = (slice + i * p.slices) * kCols;
        mbar_arrive_expect_tx(&full[stage], bytes);
        for (int w = 0; w < groups; ++w) tma_load_3d(at + w * 4096, &tmY, &full[stage], col, tile.first + 32 * w, 0, once);
        if (has)
          for (int a = 0; a < ly.atoms; ++a)
            tma_load_3d(at + kUtRows * 128 + a * kCols * 128, &tmB, &full[stage], a * 64, col, p.bs != 0 ? tile.adapter : 0, shared);
        ++used;
        if (++stage == p.stages) {
          stage = 0;
          parity ^= 1u;
        }
      }
      // This thread's copies land before the shared memory goes away.
      for (int i = min(used, p.stages); i > 0; --i) {
        if (stage-- == 0) {
          stage = p.stages - 1;
          parity ^= 1u;
        }
        mbar_wait_drain(&full[stage], parity);
      }
    }
  } else if (warp == 9) {
    if (lane == 0 && n > 0) {
      const uint32_t idesc = idesc_make(kFmt, kUtRows, kCols);
      const uint32_t a_hi = smem_u32(smem);
      bool ok = !has || mbar_wait_short(&a_ready, 0, p.err, kErrWaitMma);
      int stage = 0, acc = 0;
      uint32_t parity = 0, acc_parity = 0;
      for (int i = 0; i < n && ok; ++i) {
        ok = mbar_wait_short(&acc_empty[acc], acc_parity ^ 1u, p.err, kErrWaitMma) &&
             mbar_wait_short(&full[stage], parity, p.err, kErrWaitMma);
        if (!ok) break;
        tc_fence_after();
        const uint32_t b0 = smem_u32(ring + stage * ly.stage) + kUtRows * 128;
        for (int k = 0; has && k < ly.r16; k += 16) {
          const uint32_t at = (k >> 6) * (kUtRows * 128) + (k & 63) * 2;
          const uint64_t b = smem_desc_k_rows(b0 + (k >> 6) * (kCols * 128) + (k & 63) * 2, ly.b_row);
          const uint32_t lo = ly.r16 <= 32 ? (ly.r16 + k) * 2 : at + ly.atoms * (kUtRows * 128);
          umma_f16(tmem + acc * kCols, smem_desc_k_sw128(a_hi + at), b, idesc, k != 0 ? 1u : 0u);
          umma_f16(tmem + acc * kCols, smem_desc_k_sw128(a_hi + lo), b, idesc, 1u);
        }
        if (has) umma_commit(&acc_full[acc]);
        else mbar_arrive(&acc_full[acc]);
        if (++acc == kUtAcc) {
          acc = 0;
          acc_parity ^= 1u;
        }
        if (++stage == p.stages) {
          stage = 0;
          parity ^= 1u;
        }
      }
      if (!ok) {  // products already issued are complete before TMEM and the ring go away
        umma_commit(&drain);
        mbar_wait_drain(&drain, 0);
      }
    }
  } else if (n > 0) {
    if (p.early) griddep_wait();  // t
    // Warps 0-3 and 4-7 take steps in turn, each a row per thread.
    const int set = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane, live = min(max(rows - quarter * 32, 0), 32);  // rows of this warp
    if (has) {
      // 16 rows a warp: `lanes` lanes to a row, 4 values of k each.
      const float s = p.scale ? __ldg(p.scale + tile.adapter) : 1.f;
      const int lanes = ly.r16 <= 16 ? 4 : ly.r16 <= 32 ? 8 : ly.r16 <= 64 ? 16 : 32, k = lane % lanes * 4;
#pragma unroll 4
      for (int at = lane / lanes; at < 16; at += 32 / lanes) {
        const int r = warp * 16 + at;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && k < p.R) f = *reinterpret_cast<const float4*>(p.t + static_cast<long long>(tile.first + r) * p.ldt + k);
        f.x *= s; f.y *= s; f.z *= s; f.w *= s;
        float down = 1.f;  // (times s might be infinite, and a row of zeros then no number)
        if constexpr (std::is_same<T, __half>::value) {
          float top = fmaxf(fmaxf(fabsf(f.x), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w)));
          for (int o = lanes / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float unit = row_unit(top, &down);
          if (k == 0) units[r] = unit;
        }
        uint2 hi, lo;
        split2<T>(f.x * down, f.y * down, &hi.x, &lo.x);
        split2<T>(f.z * down, f.w * down, &hi.y, &lo.y);
        // 16-byte pieces of a 128-byte row are swizzled by the row.
        auto put = [&](uint32_t tile_at, int kk, uint2 v) {
          *reinterpret_cast<uint2*>(smem + tile_at + r * 128 + (((kk >> 3) ^ (r & 7)) << 4) + (kk & 4) * 2) = v;
        };
        const uint32_t atom = (k >> 6) * (kUtRows * 128);
        if (k < ly.r16) {
          put(atom, k & 63, hi);
          if (ly.r16 <= 32) put(0, ly.r16 + k, lo);
          else put(atom + ly.atoms * (kUtRows * 128), k & 63, lo);
        }
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&a_ready);
    }
    float unit = 1.f;
    int stage = set, acc = set;  // (three stages or more, and an even number of accumulators)
    uint32_t parity = 0, acc_parity = 0;
    for (int i = set; i < n; i += 2) {
      // The accumulator first: it is of this step or an earlier one, where the stage may still be on its way to the step
      // before, the other set's, with the same parity as this one behind it.
      const bool ok = mbar_wait_short(&acc_full[acc], acc_parity, p.err, kErrWaitEpilogue) &&
                      mbar_wait_short(&full[stage], parity, p.err, kErrWaitEpilogue);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      if (std::is_same<T, __half>::value && has) unit = units[row];  // (written before a_ready, on which the products waited)
      const int col = (slice + i * p.slices) * kCols;
      uint8_t* mine = ring + stage * ly.stage + row * 128;
#pragma unroll
      for (int h = 0; h < kCols / 32; ++h) {
        uint32_t d[32];
        if (has) tmem_ld_32x32b_x32(tmem + acc * kCols + (static_cast<uint32_t>(quarter * 32) << 16) + h * 32, d);
        else {
#pragma unroll
          for (int x = 0; x < 32; ++x) d[x] = 0u;
        }
        constexpr int kWords = sizeof(TY) / 2;  // 16-byte pieces of 8 columns
        auto piece = [&](int x0, int w) {
          return reinterpret_cast<uint4*>(mine + ((((h * 32 + x0) * static_cast<int>(sizeof(TY)) / 16 + w) ^ (row & 7)) << 4));
        };
        Eight<TY> ys[4];
#pragma unroll
        for (int x0 = 0; x0 < 32; x0 += 8)
#pragma unroll
          for (int w = 0; w < kWords; ++w) ys[x0 / 8].w[w] = *piece(x0, w);
        if (has) tmem_wait_ld();
        if (live > 0) {
#pragma unroll
          for (int x0 = 0; x0 < 32; x0 += 8) {
            Eight<TY>& y = ys[x0 / 8];
            float v[8];
            y.values(v);
#pragma unroll
            for (int x = 0; x < 8; ++x) {
              float delta = __uint_as_float(d[x0 + x]), gate = 0.f;
              if constexpr (std::is_same<T, __half>::value) delta *= unit;
              const int c = col + h * 32 + x0 + x;
              if (EPI == B2G_EPI_GATED_RESIDUAL && has) gate = c < p.N ? __ldg(p.gate + c) : 0.f;
              v[x] = lora_out<EPI>(v[x], delta, gate);
            }
            y.set(v);
#pragma unroll
            for (int w = 0; w < kWords; ++w) *piece(x0, w) = y.w[w];
          }
        }
      }
      tc_fence_before();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
      if (live == 32) {
        if (lane == 0) tma_store_3d(&tmO, ring + stage * ly.stage + quarter * 4096, col, tile.first + quarter * 32, 0);
      } else if (live > 0) {  // the request's last rows, 16 bytes a lane
        constexpr int kPiece = 16 / sizeof(TY);
        const int c = col + (lane & 7) * kPiece;
        for (int r = lane >> 3; r < live; r += 4) {
          const uint8_t* from = ring + stage * ly.stage + (quarter * 32 + r) * 128 + (((lane & 7) ^ (r & 7)) << 4);
          TY* to = static_cast<TY*>(p.out) + static_cast<long long>(tile.first + quarter * 32 + r) * p.ldo + c;
          if (c + kPiece <= p.N) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(from);
          else
            for (int x = 0; x < kPiece && c + x < p.N; ++x) to[x] = reinterpret_cast<const TY*>(from)[x];
        }
        __syncwarp();
      }
      if (lane == 0) {
        bulk_commit_group();
        bulk_wait_group_read<0>();  // (the other warps of this quarter's scheduler are at work meanwhile)
        mbar_arrive(&empty[stage]);
      }
      if ((acc += 2) >= kUtAcc) {
        acc -= kUtAcc;
        acc_parity ^= 1u;
      }
      if ((stage += 2) >= p.stages) {
        stage -= p.stages;
        parity ^= 1u;
      }
    }
    if (lane == 0) bulk_wait_group_all();
  }
  __syncwarp();
  if (p.early) griddep_wait();  // (this kernel's end stands for the end of the one in front of it too)
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kUtAcc * kCols);
  }
}

// ---------------------------------------------------------------------------- up, values in registers

// s t of a lane's rows g and g + 8 of 16 (k = 32 c + 8 t + ..), as hi + lo in the layout of the products' A operands.
template <typename T, int KK>
struct LoraRows {
  uint32_t hi[KK][2][4], lo[KK][2][4];  // [k / 32][row][pair of k]
  float unit[2];
  __device__ __forceinline__ void load(const LoraParams& p, const LoraTile& tile, const int (&row)[2], int t) {
    const bool has = tile.adapter >= 0;
    const float s = has ? (p.scale ? __ldg(p.scale + tile.adapter) : 1.f) : 0.f;
    float v[2][KK][8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int k = 32 * kk + 8 * t;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f), h = f;
        if (has && row[i] < tile.end && k < p.R) {
          f = *reinterpret_cast<const float4*>(p.t + row[i] * p.ldt + k);
          h = *reinterpret_cast<const float4*>(p.t + row[i] * p.ldt + k + 4);
        }
        v[i][kk][0] = f.x * s; v[i][kk][1] = f.y * s; v[i][kk][2] = f.z * s; v[i][kk][3] = f.w * s;
        v[i][kk][4] = h.x * s; v[i][kk][5] = h.y * s; v[i][kk][6] = h.z * s; v[i][kk][7] = h.w * s;
      }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float down = 1.f;
      unit[i] = 1.f;
      if constexpr (std::is_same<T, __half>::value) {
        float top = 0.f;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
#pragma unroll
          for (int x = 0; x < 8; ++x) top = fmaxf(top, fabsf(v[i][kk][x]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        unit[i] = row_unit(top, &down);
      }
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
#pragma unroll
        for (int x = 0; x < 4; ++x) split2<T>(v[i][kk][2 * x] * down, v[i][kk][2 * x + 1] * down, &hi[kk][i][x], &lo[kk][i][x]);
    }
  }
  __device__ __forceinline__ void multiply(float (&acc)[4], int kk, uint4 b) const {
    const uint32_t(&h)[2][4] = hi[kk];
    const uint32_t(&l)[2][4] = lo[kk];
    mma_16816<T>(acc, h[0][0], h[1][0], h[0][1], h[1][1], b.x, b.y);
    mma_16816<T>(acc, h[0][2], h[1][2], h[0][3], h[1][3], b.z, b.w);
    mma_16816<T>(acc, l[0][0], l[1][0], l[0][1], l[1][1], b.x, b.y);
    mma_16816<T>(acc, l[0][2], l[1][2], l[0][3], l[1][3], b.z, b.w);
  }
};
// Lane (g, t) has 8 neighbouring columns of y, two of each of four products: column 8 (c / 2) + 2 i + c % 2 of a group of 32 is
// column c of product i.  The column of B that lane ln loads for product i:
__device__ __forceinline__ int b_column(int i, int ln) { return 8 * (ln >> 3) + 2 * i + ((ln >> 2) & 1); }
// A lane's 8 values of row i of the 16, from y to out.
template <typename T, int KK>
__device__ __forceinline__ void lora_finish(const LoraParams& p, const LoraRows<T, KK>& rows, bool has, int i, const float (&acc)[4][4],
                                            const float (&gate)[8], float (&v)[8]) {
  float delta[8];
#pragma unroll
  for (int x = 0; x < 8; ++x) {  // column 2 t + e of product x / 2
    delta[x] = has ? acc[x >> 1][2 * i + (x & 1)] : 0.f;
    if constexpr (std::is_same<T, __half>::value) delta[x] *= rows.unit[i];
  }
  lora_out8(p.epilogue, v, delta, gate);
}
__device__ __forceinline__ void load_gate(const LoraParams& p, bool has, int col, int end, float (&gate)[8]) {
#pragma unroll
  for (int x = 0; x < 8; ++x) gate[x] = p.epilogue == B2G_EPI_GATED_RESIDUAL && has && col + x < end ? __ldg(p.gate + col + x) : 0.f;
}

// ---------------------------------------------------------------------------- up, few rows
//
// 16 rows of a request, of which often one is there: what has to be read is B.  (Round trips too: 48 single rows of 4096,
// rank 16: 5.9 us; 675 rows of 10240, rank 64: 18.0 us.)  A warp takes 32 columns at a time, whose
// rows of B it copies ahead into its own ring: every lane the 16-byte pieces that it will use (k as in lora_down_rows).
constexpr int kUrWarps = 4;
template <int KK>
constexpr int kUrStages = KK == 4 ? 3 : 4;
template <int KK>
constexpr size_t kUrSmem = static_cast<size_t>(kUrWarps) * kUrStages<KK> * KK * 2048;

template <typename T, typename TY, int KK, bool VEC>  // 32 KK >= R
__global__ void __launch_bounds__(32 * kUrWarps) lora_up_rows_kernel(const LoraParams p) {
  constexpr int NS = kUrStages<KK>;
  constexpr uint32_t kStage = KK * 2048;
  extern __shared__ __align__(16) uint8_t smem_up[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem_up) + warp * NS * kStage + lane * 16;
  const int at_tile = static_cast<int>(blockIdx.x / p.slices), slice = static_cast<int>(blockIdx.x - static_cast<unsigned>(at_tile) * p.slices);
  if (!p.early) griddep_wait();
  griddep_launch_dependents();
  const LoraTile tile = lora_tile(p, at_tile, 16, lane);
  if (tile.first < 0 || lora_nothing(p, tile)) {
    if (p.early) griddep_wait();  // (this kernel's end stands for the end of the one in front of it too)
    return;
  }
  const bool has = tile.adapter >= 0;
  // Groups of 32 columns: this CTA's from g0 on, its warps in turn.
  const int groups = (p.N + 31) / 32;
  const int g0 = static_cast<int>(static_cast<long long>(groups) * slice / p.slices), g1 = static_cast<int>(static_cast<long long>(groups) * (slice + 1) / p.slices);
  const T* b = static_cast<const T*>(p.b) + (has ? tile.adapter : 0) * p.bs;
  auto fetch = [&](int group, int st) {
    const uint32_t dst = ring + st * kStage;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int col = 32 * group + b_column(i, lane);
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int k = 32 * kk + 8 * t;
        const bool live = has && col < p.N && k < p.R;
        copy16(dst + (i * KK + kk) * 512, live ? b + col * p.ldb + k : p.b, live);
      }
    }
  };
  int ahead = g0 + warp;
#pragma unroll
  for (int i = 0; i < NS - 1; ++i, ahead += kUrWarps) {
    if (ahead < g1) fetch(ahead, i);
    copy_commit();
  }
  const int row[2] = {tile.first + g, tile.first + g + 8};
  const bool in[2] = {row[0] < tile.end, row[1] < tile.end};
  auto load_y = [&](int group, Eight<TY> (&y)[2]) {
    const int col = 32 * group + 8 * t;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const TY* from = static_cast<const TY*>(p.y) + row[i] * p.ldy + col;
      if constexpr (VEC) {
#pragma unroll
        for (int x = 0; x < static_cast<int>(sizeof(TY)) / 2; ++x)
          if (in[i] && col < p.N) y[i].w[x] = *(reinterpret_cast<const uint4*>(from) + x);
      } else {
        float v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = in[i] && col + x < p.N ? static_cast<float>(from[x]) : 0.f;
        y[i].set(v);
      }
    }
  };
  Eight<TY> y[2], y_next[2];
  if (g0 + warp < g1) load_y(g0 + warp, y);
  if (p.early) griddep_wait();
  LoraRows<T, KK> rows;
  rows.load(p, tile, row, t);
  int st = 0;
#pragma unroll 1
  for (int group = g0 + warp; group < g1; group += kUrWarps) {
    copy_wait<NS - 2>();
    if (ahead < g1) fetch(ahead, st == 0 ? NS - 1 : st - 1);  // (the stage used up in the last round)
    copy_commit();
    ahead += kUrWarps;
    if (group + kUrWarps < g1) load_y(group + kUrWarps, y_next);
    const uint32_t src = ring + st * kStage;
    st = st + 1 == NS ? 0 : st + 1;
    float acc[4][4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) rows.multiply(acc[i], kk, lds16(src + (i * KK + kk) * 512));
    const int col = 32 * group + 8 * t;
    float gate[8];
    load_gate(p, has, col, p.N, gate);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float v[8];
      y[i].values(v);
      lora_finish(p, rows, has, i, acc, gate, v);
      TY* to = static_cast<TY*>(p.out) + row[i] * p.ldo + col;
      if (!in[i] || col >= p.N) continue;
      if constexpr (VEC) {
        y[i].set(v);
#pragma unroll
        for (int x = 0; x < static_cast<int>(sizeof(TY)) / 2; ++x) *(reinterpret_cast<uint4*>(to) + x) = y[i].w[x];
      } else {
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (col + x < p.N) to[x] = static_cast<TY>(v[x]);
      }
    }
    y[0] = y_next[0];
    y[1] = y_next[1];
  }
  copy_wait<0>();
}

// ---------------------------------------------------------------------------- up, many rows, any alignment
//
// Where TMA cannot take y or out: 128 rows and 256 columns a CTA, 16 rows a warp, 256 bytes of each at a time.  B's part is
// laid out in shared memory as the products take it.  The products' sums pass through shared memory, so that a lane can
// take 16 aligned bytes of y's memory, wherever in a row they begin: of a row's values, those in whole pieces of 16
// bytes first, eight pieces a lane; then the 32 ends of the 16 rows, one a lane, value by value.  (Value by value
// throughout, through shared memory, 79 us for 1536 rows of 21503; so 73.)
constexpr int kLuWarps = 8;
constexpr int kLuCols = 256;
template <typename TY>
constexpr int kLuStep = 256 / sizeof(TY);                  // columns of a step
template <typename TY>
constexpr int kLuPitch = kLuStep<TY> / 8 * 9 + 1;          // words of a row of sums: 9 to 8 columns, for the banks
template <typename TY, int KK>
constexpr size_t kLuSmem = kLuCols / 8 * KK * 32 * sizeof(uint4) + static_cast<size_t>(kLuWarps) * 16 * kLuPitch<TY> * 4;

template <typename T, typename TY, int KK>  // 32 KK >= R
__global__ void __launch_bounds__(32 * kLuWarps) lora_up_any_kernel(const LoraParams p) {
  constexpr int kEsz = sizeof(TY), kPiece = 16 / kEsz, kStep = kLuStep<TY>, kPitch = kLuPitch<TY>;
  extern __shared__ __align__(16) uint8_t smem_up[];
  uint4* sb = reinterpret_cast<uint4*>(smem_up);  // [product][KK][lane]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  float* sums = reinterpret_cast<float*>(smem_up + kLuCols / 8 * KK * 32 * sizeof(uint4)) + warp * 16 * kPitch;
  const int at_tile = static_cast<int>(blockIdx.x / p.slices), slice = static_cast<int>(blockIdx.x - static_cast<unsigned>(at_tile) * p.slices);
  if (!p.early) griddep_wait();
  griddep_launch_dependents();
  const LoraTile tile = lora_tile(p, at_tile, 16 * kLuWarps, lane);
  if (tile.first < 0 || lora_nothing(p, tile)) {
    if (p.early) griddep_wait();  // (this kernel's end stands for the end of the one in front of it too)
    return;
  }
  const bool has = tile.adapter >= 0, gated = p.epilogue == B2G_EPI_GATED_RESIDUAL;
  const int n0 = slice * kLuCols, n1 = min(p.N, n0 + kLuCols);
  const int first = tile.first + 16 * warp, live = min(16, tile.end - first);
  // Of row r's columns [c0, c1): its values before the first whole piece of y's memory, and its whole pieces.
  auto head = [&](int r, int c0, int c1) {
    const uintptr_t at = reinterpret_cast<uintptr_t>(static_cast<const TY*>(p.y) + (first + r) * p.ldy + c0);
    return min(static_cast<int>((16 - (at & 15u)) & 15u) / kEsz, c1 - c0);
  };
  // (pieces of y are pieces of out where the two are as far from a boundary; else all values go one by one)
  const bool alike = ((reinterpret_cast<uintptr_t>(p.y) - reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0 && ((p.ldy - p.ldo) * kEsz) % 16 == 0;
  // Whole pieces: 16 lanes to a row, two rows at a time.
  uint4 y[8];
  auto load_y = [&](int c0) {
    const int c1 = min(c0 + kStep, n1);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int r = 2 * i + (lane >> 4), c = c0 + head(r, c0, c1) + (lane & 15) * kPiece;
      if (r < live && c + kPiece <= c1) y[i] = *reinterpret_cast<const uint4*>(static_cast<const TY*>(p.y) + (first + r) * p.ldy + c);
    }
  };
  if (alike) load_y(n0);
  const T* b = static_cast<const T*>(p.b) + (has ? tile.adapter : 0) * p.bs;
  if (has)
#pragma unroll 4
    for (int i = threadIdx.x; i < kLuCols / 8 * KK * 32; i += 32 * kLuWarps) {
      const int col = n0 + i / (32 * KK) * 8 + ((i >> 2) & 7), k = 32 * (i / 32 % KK) + 8 * (i & 3);
      sb[i] = col < n1 && k < p.R ? __ldg(reinterpret_cast<const uint4*>(b + col * p.ldb + k)) : make_uint4(0, 0, 0, 0);
    }
  const int row[2] = {first + g, first + g + 8};
  if (p.early) griddep_wait();
  LoraRows<T, KK> rows;
  rows.load(p, tile, row, t);
  __syncthreads();
  auto sum_at = [&](int r, int c) -> float& { return sums[r * kPitch + c + (c >> 3)]; };
#pragma unroll 1
  for (int c0 = n0; c0 < n1; c0 += kStep) {
    const int c1 = min(c0 + kStep, n1);
    __syncwarp();
#pragma unroll 2
    for (int j = 0; j < kStep / 8; ++j) {
      if (c0 + 8 * j >= c1) break;
      float acc[4] = {};
      if (has) {
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) rows.multiply(acc, kk, sb[(((c0 - n0) / 8 + j) * KK + kk) * 32 + lane]);
      }
      const int c = 8 * j + 2 * t;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float by = gated ? (c0 + c + e < c1 ? __ldg(p.gate + c0 + c + e) : 0.f) : 1.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float delta = acc[2 * i + e];
          if constexpr (std::is_same<T, __half>::value) delta *= rows.unit[i];
          sum_at(g + 8 * i, c + e) = gated ? (has ? by * delta : 0.f) : delta;
        }
      }
    }
    __syncwarp();
    const float ones[8] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};
    if (alike) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = 2 * i + (lane >> 4), c = c0 + head(r, c0, c1) + (lane & 15) * kPiece;
        if (r >= live || c + kPiece > c1) continue;
        float v[8] = {}, delta[8] = {};
        const uint32_t w[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
#pragma unroll
        for (int x = 0; x < kPiece; ++x) {
          if constexpr (kEsz == 4) v[x] = __uint_as_float(w[x]);
          else v[x] = static_cast<float>(reinterpret_cast<const TY*>(w)[x]);
          delta[x] = sum_at(r, c - c0 + x);
        }
        lora_out8(gated ? B2G_EPI_NONE : p.epilogue, v, delta, ones);
        uint4 o;
        if constexpr (kEsz == 4) o = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        else o = make_uint4(pack2<TY>(v[0], v[1]), pack2<TY>(v[2], v[3]), pack2<TY>(v[4], v[5]), pack2<TY>(v[6], v[7]));
        *reinterpret_cast<uint4*>(static_cast<TY*>(p.out) + (first + r) * p.ldo + c) = o;
      }
      if (c0 + kStep < n1) load_y(c0 + kStep);
    }
    // The ends, a lane each: before the first whole piece, and behind the last.  (not alike: half a row a lane)
    const int r = lane >> 1;
    if (r < live) {
      const int h = head(r, c0, c1);
      int from = c0, to = c0 + h;
      if (!alike) to = c0 + kStep / 2;
      if (lane & 1) {
        from = alike ? c0 + h + (c1 - c0 - h) / kPiece * kPiece : c0 + kStep / 2;
        to = c1;
      }
      to = min(to, c1);
      const TY* yr = static_cast<const TY*>(p.y) + (first + r) * p.ldy;
      TY* o = static_cast<TY*>(p.out) + (first + r) * p.ldo;
      for (; from < to; from += 8) {
        float v[8], delta[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          v[x] = from + x < to ? static_cast<float>(yr[from + x]) : 0.f;
          delta[x] = from + x < to ? sum_at(r, from + x - c0) : 0.f;
        }
        lora_out8(gated ? B2G_EPI_NONE : p.epilogue, v, delta, ones);
#pragma unroll
        for (int x = 0; x < 8; ++x)
          if (from + x < to) o[from + x] = static_cast<TY>(v[x]);
      }
    }
  }
}

// ---------------------------------------------------------------------------- host side

// Which form takes a call.  Few rows cost by tiles of 16 rows, each of which reads its adapter, many by tiles of 128, of
// which a request of 30 rows fills a quarter.  us, few and many, K 4096, N 8192, bf16:
//   requests x rows   1 x 700      1 x 1536     16 x 64      64 x 32      64 x 64      9 x 75 (rank 64)
//   down, rank 16     6.7, 7.9     7.2, 8.8     6.4, 8.9     7.7, 13.2    11.1, 13.5   10.4, 9.7
//   down, rank 128    16.5, 11.5   23.5, 12.5   16.0, 11.8   32.1, 17.2   58.9, 18.8
//   up, rank 16       10.5, 10.5   19.9, 13.2   15.7, 11.8   30.3, 32.3   72.6, 37.1   13.3, 15.0
//   up, rank 128      17.8, 21.5   32.4, 31.0   30.8, 41.2   76.0, 103    82.9, 131
// (64 x 64 at rank 16 is the one of these whose down is on the wrong side.)
bool few_down(int64_t rows, int64_t batch, int64_t R) {
  return rows <= (R > 32 ? 16 : 32) * batch || (rows / 16 + batch) * R <= 2600;
}
bool few_up(int64_t rows, int64_t batch, int64_t R) { return rows <= (R > 64 ? 64 : 32) * batch || rows <= 768; }

b2g_status lora_launch_cluster(const void* kern, int64_t tiles, int64_t S, int threads, size_t smem, cudaStream_t st,
                               const char* what, void** args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * S));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(S);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = S > 1 ? 2 : 1;
  b2g_status s = check_cuda(cudaLaunchKernelExC(&cfg, kern, args), what);
  if (s == B2G_OK) note_launch();
  return s;
}

template <typename T>
b2g_status run_down(const b2g_lora_desc* d, LoraParams& p, int sms, cudaStream_t st) {
  if (few_down(d->rows, d->batch, d->R) || d->adapters == 0) {  // (without adapters there is nothing to load)
    // 8 rows of A a CTA; 16 where that still leaves every SM two.
    const int64_t tiles = d->rows / 16 + d->batch;
    const int NT = p.R > 8 && tiles * ((p.R + 15) / 16) >= 2 * sms ? 2 : 1;
    const int64_t items = tiles * ((p.R + 8 * NT - 1) / (8 * NT));
    // Clusters where half of the SMs would have no CTA; a warp's part of K is at least one step of its loads.
    int64_t S = sms / items;
    const int64_t most = (d->K + 32 * kLrAhead * kLrWarps - 1) / (32 * kLrAhead * kLrWarps);
    S = S > most ? most : S;
    p.splits = static_cast<int>(S < 1 ? 1 : S > 8 ? 8 : S);
    const void* kern = NT == 2 ? reinterpret_cast<const void*>(lora_down_rows_kernel<T, 2>)
                               : reinterpret_cast<const void*>(lora_down_rows_kernel<T, 1>);
    void* args[] = {&p};
    return lora_launch_cluster(kern, items, p.splits, 32 * kLrWarps, 0, st, "lora_down_rows launch", args);
  }
  const int Rp = (p.R + 15) & ~15;
  CUtensorMap tx, ta;
  b2g_status s;
  if ((s = make_operand_map(&tx, p.x, d->dtype, p.K, p.rows, p.ldx, 1, p.ldx * p.rows, kLdRows)) != B2G_OK) return s;
  if ((s = make_operand_map(&ta, p.a, d->dtype, p.K, p.R, p.lda, p.as != 0 ? p.adapters : 1, p.as != 0 ? p.as : p.lda * p.R,
                            static_cast<uint32_t>(Rp))) != B2G_OK)  // (a stride of 0: one matrix for all)
    return s;
  const int64_t tiles = d->rows / kLdRows + d->batch;
  int64_t S = 2ll * sms / tiles;
  const int64_t most = (d->K + 255) / 256;
  S = S > most ? most : S;
  p.splits = static_cast<int>(S < 1 ? 1 : S > 8 ? 8 : S);
  p.stages = static_cast<int>(100 * 1024 / ld_stage_bytes(Rp));
  if (p.stages > kLdMostStages) p.stages = kLdMostStages;
  const size_t smem = 1024 + static_cast<size_t>(p.stages) * ld_stage_bytes(Rp);
  if (static_cast<size_t>(p.stages) * ld_stage_bytes(Rp) < sizeof(float) * kLdRows * (Rp + 4))  // (the sums take the ring's place)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_lora_down: shared memory");
  auto kern = lora_down_tiles_kernel<T>;
  s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 110 * 1024), "cudaFuncSetAttribute(lora_down)");
  if (s != B2G_OK) return s;
  void* args[] = {&tx, &ta, &p};
  return lora_launch_cluster(reinterpret_cast<const void*>(kern), tiles, p.splits, kLdThreads, smem, st, "lora_down_tiles launch", args);
}

b2g_status lora_launch_up(void (*kern)(LoraParams), const LoraParams& p, int64_t tiles, int threads, size_t smem, cudaStream_t st) {
  if (smem > 48 * 1024) {
    b2g_status s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                              "cudaFuncSetAttribute(lora_up)");
    if (s != B2G_OK) return s;
  }
  return launch_pdl(kern, dim3(static_cast<unsigned>(tiles * p.slices)), dim3(static_cast<unsigned>(threads)), smem, st, "lora_up launch", p);
}
template <typename T, typename TY, int KK>
b2g_status launch_up(LoraParams& p, bool few, bool vec, int sms, cudaStream_t st) {
  if (few) {
    // As many CTAs as run at the same time, or, with few requests, a step a warp.
    const int64_t tiles = static_cast<int64_t>(p.rows) / 16 + p.batch, steps = (p.N + 32 * kUrWarps - 1) / (32 * kUrWarps);
    const int64_t per_sm = KK == 4 ? 2 : KK == 2 ? 3 : 4, slices = per_sm * sms / tiles;
    p.slices = static_cast<int>(slices < 1 ? 1 : slices < steps ? slices : steps);
    return lora_launch_up(vec ? lora_up_rows_kernel<T, TY, KK, true> : lora_up_rows_kernel<T, TY, KK, false>, p, tiles, 32 * kUrWarps,
                          kUrSmem<KK>, st);
  }
  p.slices = (p.N + kLuCols - 1) / kLuCols;
  return lora_launch_up(lora_up_any_kernel<T, TY, KK>, p, static_cast<int64_t>(p.rows) / (16 * kLuWarps) + p.batch, 32 * kLuWarps,
                        kLuSmem<TY, KK>, st);
}
template <typename T, typename TY>
b2g_status launch_up(LoraParams& p, bool few, bool vec, int sms, cudaStream_t st) {
  if (p.R <= 32) return launch_up<T, TY, 1>(p, few, vec, sms, st);
  if (p.R <= 64) return launch_up<T, TY, 2>(p, few, vec, sms, st);
  return launch_up<T, TY, 4>(p, few, vec, sms, st);
}
template <typename T, typename TY>
b2g_status run_up(const b2g_lora_desc* d, LoraParams& p, bool vec, int sms, cudaStream_t st) {
  const bool few = few_up(d->rows, d->batch, d->R);
  if (few) return launch_up<T, TY>(p, true, vec, sms, st);
  // TMA: 16-byte aligned rows, whatever their width.
  const int64_t esz = sizeof(TY);
  const bool tma = (p.ldy * esz) % 16 == 0 && (p.ldo * esz) % 16 == 0 && p.adapters > 0 &&
                   ((reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0;
  if (!tma) return launch_up<T, TY>(p, false, false, sms, st);
  constexpr int kCols = 128 / sizeof(TY);
  CUtensorMap ty, to, tb;
  b2g_status s;
  if ((s = make_operand_map(&ty, p.y, d->y_dtype, p.N, p.rows, p.ldy, 1, p.ldy * p.rows, 32)) != B2G_OK) return s;
  if ((s = make_operand_map(&to, p.out, d->y_dtype, p.N, p.rows, p.ldo, 1, p.ldo * p.rows, 32)) != B2G_OK) return s;
  const UtLayout ly = ut_layout(p.R, kCols);
  if ((s = make_operand_map(&tb, p.b, d->dtype, p.R, p.N, p.ldb, p.bs != 0 ? p.adapters : 1, p.bs != 0 ? p.bs : p.ldb * p.N, kCols,
                            ly.b_row)) != B2G_OK)
    return s;
  // Two CTAs an SM where three stages fit beside the A operand, else one.
  const int two = static_cast<int>((111 * 1024 - ly.a_bytes) / ly.stage), one = static_cast<int>((225 * 1024 - ly.a_bytes) / ly.stage);
  p.stages = two >= 3 ? two : one;
  if (p.stages > kUtMostStages) p.stages = kUtMostStages;
  const int64_t tiles = static_cast<int64_t>(p.rows) / kUtRows + p.batch, chunks = (p.N + kCols - 1) / kCols;
  // Parts of N: rounds of CTAs times what one takes, its steps and what it costs once (in steps; little where another
  // CTA of the SM is at work meanwhile and A is small).  More of them side by side read and write longer runs of a row
  // (13938 rows of 9216, rank 16: 5 parts 108 us, 16 parts 93 us).
  const int64_t at_once = (p.stages == one ? 1ll : 2ll) * sms, once = p.stages == one ? 8 : ly.a_bytes <= 16 * 1024 ? 1 : 4;
  double best = 0;
  for (int64_t s2 = 1; s2 <= 64 && s2 <= chunks; ++s2) {
    const double cost = static_cast<double>((tiles * s2 + at_once - 1) / at_once) *
                        static_cast<double>((chunks + s2 - 1) / s2 + once) * (1.0 + 1.0 / static_cast<double>(s2));
    if (best == 0 || cost < best) {
      best = cost;
      p.slices = static_cast<int>(s2);
    }
  }
  auto kern = p.epilogue == B2G_EPI_GATED_RESIDUAL ? lora_up_tiles_kernel<T, TY, B2G_EPI_GATED_RESIDUAL>
              : p.epilogue == B2G_EPI_GELU           ? lora_up_tiles_kernel<T, TY, B2G_EPI_GELU>
              : p.epilogue == B2G_EPI_SILU           ? lora_up_tiles_kernel<T, TY, B2G_EPI_SILU>
                                                     : lora_up_tiles_kernel<T, TY, B2G_EPI_NONE>;
  if ((s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024 - 1024),
                      "cudaFuncSetAttribute(lora_up_tiles)")) != B2G_OK)
    return s;
  return launch_pdl(kern, dim3(static_cast<unsigned>(tiles * p.slices)), dim3(kUtThreads), 1024 + ly.a_bytes + p.stages * ly.stage, st,
                    "lora_up_tiles launch", ty, to, tb, p);
}

// The checks of both halves, and the parameters.
b2g_status lora_params(const b2g_lora_desc* d, const char* who, bool down, LoraParams* p) {
  auto fail = [&](b2g_status st, const char* why) { return set_error(st, std::string(who) + ": " + why); };
  if (!d) return fail(B2G_ERR_INVALID, "null descriptor");
  if (d->rows < 0 || d->K < 0 || d->N < 0 || d->R < 0 || d->adapters < 0 || d->batch < 0) return fail(B2G_ERR_INVALID, "negative size");
  if (d->dtype != B2G_BF16 && d->dtype != B2G_F16) return fail(B2G_ERR_UNSUPPORTED, "BF16 or F16 operands");
  if (d->R < 8 || d->R > 128 || d->R % 8 != 0) return fail(B2G_ERR_UNSUPPORTED, "the rank must be a multiple of 8 up to 128");
  if (d->rows > (1ll << 30) || d->K > (1ll << 30) || d->N > (1ll << 30) || d->batch > 65536 || d->adapters > (1 << 24))
    return fail(B2G_ERR_UNSUPPORTED, "size");
  if (d->rows == 0 || d->batch == 0) return B2G_OK;
  if (!d->cu || !d->t) return fail(B2G_ERR_INVALID, "null operand");
  if (d->ldt < d->R) return fail(B2G_ERR_INVALID, "a row stride is below the width");
  if (d->ldt % 4 != 0 || (reinterpret_cast<uintptr_t>(d->t) & 15u)) return fail(B2G_ERR_UNSUPPORTED, "t needs 16-byte aligned rows");
  const int64_t E = d->adapters;
  auto operand = [&](const void* at, int64_t ld, int64_t stride, int64_t rows, int64_t width) -> b2g_status {
    if (!at) return fail(B2G_ERR_INVALID, "null operand");
    if ((rows > 1 && ld < width) || (E > 1 && stride < 0)) return fail(B2G_ERR_INVALID, "a row stride is below the width");
    if (ld % 8 != 0 || stride % 8 != 0 || ld >= (1ll << 38) || stride >= (1ll << 38) || (reinterpret_cast<uintptr_t>(at) & 15u))
      return fail(B2G_ERR_UNSUPPORTED, "16-byte aligned rows required");
    return B2G_OK;
  };
  p->ldx = used(d->ldx, d->rows, (d->K + 7) / 8 * 8);
  p->lda = used(d->lda, d->R, (d->K + 7) / 8 * 8);
  p->as = used(d->a_stride, E, p->lda * d->R);
  p->ldb = used(d->ldb, d->N, d->R);
  p->bs = used(d->b_stride, E, p->ldb * d->N);
  b2g_status s;
  if (down) {
    if (d->K < 8 || d->K % 8 != 0) return fail(B2G_ERR_UNSUPPORTED, "K must be a multiple of 8");
    if ((s = operand(d->x, p->ldx, 0, d->rows, d->K)) != B2G_OK) return s;
    if (E > 0 && (s = operand(d->a, p->lda, p->as, d->R, d->K)) != B2G_OK) return s;
  } else {
    if (d->y_dtype != B2G_F32 && d->y_dtype != d->dtype) return fail(B2G_ERR_UNSUPPORTED, "y must be F32 or of the operands' type");
    if (d->epilogue != B2G_EPI_NONE && d->epilogue != B2G_EPI_GELU && d->epilogue != B2G_EPI_SILU && d->epilogue != B2G_EPI_GATED_RESIDUAL)
      return fail(B2G_ERR_UNSUPPORTED, "epilogue");
    if (d->N == 0) return B2G_OK;
    if (!d->y || !d->out) return fail(B2G_ERR_INVALID, "null operand");
    if ((reinterpret_cast<uintptr_t>(d->y) | reinterpret_cast<uintptr_t>(d->out)) & (d->y_dtype == B2G_F32 ? 3u : 1u))
      return fail(B2G_ERR_UNSUPPORTED, "y and out must be aligned to their elements");
    if (d->epilogue == B2G_EPI_GATED_RESIDUAL && !d->gate) return fail(B2G_ERR_INVALID, "gated_residual needs a gate");
    p->ldy = used(d->ldy, d->rows, d->N);
    p->ldo = used(d->ldo, d->rows, d->N);
    if (p->ldy < d->N || p->ldo < d->N) return fail(B2G_ERR_INVALID, "a row stride is below the width");
    if (p->ldy >= (1ll << 38) || p->ldo >= (1ll << 38)) return fail(B2G_ERR_UNSUPPORTED, "size");
    if (E > 0 && (s = operand(d->b, p->ldb, p->bs, d->N, d->R)) != B2G_OK) return s;
    if ((d->rows / 16 + d->batch) * ((d->N + 31) / 32) > (1ll << 31) - 1) return fail(B2G_ERR_UNSUPPORTED, "size");
  }
  p->cu = d->cu; p->ids = d->ids; p->scale = d->scale; p->gate = d->gate;
  p->batch = static_cast<int>(d->batch); p->rows = static_cast<int>(d->rows); p->adapters = static_cast<int>(E);
  p->K = static_cast<int>(d->K); p->N = static_cast<int>(d->N); p->R = static_cast<int>(d->R);
  p->x = d->x; p->a = d->a; p->b = d->b;
  p->t = d->t; p->ldt = d->ldt;
  p->y = d->y; p->out = d->out;
  p->epilogue = d->epilogue;
  return B2G_OK;
}

}  // namespace

b2g_status lora_down(const b2g_lora_desc* d, cudaStream_t st) {
  LoraParams p{};
  b2g_status s = lora_params(d, "b2g_lora_down", true, &p);
  if (s != B2G_OK || p.rows == 0) return s;
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  p.err = dev->err_word;
  if (d->dtype == B2G_F16) return run_down<__half>(d, p, dev->num_sms, st);
  return run_down<__nv_bfloat16>(d, p, dev->num_sms, st);
}

b2g_status lora_up(const b2g_lora_desc* d, cudaStream_t st, bool early) {
  LoraParams p{};
  b2g_status s = lora_params(d, "b2g_lora_up", false, &p);
  if (s != B2G_OK || p.rows == 0) return s;
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  p.err = dev->err_word;
  p.early = early ? 1 : 0;
  const int64_t esz = d->y_dtype == B2G_F32 ? 4 : 2;
  const bool vec = p.N % 8 == 0 && (p.ldy * esz) % 16 == 0 && (p.ldo * esz) % 16 == 0 &&
                   ((reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0;
  p.in_place = p.y == p.out && p.ldy == p.ldo;
  const int sms = dev->num_sms;
  if (d->dtype == B2G_F16)
    return d->y_dtype == B2G_F32 ? run_up<__half, float>(d, p, vec, sms, st) : run_up<__half, __half>(d, p, vec, sms, st);
  return d->y_dtype == B2G_F32 ? run_up<__nv_bfloat16, float>(d, p, vec, sms, st)
                               : run_up<__nv_bfloat16, __nv_bfloat16>(d, p, vec, sms, st);
}

b2g_status lora(const b2g_lora_desc* d, cudaStream_t st) {
  LoraParams p{};
  // (both halves' arguments are checked before one runs: up's here, down's at its start)
  b2g_status s = lora_params(d, "b2g_lora", false, &p);
  if (s != B2G_OK || (s = lora_down(d, st)) != B2G_OK) return s;
  return lora_up(d, st, true);
}

}  // namespace b2g
