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
//   lora_up          m16n8k16 products; t is two 16-bit numbers a value, so that its rounding is 2^-16 or less
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
  int in_place;            // lora_up: out is y
  int* err;
};

// Tile `tile` of `span` rows: its first row, the end of its request's rows, its adapter (-1: none).  first < 0: no such tile.
struct LoraTile {
  int first, end, adapter;
};
__device__ __forceinline__ LoraTile lora_tile(const LoraParams& p, int tile, int span, int lane) {
  int before = 0;
  const int b = find_seq(p.batch, tile, lane, [&](int i) {
    const int lo = clampi(__ldg(p.cu + i), 0, p.rows);
    return (clampi(__ldg(p.cu + i + 1), lo, p.rows) - lo + span - 1) / span;
  }, &before);
  if (b < 0) return {-1, 0, -1};
  const int lo = clampi(__ldg(p.cu + b), 0, p.rows);
  LoraTile t;
  t.first = lo + (tile - before) * span;
  t.end = clampi(__ldg(p.cu + b + 1), lo, p.rows);
  t.adapter = p.ids ? __ldg(p.ids + b) : b;
  if (t.adapter < 0 || t.adapter >= p.adapters) t.adapter = -1;
  return t;
}

// ---------------------------------------------------------------------------- down, many rows
//
// 128 rows x R sums in TMEM.  Warp 0 loads 64 values of K of x's rows and of A per stage, one thread of warp 1 issues
// the MMAs, all four warps read the sums out.  The CTAs of a cluster take a part of K each and meet in distributed
// shared memory, in rank order.
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
      tma_load_3d(at + kLdRows * 128, &tmA, &full[stage], (k0 + i) * 64, 0, tile.adapter, shared);
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
// 16 rows of a request, of which often one is there: what has to be read is the adapter.  A warp takes 32 values
// of K in turn: lane (g, t) holds 16 bytes of row g (of x, of A) at k = 32 c + 8 t, words (0, 1) and (2, 3) of which are
// the operands of two products.  kAhead chunks are loaded together.  The warps' sums meet in shared memory, a cluster's
// in distributed shared memory, in a fixed order.
constexpr int kLrWarps = 4;

template <typename T, int NT>  // NT * 8 >= R
__global__ void __launch_bounds__(32 * kLrWarps) lora_down_rows_kernel(const LoraParams p) {
  constexpr int kAhead = NT <= 2 ? 4 : NT == 4 ? 2 : 1;
  constexpr int kCols = 8 * NT;
  __shared__ float sums[kLrWarps][16][kCols + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  griddep_wait();
  griddep_launch_dependents();
  const int S = p.splits, rank = S > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const LoraTile tile = lora_tile(p, static_cast<int>(blockIdx.x) / S, 16, lane);
  if (tile.first < 0) return;  // (the whole cluster)
  const int rows = min(16, tile.end - tile.first);
  float acc[NT][4] = {};
  if (tile.adapter >= 0) {
    const int chunks = (p.K + 31) / 32;
    const int c0 = static_cast<int>(static_cast<long long>(chunks) * rank / S);
    const int c1 = static_cast<int>(static_cast<long long>(chunks) * (rank + 1) / S);
    const T* x = static_cast<const T*>(p.x) + static_cast<long long>(tile.first + g) * p.ldx + 8 * t;
    const T* a = static_cast<const T*>(p.a) + tile.adapter * p.as + g * p.lda + 8 * t;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (int c = c0 + warp * kAhead; c < c1; c += kLrWarps * kAhead) {
      uint4 xr[kAhead][2], ar[kAhead][NT];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const bool in = c + u < c1 && 32 * (c + u) + 8 * t < p.K;
        const int k = 32 * (c + u);
        xr[u][0] = in && g < rows ? __ldg(reinterpret_cast<const uint4*>(x + k)) : zero;
        xr[u][1] = in && g + 8 < rows ? __ldg(reinterpret_cast<const uint4*>(x + 8 * p.ldx + k)) : zero;
#pragma unroll
        for (int i = 0; i < NT; ++i)
          ar[u][i] = in && 8 * i < p.R ? __ldg(reinterpret_cast<const uint4*>(a + 8 * i * p.lda + k)) : zero;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
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
  const int count = rows * p.R;
  for (int i = threadIdx.x; i < count; i += 32 * kLrWarps) {
    const int m = i / p.R, c = i - m * p.R;
    const float sum = (sums[0][m][c] + sums[1][m][c]) + (sums[2][m][c] + sums[3][m][c]);
    if (S == 1) p.t[static_cast<long long>(tile.first + m) * p.ldt + c] = sum;
    else sums[0][m][c] = sum;  // (read by this thread alone until here)
  }
  if (S == 1) return;
  cluster_sync_all();
  const uint32_t from = smem_u32(&sums[0][0][0]);
  for (int i = rank * 32 * kLrWarps + threadIdx.x; i < count; i += S * 32 * kLrWarps) {
    const int m = i / p.R, c = i - m * p.R;
    float v[8];
#pragma unroll
    for (int s = 0; s < 8; ++s) v[s] = s < S ? ld_cluster_f1(map_to_cta(from + (m * (kCols + 1) + c) * 4, s)) : 0.f;
    p.t[static_cast<long long>(tile.first + m) * p.ldt + c] = ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
  }
  cluster_sync_all();
}

// ---------------------------------------------------------------------------- up
//
// A CTA of 8 warps, WM of them along rows (16 each) and 8 / WM along columns, takes one tile of rows and one part of N.
// A lane's 8 neighbouring columns are two columns of each of four products (column 8 (c / 2) + 2 i + c % 2 of the
// group of 32 is column c of product i), so y is read and written 16 or 32 bytes a lane; k is taken in the order in
// which a lane's 4 values are neighbours.  s t = hi + lo in the operands' type: bf16 keeps 2^-17 of a value, fp16, whose
// range is small, 2^-22 of the row's largest, as the row is brought to [1, 2) by a power of two.
constexpr int kLuThreads = 256;
constexpr int kLuCols = 256;  // columns of a part

// N values of type T at p, or where !live of any memory 0; VEC: aligned.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(float (&v)[8], const T* p, int n) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 w = *reinterpret_cast<const uint4*>(p);
      const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float2 f;
        if constexpr (std::is_same<T, __half>::value) f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        else f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? static_cast<float>(p[i]) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&v)[8], int n) {
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
      *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(p) = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = static_cast<T>(v[i]);
  }
}

template <typename T, typename TY, int KC, int WM, bool VEC>
__global__ void __launch_bounds__(kLuThreads) lora_up_kernel(const LoraParams p) {
  constexpr int WN = 8 / WM;
  constexpr bool kStaged = WM > 1;  // B passes through shared memory where several warps use it
  extern __shared__ uint2 sb[];     // [column group of 8][KC][lane]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int wm = warp % WM, wn = warp / WM;
  const int at_tile = static_cast<int>(blockIdx.x / p.slices), slice = static_cast<int>(blockIdx.x - static_cast<unsigned>(at_tile) * p.slices);
  griddep_wait();
  griddep_launch_dependents();
  const LoraTile tile = lora_tile(p, at_tile, 16 * WM, lane);
  if (tile.first < 0) return;
  const bool has = tile.adapter >= 0;
  if (!has && p.in_place && (p.epilogue == B2G_EPI_NONE || p.epilogue == B2G_EPI_GATED_RESIDUAL)) return;
  const int n0 = slice * kLuCols, n1 = min(p.N, n0 + kLuCols);
  const T* b = static_cast<const T*>(p.b) + (has ? tile.adapter : 0) * p.bs;
  // Operand B of product i of column group j: 4 values of k at 16 kc + 4 t of the column that lane g stands for.
  auto load_b = [&](int group, int kc, int ln) {
    const int gg = ln >> 2, col = n0 + (group >> 2) * 32 + 8 * (gg >> 1) + 2 * (group & 3) + (gg & 1), k = 16 * kc + 4 * (ln & 3);
    if (col >= n1 || k >= p.R) return make_uint2(0, 0);
    return __ldg(reinterpret_cast<const uint2*>(b + col * p.ldb + k));
  };
  if (kStaged && has)
    for (int i = threadIdx.x; i < kLuCols / 8 * KC * 32; i += kLuThreads) sb[i] = load_b(i / (32 * KC), i / 32 % KC, i & 31);
  const int row[2] = {tile.first + 16 * wm + g, tile.first + 16 * wm + g + 8};
  const bool in[2] = {row[0] < tile.end, row[1] < tile.end};
  uint32_t hi[KC][4], lo[KC][4];
  float unit[2] = {1.f, 1.f};
  {
    const float s = has ? (p.scale ? __ldg(p.scale + tile.adapter) : 1.f) : 0.f;
    float v[2][KC][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float top = 0.f;
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
        const int k = 16 * kc + 4 * t;
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (has && in[i] && k < p.R) f = *reinterpret_cast<const float4*>(p.t + row[i] * p.ldt + k);
        v[i][kc][0] = f.x * s;
        v[i][kc][1] = f.y * s;
        v[i][kc][2] = f.z * s;
        v[i][kc][3] = f.w * s;
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, fabsf(v[i][kc][e]));
      }
      if constexpr (std::is_same<T, __half>::value) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // 2^e <= top < 2^(e + 1), e in [-126, 126]
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127, -126), 126);
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
        unit[i] = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
#pragma unroll
        for (int kc = 0; kc < KC; ++kc)
#pragma unroll
          for (int x = 0; x < 4; ++x) v[i][kc][x] *= down;
      }
#pragma unroll
      for (int kc = 0; kc < KC; ++kc) {
        float rest[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float f = v[i][kc][x];
          const float h = static_cast<float>(static_cast<T>(f));
          rest[x] = isfinite(h) ? f - h : 0.f;
        }
        hi[kc][i] = pack2<T>(v[i][kc][0], v[i][kc][1]);
        hi[kc][2 + i] = pack2<T>(v[i][kc][2], v[i][kc][3]);
        lo[kc][i] = pack2<T>(rest[0], rest[1]);
        lo[kc][2 + i] = pack2<T>(rest[2], rest[3]);
      }
    }
  }
  if (kStaged) __syncthreads();
  for (int j = wn; j < kLuCols / 32; j += WN) {
    const int col = n0 + 32 * j + 8 * t, left = n1 - col;
    if (n0 + 32 * j >= n1) break;
    float v[2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (in[i] && left > 0) load8<TY, VEC>(v[i], static_cast<const TY*>(p.y) + row[i] * p.ldy + col, left);
    float acc[4][4] = {};
    if (has) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int kc = 0; kc < KC; ++kc) {
          const uint2 w = kStaged ? sb[((4 * j + i) * KC + kc) * 32 + lane] : load_b(4 * j + i, kc, lane);
          mma_16816<T>(acc[i], hi[kc][0], hi[kc][1], hi[kc][2], hi[kc][3], w.x, w.y);
          mma_16816<T>(acc[i], lo[kc][0], lo[kc][1], lo[kc][2], lo[kc][3], w.x, w.y);
        }
    }
    if (left <= 0) continue;
    float gate[8];
    if (p.epilogue == B2G_EPI_GATED_RESIDUAL) {
#pragma unroll
      for (int x = 0; x < 8; ++x) gate[x] = x < left ? __ldg(p.gate + col + x) : 0.f;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      if (!in[i]) continue;
#pragma unroll
      for (int x = 0; x < 8; ++x) {  // column 2 t + e of product x / 2
        float delta = acc[x >> 1][2 * i + (x & 1)];
        if constexpr (std::is_same<T, __half>::value) delta *= unit[i];
        if (p.epilogue == B2G_EPI_GATED_RESIDUAL) v[i][x] = has ? fmaf(gate[x], delta, v[i][x]) : v[i][x];
        else {
          v[i][x] += delta;
          if (p.epilogue == B2G_EPI_GELU) v[i][x] = gelu_tanh<true>(v[i][x]);
          else if (p.epilogue == B2G_EPI_SILU) v[i][x] = silu_fast<true>(v[i][x]);
        }
      }
      store8<TY, VEC>(static_cast<TY*>(p.out) + row[i] * p.ldo + col, v[i], left);
    }
  }
}

// ---------------------------------------------------------------------------- host side

// Average rows of a request up to which the few-rows forms take a call; up's middle form, of 32-row tiles.
constexpr int64_t kLoraFewRows = 16, kLoraMiddleRows = 64;

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
  if (d->rows <= kLoraFewRows * d->batch || d->adapters == 0) {  // (without adapters there is nothing to load)
    const int64_t tiles = d->rows / 16 + d->batch;
    // Two CTAs an SM; a warp's part of K is at least one step of its loads.
    int64_t S = 4ll * sms / tiles;
    const int64_t most = (d->K + 32 * kLrWarps - 1) / (32 * kLrWarps);
    S = S > most ? most : S;
    p.splits = static_cast<int>(S < 1 ? 1 : S > 8 ? 8 : S);
    const void* kern = p.R <= 8 ? reinterpret_cast<const void*>(lora_down_rows_kernel<T, 1>)
                       : p.R <= 16 ? reinterpret_cast<const void*>(lora_down_rows_kernel<T, 2>)
                       : p.R <= 32 ? reinterpret_cast<const void*>(lora_down_rows_kernel<T, 4>)
                       : p.R <= 64 ? reinterpret_cast<const void*>(lora_down_rows_kernel<T, 8>)
                                   : reinterpret_cast<const void*>(lora_down_rows_kernel<T, 16>);
    void* args[] = {&p};
    return lora_launch_cluster(kern, tiles, p.splits, 32 * kLrWarps, 0, st, "lora_down_rows launch", args);
  }
  const int Rp = (p.R + 15) & ~15;
  CUtensorMap tx, ta;
  b2g_status s;
  if ((s = make_operand_map(&tx, p.x, d->dtype, p.K, p.rows, p.ldx, 1, p.ldx * p.rows, kLdRows)) != B2G_OK) return s;
  if ((s = make_operand_map(&ta, p.a, d->dtype, p.K, p.R, p.lda, p.adapters, p.as, static_cast<uint32_t>(Rp))) != B2G_OK) return s;
  const int64_t tiles = d->rows / kLdRows + d->batch;
  int64_t S = 2ll * sms / tiles;
  const int64_t most = (d->K + 255) / 256;
  S = S > most ? most : S;
  p.splits = static_cast<int>(S < 1 ? 1 : S > 8 ? 8 : S);
  p.stages = static_cast<int>(100 * 1024 / ld_stage_bytes(Rp));
  if (p.stages > kLdMostStages) p.stages = kLdMostStages;
  const size_t smem = 1024 + static_cast<size_t>(p.stages) * ld_stage_bytes(Rp);
  auto kern = lora_down_tiles_kernel<T>;
  s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 110 * 1024), "cudaFuncSetAttribute(lora_down)");
  if (s != B2G_OK) return s;
  void* args[] = {&tx, &ta, &p};
  return lora_launch_cluster(reinterpret_cast<const void*>(kern), tiles, p.splits, kLdThreads, smem, st, "lora_down_tiles launch", args);
}

template <typename T, typename TY, int KC, int WM, bool VEC>
b2g_status launch_up(const LoraParams& p, int64_t tiles, cudaStream_t st) {
  constexpr size_t smem = WM > 1 ? kLuCols / 8 * KC * 32 * sizeof(uint2) : 0;
  auto kern = lora_up_kernel<T, TY, KC, WM, VEC>;
  if constexpr (smem > 48 * 1024) {
    b2g_status s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                              "cudaFuncSetAttribute(lora_up)");
    if (s != B2G_OK) return s;
  }
  return launch_pdl(kern, dim3(static_cast<unsigned>(tiles * p.slices)), dim3(kLuThreads), smem, st, "lora_up launch", p);
}
template <typename T, typename TY, int KC, int WM>
b2g_status launch_up(const LoraParams& p, bool vec, int64_t tiles, cudaStream_t st) {
  return vec ? launch_up<T, TY, KC, WM, true>(p, tiles, st) : launch_up<T, TY, KC, WM, false>(p, tiles, st);
}
template <typename T, typename TY, int KC>
b2g_status launch_up(const LoraParams& p, bool vec, cudaStream_t st) {
  const int64_t batch = p.batch, rows = p.rows;
  if (rows <= kLoraFewRows * batch) return launch_up<T, TY, KC, 1>(p, vec, rows / 16 + batch, st);
  if (rows <= kLoraMiddleRows * batch) return launch_up<T, TY, KC, 2>(p, vec, rows / 32 + batch, st);
  return launch_up<T, TY, KC, 8>(p, vec, rows / 128 + batch, st);
}
template <typename T, typename TY>
b2g_status launch_up(const LoraParams& p, bool vec, cudaStream_t st) {
  if (p.R <= 16) return launch_up<T, TY, 1>(p, vec, st);
  if (p.R <= 32) return launch_up<T, TY, 2>(p, vec, st);
  if (p.R <= 64) return launch_up<T, TY, 4>(p, vec, st);
  return launch_up<T, TY, 8>(p, vec, st);
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
    if (d->epilogue == B2G_EPI_GATED_RESIDUAL && !d->gate) return fail(B2G_ERR_INVALID, "gated_residual needs a gate");
    p->ldy = used(d->ldy, d->rows, d->N);
    p->ldo = used(d->ldo, d->rows, d->N);
    if (p->ldy < d->N || p->ldo < d->N) return fail(B2G_ERR_INVALID, "a row stride is below the width");
    if (p->ldy >= (1ll << 38) || p->ldo >= (1ll << 38)) return fail(B2G_ERR_UNSUPPORTED, "size");
    if (E > 0 && (s = operand(d->b, p->ldb, p->bs, d->N, d->R)) != B2G_OK) return s;
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

b2g_status lora_up(const b2g_lora_desc* d, cudaStream_t st) {
  LoraParams p{};
  b2g_status s = lora_params(d, "b2g_lora_up", false, &p);
  if (s != B2G_OK || p.rows == 0) return s;
  p.slices = (p.N + kLuCols - 1) / kLuCols;
  if ((static_cast<int64_t>(p.rows) / 16 + p.batch) * p.slices > (1ll << 31) - 1) return set_error(B2G_ERR_UNSUPPORTED, "b2g_lora_up: size");
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  const int64_t esz = d->y_dtype == B2G_F32 ? 4 : 2;
  const bool vec = p.N % 8 == 0 && (p.ldy * esz) % 16 == 0 && (p.ldo * esz) % 16 == 0 &&
                   ((reinterpret_cast<uintptr_t>(p.y) | reinterpret_cast<uintptr_t>(p.out)) & 15u) == 0;
  p.in_place = p.y == p.out && p.ldy == p.ldo;
  if (d->dtype == B2G_F16)
    return d->y_dtype == B2G_F32 ? launch_up<__half, float>(p, vec, st) : launch_up<__half, __half>(p, vec, st);
  return d->y_dtype == B2G_F32 ? launch_up<__nv_bfloat16, float>(p, vec, st) : launch_up<__nv_bfloat16, __nv_bfloat16>(p, vec, st);
}

}  // namespace b2g
