// qk_norm_rope.cu — per-head RMSNorm of queries and keys and their rotation by positions of
// several axes, in one pass.
//
//   x'    = x * rsqrt(mean(x^2) + eps) * w            per head of D values (w NULL: x' = x)
//   pair p turned by a = position[axis] * theta^(-2 j / d_axis), the j-th pair of its axis:
//           (x0, x1) -> (x0 cos a - x1 sin a, x0 sin a + x1 cos a)
//
// The axes (time, height, width, ..) take their d_axis / 2 pairs one after the other; values past
// the sum of the d_axis are normed and not turned.  A pair is two neighbouring values (as the
// reference's apply_rope_fused_bf16 has it, rope.cuh:180-221, on the table gen_pe builds, rope.cuh:84)
// or one value of each half of the turned part.  The reference takes the angles from a table made
// on the host for one image size; here a token's positions are all there is to it, so tokens of
// images of any size, of clips and of text can be packed in any order.
//
// Bound by memory: q and k are read and written once.  A head is 8 values in each of D / 8 lanes, so
// its sum of squares takes log2(D / 8) shuffles, and a lane turns the same 4 pairs of every head of a
// token: it computes their cosines and sines once per token and keeps them in registers.  Warps
// work alone, on kNrAhead steps' heads at a time: the loads of the next ones are on their way meanwhile,
// and the four chains of sums, shuffles and roots run side by side.  (One step at a time through
// copies in shared memory, the chain's latency bound the kernel: 190 us for 29120 tokens of 24 + 8 heads;
// blocks that share a table of a token's angles, behind a barrier: 150 us, and 21 us for 1536 tokens.)
// As it is: 111 us at 29120 tokens, F32 to bf16 (the copy rate), 11.5 us at 1536 of 24 + 24 heads in bf16 (half of
// it the chain of one round: positions, angles, load, sum, store), 2.5 us at 64.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cmath>
#include <cstdint>
#include "engine.cuh"
#include "ptx_sm100.cuh"

namespace b2g {

namespace {

constexpr int kNrThreads = 256;
constexpr int kNrMaxPairs = 128;  // D <= 256
constexpr int kNrMaxTokens = 8;   // tokens a block of the any-layout kernel takes at a time
constexpr int kNrAhead = 4;       // steps (of 32 / G heads) that a warp takes at a time

// Pair layouts: neighbours or halves in groups of 8 values per lane, or any (value by value).
enum { kPairsNeighbours = 0, kPairsHalves = 1, kPairsAny = 2 };

constexpr int kNrFewHeads = 8, kNrFewTokens = 1024;  // qk_norm_rope_few_kernel's heads at most, tokens at least

struct NrArgs {
  const void* x[2];   // q, k
  void* y[2];
  long long ldx[2], hsx[2], ldy[2], hsy[2];  // token and head strides in elements
  const float* norm[2];
  float eps;
  const float* pos;
  long long ldp;
  long long tokens;
  int heads, q_heads;  // q heads, then k heads
  int D, rot;          // head width, values turned
  int halves;          // kPairsAny: 1 = pairs (p, p + rot / 2)
  int block_tokens;    // kPairsAny: tokens per block and step
  int parts_log2;      // otherwise: a token's heads are shared out among 2^parts_log2 warps
  // Per pair: turns per unit of position, theta^(-2j/d) / (2 pi), as the sum of two floats.
  float2 turn[kNrMaxPairs];
  unsigned char axis[kNrMaxPairs];
};

// cos and sin of 2 pi pos (hi + lo).  The product's whole turns are taken off before anything
// is rounded away: pos * hi and its rounding error are exact as two floats.  hi + lo holds the frequency, of a radian at
// most, to 2^-45 of itself (128 products in doubles and their ratio's rounding), so that the angle is right to 2^-22 of a
// turn for |pos| up to 2^24; the error grows with the angle from there on (largest in a sample against rationals: 2^-24.6 of
// a turn up to 2^24, 2^-23.4 up to 2^26, 2^-20.1 up to 2^30).  A product in fp32 radians is off by 2^-24 of the angle,
// 0.0005 at a position of 8000.
__device__ __forceinline__ float2 cos_sin_turns(float pos, float2 turn) {
  const float p = pos * turn.x;
  const float rest = fmaf(pos, turn.y, fmaf(pos, turn.x, -p));
  const float r = (p - rintf(p)) + rest;
  float s, c;
  sincospif(2.f * r, &s, &c);
  return make_float2(c, s);
}

__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f<float>(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }

// N values at p (a multiple of N values' bytes).
template <typename T, int N>
__device__ __forceinline__ void load_n(const T* p, float* v) {
  constexpr int kWords = static_cast<int>(sizeof(T)) * N / 4;
  uint32_t w[kWords];
  if constexpr (kWords == 2) *reinterpret_cast<uint2*>(w) = *reinterpret_cast<const uint2*>(p);
  else {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(w)[i] = reinterpret_cast<const uint4*>(p)[i];
  }
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = to_f(reinterpret_cast<const T*>(w)[i]);
}
template <typename T, int N>
__device__ __forceinline__ void store_n(T* p, const float* v) {
  constexpr int kWords = static_cast<int>(sizeof(T)) * N / 4;
  uint32_t w[kWords];
#pragma unroll
  for (int i = 0; i < N; ++i) reinterpret_cast<T*>(w)[i] = from_f<T>(v[i]);
  if constexpr (kWords == 2) *reinterpret_cast<uint2*>(p) = *reinterpret_cast<uint2*>(w);
  else {
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<uint4*>(w)[i];
  }
}

// The cosines and sines of `count` tokens from t0 on, [token][pair].
__device__ __forceinline__ void fill_table(const NrArgs& a, float2* tab, long long t0, int count, int pairs) {
  for (int i = threadIdx.x; i < count * pairs; i += kNrThreads) {
    const int b = i / pairs, p = i - b * pairs;
    tab[b * kNrMaxPairs + p] = cos_sin_turns(__ldg(a.pos + (t0 + b) * a.ldp + a.axis[p]), a.turn[p]);
  }
}

// The raw bits of a lane's 8 values: four at `at`, four at `at + apart` (kHalves), or all at `at`.
template <typename T, bool kHalves>
struct Raw {
  static constexpr int kWords = 2 * static_cast<int>(sizeof(T));
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* at, int apart) {
    if constexpr (kWords == 4 && kHalves) {
      *reinterpret_cast<uint2*>(w) = __ldcs(reinterpret_cast<const uint2*>(at));
      *reinterpret_cast<uint2*>(w + 2) = __ldcs(reinterpret_cast<const uint2*>(at + apart));
    } else if constexpr (kWords == 4) {
      *reinterpret_cast<uint4*>(w) = __ldcs(reinterpret_cast<const uint4*>(at));
    } else {
      *reinterpret_cast<uint4*>(w) = __ldcs(reinterpret_cast<const uint4*>(at));
      *reinterpret_cast<uint4*>(w + 4) = __ldcs(reinterpret_cast<const uint4*>(at + (kHalves ? apart : 4)));
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = to_f(t[i]);
  }
};

// A warp's place in its work.  A token's query heads, then its key heads, are taken kNrAhead steps of
// 32 / G heads at a time (so that such a group has one set of scales and strides); the warp takes the
// groups [first, end) of a token, then those of the token `stride` further on.
struct Place {
  int token, group;
};

template <typename TI, typename TO, int G, bool kHalves>
__global__ void __launch_bounds__(kNrThreads, 2) qk_norm_rope_kernel(const __grid_constant__ NrArgs a) {
  constexpr int kHeads = 32 / G, U = kNrAhead;
  __shared__ float2 turns[kNrMaxPairs];
  __shared__ unsigned char axes[kNrMaxPairs];
  for (int p = threadIdx.x; p < a.rot / 2; p += kNrThreads) {
    turns[p] = a.turn[p];
    axes[p] = a.axis[p];
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % G, sub = lane / G;
  const bool live = l < a.D / 8;  // (D / 8 is not a power of two for every D)
  const bool turned = 8 * l < a.rot;
  const int e0 = !kHalves || !turned ? 8 * l : 4 * l, apart = !kHalves || !turned ? 4 : a.rot / 2;
  const float inv_d = 1.f / static_cast<float>(a.D);
  const int hq = live ? a.q_heads - sub : 0, hk = live ? a.heads - a.q_heads - sub : 0;  // (this lane's, counted from sub)
  const int unit = blockIdx.x * (kNrThreads / 32) + warp, parts = 1 << a.parts_log2, part = unit & (parts - 1);
  const int q_groups = (a.q_heads + kHeads * U - 1) / (kHeads * U);
  const int groups = q_groups + (a.heads - a.q_heads + kHeads * U - 1) / (kHeads * U);
  const int first = groups * part / parts, end = groups * (part + 1) / parts;
  const int stride = static_cast<int>(gridDim.x * (kNrThreads / 32)) >> a.parts_log2;  // (parts divide 8)
  const int tokens = static_cast<int>(a.tokens);
  if (first == end) return;
  auto next = [&](Place at) {
    if (++at.group == end) {
      at.group = first;
      at.token += stride;
    }
    return at;
  };
  griddep_wait();
  griddep_launch_dependents();

  Raw<TI, kHalves> raw[U];
  auto load = [&](Place at) {
    const bool k = at.group >= q_groups;
    const int h0 = (k ? at.group - q_groups : at.group) * (kHeads * U), n = at.token < tokens ? (k ? hk : hq) - h0 : 0;
    const long long hs = k ? a.hsx[1] : a.hsx[0];
    const TI* from = static_cast<const TI*>(k ? a.x[1] : a.x[0]) + at.token * (k ? a.ldx[1] : a.ldx[0]) + (h0 + sub) * hs + e0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * kHeads < n) raw[u].load(from + u * (kHeads * hs), apart);
      else raw[u].zero();
    }
  };
  Place at{unit >> a.parts_log2, first};
  load(at);
  float w[8];  // the scales of the kind of head at hand
  float2 cs[4];
  const float* norm = nullptr;
  int seen = -1;  // the token of cs
  while (at.token < tokens) {
    const bool k = at.group >= q_groups;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].values(v[u]);
    const Place then = next(at);
    load(then);
    if (at.token != seen) {
      seen = at.token;
      if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          cs[i] = cos_sin_turns(__ldg(a.pos + at.token * a.ldp + axes[4 * l + i]), turns[4 * l + i]);
      }
    }
    if (at.group == first || at.group == q_groups) {
      norm = k ? a.norm[1] : a.norm[0];
      if (norm && live) {
        load_n<float, 4>(norm + e0, w);
        load_n<float, 4>(norm + e0 + apart, w + 4);
      }
    }
    if (norm) {
      float ss[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        ss[u] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss[u] = fmaf(v[u][i], v[u][i], ss[u]);
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
        for (int u = 0; u < U; ++u) ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float inv = rsqrtf(fmaf(ss[u], inv_d, a.eps));
#pragma unroll
        for (int i = 0; i < 8; ++i) v[u][i] = v[u][i] * inv * w[i];
      }
    }
    if (turned) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int i0 = kHalves ? i : 2 * i, i1 = kHalves ? i + 4 : 2 * i + 1;
          const float x0 = v[u][i0], x1 = v[u][i1];
          v[u][i0] = fmaf(x0, cs[i].x, -(x1 * cs[i].y));
          v[u][i1] = fmaf(x0, cs[i].y, x1 * cs[i].x);
        }
    }
    const int h0 = (k ? at.group - q_groups : at.group) * (kHeads * U), n = (k ? hk : hq) - h0;
    const long long hs = k ? a.hsy[1] : a.hsy[0];
    TO* to = static_cast<TO*>(k ? a.y[1] : a.y[0]) + at.token * (k ? a.ldy[1] : a.ldy[0]) + (h0 + sub) * hs + e0;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u * kHeads >= n) break;
      if constexpr (!kHalves) store_n<TO, 8>(to + u * (kHeads * hs), v[u]);
      else {
        store_n<TO, 4>(to + u * (kHeads * hs), v[u]);
        store_n<TO, 4>(to + u * (kHeads * hs) + apart, v[u] + 4);
      }
    }
    at = then;
  }
}

// Few heads, many tokens: G lanes work on a token, so that a warp takes 32 / G neighbouring tokens at a time and
// the heads of each (query heads, then key heads) kNrAhead after one another.  A warp per token computes
// its angles in every group of lanes, which with few heads is most of the work.  us here and with a warp
// per token, tokens of q + k heads: 300 of 2 + 1: 2.8, 2.3; 1536 of 2 + 1: 2.9, 4.1; of 4 + 2: 4.1, 4.1; of 8 + 2: 6.1, 4.8;
// 29120 of 2 + 1: 16.8, 38.2; of 4 + 2: 17.6, 39.3; of 8 + 2: 42.9, 43.9; of 12 + 12 (width 96): 89.0, 76.1.
template <typename TI, typename TO, int G, bool kHalves>
__global__ void __launch_bounds__(kNrThreads, 2) qk_norm_rope_few_kernel(const __grid_constant__ NrArgs a) {
  constexpr int kTokens = 32 / G, U = kNrAhead;
  __shared__ float2 turns[kNrMaxPairs];
  __shared__ unsigned char axes[kNrMaxPairs];
  for (int p = threadIdx.x; p < a.rot / 2; p += kNrThreads) {
    turns[p] = a.turn[p];
    axes[p] = a.axis[p];
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % G, sub = lane / G;
  const bool live = l < a.D / 8;  // (D / 8 is not a power of two for every D)
  const bool turned = 8 * l < a.rot;
  const int e0 = !kHalves || !turned ? 8 * l : 4 * l, apart = !kHalves || !turned ? 4 : a.rot / 2;
  const float inv_d = 1.f / static_cast<float>(a.D);
  const int stride = static_cast<int>(gridDim.x * (kNrThreads / 32)) * kTokens, tokens = static_cast<int>(a.tokens);
  int base = static_cast<int>(blockIdx.x * (kNrThreads / 32) + warp) * kTokens;
  griddep_wait();
  griddep_launch_dependents();
  // The scales of query and key heads (1 where there are none, and the norm is left out).
  float w[2][8];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
#pragma unroll
    for (int i = 0; i < 8; ++i) w[k][i] = 1.f;
    if (a.norm[k] && live) {
      load_n<float, 4>(a.norm[k] + e0, w[k]);
      load_n<float, 4>(a.norm[k] + e0 + apart, w[k] + 4);
    }
  }
  Raw<TI, kHalves> raw[U];
  float pos[4];
  auto load = [&](int t, int h0) {
    const bool ok = live && t < tokens;
    if (h0 == 0 && turned && ok) {
#pragma unroll
      for (int i = 0; i < 4; ++i) pos[i] = __ldg(a.pos + t * a.ldp + axes[4 * l + i]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + u;
      const bool k = h >= a.q_heads;
      const TI* from = static_cast<const TI*>(k ? a.x[1] : a.x[0]) + t * (k ? a.ldx[1] : a.ldx[0]) +
                       (k ? h - a.q_heads : h) * (k ? a.hsx[1] : a.hsx[0]) + e0;
      if (ok && h < a.heads) raw[u].load(from, apart);
      else raw[u].zero();
    }
  };
  int h0 = 0;
  load(base + sub, h0);
  float2 cs[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) cs[i] = make_float2(1.f, 0.f);
  while (base < tokens) {
    const int t = base + sub, at = h0;
    float v[U][8];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u].values(v[u]);
    if (at == 0 && turned) {
#pragma unroll
      for (int i = 0; i < 4; ++i) cs[i] = cos_sin_turns(pos[i], turns[4 * l + i]);
    }
    h0 += U;
    if (h0 >= a.heads) {
      h0 = 0;
      base += stride;
    }
    load(base + sub, h0);
    float ss[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      ss[u] = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss[u] = fmaf(v[u][i], v[u][i], ss[u]);
    }
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
      for (int u = 0; u < U; ++u) ss[u] += __shfl_xor_sync(0xffffffffu, ss[u], o);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = at + u;
      if (h >= a.heads) break;
      const bool k = h >= a.q_heads;
      const float inv = (k ? a.norm[1] : a.norm[0]) ? rsqrtf(fmaf(ss[u], inv_d, a.eps)) : 1.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[u][i] = v[u][i] * inv * (k ? w[1][i] : w[0][i]);
      if (turned) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int i0 = kHalves ? i : 2 * i, i1 = kHalves ? i + 4 : 2 * i + 1;
          const float x0 = v[u][i0], x1 = v[u][i1];
          v[u][i0] = fmaf(x0, cs[i].x, -(x1 * cs[i].y));
          v[u][i1] = fmaf(x0, cs[i].y, x1 * cs[i].x);
        }
      }
      if (!live || t >= tokens) continue;
      TO* to = static_cast<TO*>(k ? a.y[1] : a.y[0]) + t * (k ? a.ldy[1] : a.ldy[0]) +
               (k ? h - a.q_heads : h) * (k ? a.hsy[1] : a.hsy[0]) + e0;
      if constexpr (!kHalves) store_n<TO, 8>(to, v[u]);
      else {
        store_n<TO, 4>(to, v[u]);
        store_n<TO, 4>(to + apart, v[u] + 4);
      }
    }
  }
}

// Any even D and rot, any alignment: a warp per head, a lane's pairs p = lane, lane + 32, ..
template <typename TI, typename TO>
__global__ void __launch_bounds__(kNrThreads) qk_norm_rope_any_kernel(const __grid_constant__ NrArgs a) {
  __shared__ float2 tab[2][kNrMaxTokens * kNrMaxPairs];
  const int pairs = a.rot / 2;
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int buf = 0;
  for (long long t0 = static_cast<long long>(blockIdx.x) * a.block_tokens; t0 < a.tokens;
       t0 += static_cast<long long>(gridDim.x) * a.block_tokens, buf ^= 1) {
    const int count = static_cast<int>(min(static_cast<long long>(a.block_tokens), a.tokens - t0));
    fill_table(a, tab[buf], t0, count, pairs);
    __syncthreads();
    for (int item = warp; item < count * a.heads; item += kNrThreads / 32) {
      const int b = item / a.heads, h = item - b * a.heads, s = h >= a.q_heads;
      const TI* x = static_cast<const TI*>(s ? a.x[1] : a.x[0]) + (t0 + b) * (s ? a.ldx[1] : a.ldx[0]) +
                    (s ? h - a.q_heads : h) * (s ? a.hsx[1] : a.hsx[0]);
      TO* y = static_cast<TO*>(s ? a.y[1] : a.y[0]) + (t0 + b) * (s ? a.ldy[1] : a.ldy[0]) +
              (s ? h - a.q_heads : h) * (s ? a.hsy[1] : a.hsy[0]);
      const float* norm = s ? a.norm[1] : a.norm[0];
      float v[kNrMaxPairs / 32][2];
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < kNrMaxPairs / 32; ++j) {
        const int p = lane + 32 * j;
        if (2 * p >= a.D) continue;
        const bool split = a.halves && p < pairs;
        v[j][0] = to_f(x[split ? p : 2 * p]);
        v[j][1] = to_f(x[split ? p + pairs : 2 * p + 1]);
        ss = fmaf(v[j][0], v[j][0], fmaf(v[j][1], v[j][1], ss));
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float inv = norm ? rsqrtf(ss / static_cast<float>(a.D) + a.eps) : 1.f;
#pragma unroll
      for (int j = 0; j < kNrMaxPairs / 32; ++j) {
        const int p = lane + 32 * j;
        if (2 * p >= a.D) continue;
        const bool split = a.halves && p < pairs;
        const int i0 = split ? p : 2 * p, i1 = split ? p + pairs : 2 * p + 1;
        float x0 = v[j][0], x1 = v[j][1];
        if (norm) {
          x0 = x0 * inv * __ldg(norm + i0);
          x1 = x1 * inv * __ldg(norm + i1);
        }
        float y0 = x0, y1 = x1;
        if (p < pairs) {
          const float2 t = tab[buf][b * kNrMaxPairs + p];
          y0 = fmaf(x0, t.x, -(x1 * t.y));
          y1 = fmaf(x0, t.y, x1 * t.x);
        }
        y[i0] = from_f<TO>(y0);
        y[i1] = from_f<TO>(y1);
      }
    }
  }
}

template <typename TI, typename TO, int G>
b2g_status launch_nr_vec(const NrArgs& a, bool halves, bool few, dim3 grid, cudaStream_t st) {
  const char* what = "qk_norm_rope launch";
  const dim3 block(kNrThreads);
  if (few)
    return halves ? launch_pdl(qk_norm_rope_few_kernel<TI, TO, G, true>, grid, block, 0, st, what, a)
                  : launch_pdl(qk_norm_rope_few_kernel<TI, TO, G, false>, grid, block, 0, st, what, a);
  return halves ? launch_pdl(qk_norm_rope_kernel<TI, TO, G, true>, grid, block, 0, st, what, a)
                : launch_pdl(qk_norm_rope_kernel<TI, TO, G, false>, grid, block, 0, st, what, a);
}

template <typename TI, typename TO>
b2g_status launch_nr(const NrArgs& a, int mode, bool few, dim3 grid, cudaStream_t st) {
  if (mode == kPairsAny)
    return launch_pdl(qk_norm_rope_any_kernel<TI, TO>, grid, dim3(kNrThreads), 0, st, "qk_norm_rope launch", a);
  const bool h = mode == kPairsHalves;
  if (a.D <= 64) return launch_nr_vec<TI, TO, 8>(a, h, few, grid, st);
  if (a.D <= 128) return launch_nr_vec<TI, TO, 16>(a, h, few, grid, st);
  return launch_nr_vec<TI, TO, 32>(a, h, few, grid, st);
}

template <typename TI>
b2g_status launch_nr_in(const NrArgs& a, int mode, bool few, b2g_dtype out, dim3 grid, cudaStream_t st) {
  if (out == B2G_BF16) return launch_nr<TI, __nv_bfloat16>(a, mode, few, grid, st);
  if (out == B2G_F16) return launch_nr<TI, __half>(a, mode, few, grid, st);
  return launch_nr<TI, float>(a, mode, few, grid, st);
}

bool is_float(b2g_dtype t) { return t == B2G_F32 || t == B2G_F16 || t == B2G_BF16; }

}  // namespace

b2g_status qk_norm_rope(const b2g_qk_norm_rope_desc* d, cudaStream_t st) {
  if (!d) return set_error(B2G_ERR_INVALID, "b2g_qk_norm_rope: null descriptor");
  if (d->tokens < 0 || d->n_head < 0 || d->n_kv_head < 0 || d->d_head < 0)
    return set_error(B2G_ERR_INVALID, "b2g_qk_norm_rope: negative size");
  if (d->tokens == 0 || d->n_head + d->n_kv_head == 0) return B2G_OK;
  if (d->d_head < 2 || d->d_head % 2 != 0 || d->d_head > 2 * kNrMaxPairs)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_qk_norm_rope: d_head must be even and at most 256");
  if (!is_float(d->dtype) || !is_float(d->out_dtype))
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_qk_norm_rope: F32, F16 or BF16 inputs and outputs");
  if (d->tokens > (1ll << 30) || d->n_head > 65536 || d->n_kv_head > 65536)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_qk_norm_rope: size");
  if ((d->n_head > 0 && (!d->q || !d->q_out)) || (d->n_kv_head > 0 && (!d->k || !d->k_out)))
    return set_error(B2G_ERR_INVALID, "b2g_qk_norm_rope: null operand");
  if (d->n_axes < 0 || d->n_axes > 4 || (d->n_axes > 0 && (!d->positions || d->ldp < d->n_axes)))
    return set_error(B2G_ERR_INVALID, "b2g_qk_norm_rope: 0 to 4 axes with positions [tokens, n_axes]");
  if (!(d->theta > 0.0) || !std::isfinite(d->theta) || !(d->eps >= 0.f) || !std::isfinite(d->eps))
    return set_error(B2G_ERR_INVALID, "b2g_qk_norm_rope: theta must be positive, eps not negative");
  NrArgs a{};
  int pairs = 0;
  for (int i = 0; i < d->n_axes; ++i) {
    const int w = d->axis_dim[i];
    if (w < 0 || w % 2 != 0 || 2 * pairs + w > d->d_head)
      return set_error(B2G_ERR_INVALID, "b2g_qk_norm_rope: axis widths must be even and fit in the head");
    // (a product per pair instead of a power: 64 roundings of 2^-53 at most)
    const double ratio = w ? std::pow(d->theta, -2.0 / w) : 1.0;
    double turns = 1.0 / 6.283185307179586476925286766559;
    for (int j = 0; j < w / 2; ++j, ++pairs, turns *= ratio) {
      a.turn[pairs].x = static_cast<float>(turns);
      a.turn[pairs].y = static_cast<float>(turns - static_cast<double>(a.turn[pairs].x));
      a.axis[pairs] = static_cast<unsigned char>(i);
    }
  }
  DeviceInfo* dev = nullptr;
  b2g_status s = device_info(&dev);
  if (s != B2G_OK) return s;
  a.x[0] = d->q; a.x[1] = d->k;
  a.y[0] = d->q_out; a.y[1] = d->k_out;
  a.ldx[0] = d->ldq; a.ldx[1] = d->ldk; a.hsx[0] = d->hsq; a.hsx[1] = d->hsk;
  a.ldy[0] = d->ldq_out; a.ldy[1] = d->ldk_out; a.hsy[0] = d->hsq_out; a.hsy[1] = d->hsk_out;
  a.norm[0] = d->q_norm; a.norm[1] = d->k_norm;
  a.eps = d->eps;
  a.pos = d->positions; a.ldp = d->ldp;
  a.tokens = d->tokens;
  a.heads = d->n_head + d->n_kv_head; a.q_heads = d->n_head;
  a.D = d->d_head; a.rot = 2 * pairs;
  a.halves = d->interleaved ? 0 : 1;
  // Groups of 8 values need widths in eighths and rows (heads) that start on a group's boundary:
  // 8 values for neighbours, 4 for halves.
  const int n = d->interleaved ? 8 : 4;
  const int64_t ib = d->dtype == B2G_F32 ? 4 : 2, ob = d->out_dtype == B2G_F32 ? 4 : 2;
  const int64_t ia = n * ib < 16 ? n * ib : 16, oa = n * ob < 16 ? n * ob : 16;
  bool vec = a.D % 8 == 0 && a.rot % 8 == 0 &&
             ((reinterpret_cast<uintptr_t>(a.norm[0]) | reinterpret_cast<uintptr_t>(a.norm[1])) & 15u) == 0;
  for (int i = 0; i < 2; ++i) {
    if ((i ? d->n_kv_head : d->n_head) == 0) continue;
    vec = vec && (reinterpret_cast<uintptr_t>(a.x[i]) % ia | (a.ldx[i] * ib) % ia | (a.hsx[i] * ib) % ia) == 0 &&
          (reinterpret_cast<uintptr_t>(a.y[i]) % oa | (a.ldy[i] * ob) % oa | (a.hsy[i] * ob) % oa) == 0;
  }
  const int mode = !vec ? kPairsAny : (d->interleaved ? kPairsNeighbours : kPairsHalves);
  const bool few = mode != kPairsAny && a.heads <= kNrFewHeads && d->tokens >= kNrFewTokens;
  int64_t blocks;
  if (mode == kPairsAny) {
    // As many tokens per block as give every warp a head, but a block for every SM.
    int64_t bt = kNrThreads / 32 / a.heads;
    if (bt > d->tokens / dev->num_sms) bt = d->tokens / dev->num_sms;
    if (bt < 1) bt = 1;
    a.block_tokens = static_cast<int>(bt);
    const int64_t most = 16ll * dev->num_sms;
    blocks = (d->tokens + bt - 1) / bt < most ? (d->tokens + bt - 1) / bt : most;
  } else {
    // A token's heads go to several warps (which all compute its angles) while that still brings
    // more warps to work, at 16 warps per SM.
    const int64_t most = 2ll * dev->num_sms, warps = most * (kNrThreads / 32);
    const int64_t per_warp = !few ? 1 : a.D <= 64 ? 4 : a.D <= 128 ? 2 : 1;
    while (!few && a.parts_log2 < 3 && (d->tokens << (a.parts_log2 + 1)) <= warps) ++a.parts_log2;
    const int64_t units = ((d->tokens << a.parts_log2) + per_warp - 1) / per_warp;
    const int64_t need = (units + kNrThreads / 32 - 1) / (kNrThreads / 32);
    // As many tokens for every warp: the rounds that `most` blocks need, shared out evenly.
    const int64_t rounds = (need + most - 1) / most;
    blocks = (need + rounds - 1) / rounds;
  }
  const dim3 grid(static_cast<unsigned>(blocks));
  if (d->dtype == B2G_BF16) return launch_nr_in<__nv_bfloat16>(a, mode, few, d->out_dtype, grid, st);
  if (d->dtype == B2G_F16) return launch_nr_in<__half>(a, mode, few, d->out_dtype, grid, st);
  return launch_nr_in<float>(a, mode, few, d->out_dtype, grid, st);
}

}  // namespace b2g
