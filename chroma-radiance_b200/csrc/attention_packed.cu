// attention_packed.cu — attention over packed sequences of different lengths.
//
//   out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, h / group]) v[j, h / group]
//
// Sequence b has the query rows [cu_q[b], cu_q[b+1]) and the keys from row cu_k[b] on, as many as
// k_lens[b] says or up to cu_k[b+1]; each attends within itself.  causal: query i of lq sees the keys
// j <= i + lk - lq (the last query sees the last key).  A row that sees no key is 0.  A group of
// n_head / n_kv_head query heads shares a key head.  The offsets are read on the device (a captured
// graph replays with other lengths), clamped to the buffers' rows: bad offsets cannot make a kernel
// read or write outside them.
//
//   packed_tiles    long queries: two 128-row tiles per CTA on the tensor cores through TMEM
//   packed_rows     few query rows per key head (single tokens): the keys are read once by
//                   blocks that share out the key axis; packed_combine joins the shares
//
// Statistics (row maximum and sum) and the output sums are fp32.  P is rounded to the operands' 16-bit
// type as the tensor cores need it; the row sum is taken before that rounding.
#include "attention_packed.cuh"

namespace b2g {

namespace {

// ---------------------------------------------------------------------------- few rows
//
// The query rows of one key head (lq tokens x group heads) in tiles of 16.  The tiles of all sequences
// lie end to end on a line, each as long as its 16-key chunks and kPrTileCost more, and the line is
// cut into equal shares; a block takes a share for one key head (the heads of a share are
// neighbouring blocks, which read whole rows of the cache together).  So blocks have equal work
// whatever the lengths; a tile that lies in several shares is joined by packed_combine.  In a block,
// 4 warps take 16 keys in turn and multiply them by m16n8k16 products:
//   S = Q K^T  lane (g, t) holds 16 bytes of key g at d = 32 c + 8 t: words (0, 1) and (2, 3) are
//              the B operands of two products; Q is held in the same (permuted) order of d.
//   O += P V   lane (g, t) holds 16 bytes of keys 2t, 2t+1, 2t+8, 2t+9 at d = 64 c + 8 g; value i of
//              these pairs up to the B operand of product i, whose column g is d = 64 c + 8 g + i.
// Bound by memory, so what counts is bytes in flight: every lane copies exactly the 16-byte pieces
// that it will use into its own slots of shared memory (cp.async, kPrStages chunks ahead; nothing
// is shared between lanes, so there is nothing to wait for but a lane's own copies).  Loaded into
// registers one chunk ahead instead, the same loop ran at 2.8 TB/s.  The warps' sums meet in
// shared memory.  48 single queries, 32 and 8 heads, caches of 1 to 8191 keys: 36.4 us with the joining
// launch, 3.7 TB/s of the cache; 8 us of that are the two launches' first and last round trips.
constexpr int kPrWarps = 4;
constexpr int kPrRows = 16;
constexpr int kPrKeys = 16;  // keys of a chunk
template <int D>
constexpr int kPrPieces = D / 8;  // 16-byte pieces of K and V that a lane has of a chunk
template <int D>
constexpr int kPrStages = D == 128 ? 3 : 6;  // 24 KB per warp
template <int D>
constexpr uint32_t kPrSmem = kPrWarps * kPrStages<D> * kPrPieces<D> * 512u;
constexpr int kPrBlocksPerSm = 2;

constexpr int kPrTileCost = 6;   // what a tile costs beside its chunks, in chunks
constexpr int kPrMinShare = 16;  // a share is at least so long

__device__ __forceinline__ int rows_tiles(const PkParams& p, const Seq& s) {
  return static_cast<int>((static_cast<long long>(s.lq) * p.group + kPrRows - 1) / kPrRows);
}
__device__ __forceinline__ int tile_length(const Seq& s) { return (s.lk + kPrKeys - 1) / kPrKeys + kPrTileCost; }
__device__ __forceinline__ long long seq_length(const PkParams& p, int b) {
  const Seq s = load_seq(p, b);
  return static_cast<long long>(rows_tiles(p, s)) * tile_length(s);
}
// The line's length and the number of shares.  Share i is [total * i / shares, total * (i + 1) / shares).
struct Line {
  long long total;
  int shares;
};
__device__ __forceinline__ Line the_line(const PkParams& p, int lane) {
  long long sum = 0;
  for (int b = lane; b < p.batch; b += 32) sum += seq_length(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const long long most = (sum + kPrMinShare - 1) / kPrMinShare;
  return {sum, static_cast<int>(min(static_cast<long long>(p.shares), most))};
}
// A partial result's slot: of share i and one key head, the part of a tile that begins in the share
// (1) or before it (0).
__device__ __forceinline__ int part_slot(const PkParams& p, int share, int begins, int head) {
  return (2 * share + begins) * p.hk + head;
}

template <typename T, int D>
__global__ void __launch_bounds__(32 * kPrWarps, kPrBlocksPerSm) packed_rows_kernel(const PkParams p) {
  constexpr int KC = D / 32;  // 16-byte pieces of a lane's key
  constexpr int VC = D / 64;  // 16-byte pieces of each of a lane's four value rows
  constexpr int NS = kPrStages<D>;
  constexpr uint32_t kStage = kPrPieces<D> * 512u;
  extern __shared__ __align__(16) uint8_t smem_rows[];
  __shared__ float2 sml[kPrWarps][kPrRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem_rows) + warp * NS * kStage + lane * 16;
  // The warps' sums [kPrRows][D + 4], each over its own ring.
  auto so = [&](int w) { return reinterpret_cast<float*>(smem_rows + w * NS * kStage); };
  static_assert(kPrRows * (D + 4) * 4 <= NS * kStage, "sums fit a ring");
  griddep_wait();
  griddep_launch_dependents();
  const Line line = the_line(p, lane);
  for (int block = blockIdx.x; block < line.shares * p.hk; block += gridDim.x) {
   const int share = block / p.hk, head = block - share * p.hk;
   const long long end = line.total * (share + 1) / line.shares;
   long long before = 0;
   int b = 0;
   for (long long at = line.total * share / line.shares; at < end;) {
    b = find_seq(p.batch, at, lane, [&](int i) { return seq_length(p, i); }, &before, b);
    if (b < 0) break;
    const Seq s = load_seq(p, b);
    const int length = tile_length(s), tile = static_cast<int>((at - before) / length);
    const long long tile_at = before + static_cast<long long>(tile) * length;
    const int from = static_cast<int>(at - tile_at);
    const int to = static_cast<int>(min(static_cast<long long>(length), end - tile_at));
    at = tile_at + to;
    const int rows = s.lq * p.group, row0 = tile * kPrRows;
    // The chunks [c0, c1) of this part, cut at the last key that any row of the tile sees.
    const int last_token = min(row0 + kPrRows, rows) - 1;
    const int tile_sees = p.causal ? clampi(last_token / p.group + 1 + s.lk - s.lq, 0, s.lk) : s.lk;
    const int c0 = max(0, from - kPrTileCost);
    const int c1 = min(max(0, to - kPrTileCost), (tile_sees + kPrKeys - 1) / kPrKeys);
    const T* kbase = static_cast<const T*>(p.k) + s.k0 * p.ldk + head * p.hsk + 8 * t;
    const T* vbase = static_cast<const T*>(p.v) + s.k0 * p.ldv + head * p.hsv + 8 * g;
    // Copies chunk c into stage st: keys that no row of the tile sees are zeros.
    auto fetch = [&](int c, int st) {
      const uint32_t dst = ring + st * kStage;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int key = c * kPrKeys + nt * 8 + g;
        const bool live = key < tile_sees;
        const T* src = live ? kbase + key * p.ldk : kbase;
#pragma unroll
        for (int i = 0; i < KC; ++i) copy16(dst + (nt * KC + i) * 512, src + 32 * i, live);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = c * kPrKeys + 2 * t + (i & 1) + 8 * (i >> 1);
        const bool live = key < tile_sees;
        const T* src = live ? vbase + key * p.ldv : vbase;
#pragma unroll
        for (int k = 0; k < VC; ++k) copy16(dst + (2 * KC + i * VC + k) * 512, src + 64 * k, live);
      }
    };
    int ahead = c0 + warp;
#pragma unroll
    for (int i = 0; i < NS - 1; ++i, ahead += kPrWarps) {
      if (ahead < c1) fetch(ahead, i);
      copy_commit();
    }

    // Q: rows g and g + 8 of the tile (row r is token r / group, head r % group of the group).
    uint4 q[2][KC];
    int sees[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = min(row0 + g + 8 * i, rows - 1);
      const int token = r / p.group, h = r - token * p.group;
      sees[i] = p.causal ? min(s.lk, token + 1 + s.lk - s.lq) : s.lk;
      const T* src = static_cast<const T*>(p.q) + (s.q0 + token) * p.ldq +
                     (static_cast<long long>(head) * p.group + h) * p.hsq + 8 * t;
#pragma unroll
      for (int c = 0; c < KC; ++c) q[i][c] = __ldg(reinterpret_cast<const uint4*>(src + 32 * c));
    }

    float o[D / 8][4];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int st = 0;
    for (int c = c0 + warp; c < c1; c += kPrWarps) {
      copy_wait<NS - 2>();
      if (ahead < c1) fetch(ahead, st == 0 ? NS - 1 : st - 1);  // (the stage used up in the last round)
      copy_commit();
      ahead += kPrWarps;
      const uint32_t src = ring + st * kStage;
      st = st + 1 == NS ? 0 : st + 1;
      float sc[2][4] = {};
#pragma unroll
      for (int i = 0; i < KC; ++i)
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const uint4 kr = lds16(src + (nt * KC + i) * 512);
          mma_16816<T>(sc[nt], q[0][i].x, q[1][i].x, q[0][i].y, q[1][i].y, kr.x, kr.y);
          mma_16816<T>(sc[nt], q[0][i].z, q[1][i].z, q[0][i].w, q[1][i].w, kr.z, kr.w);
        }
      // Scores in log2 units; sc[nt][2i + e] is row g + 8i, key 16c + 8nt + 2t + e.
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = c * kPrKeys + nt * 8 + 2 * t + (j & 1);
          sc[nt][j] = key < sees[j >> 1] ? sc[nt][j] * p.scale_log2 : -INFINITY;
          mx[j >> 1] = fmaxf(mx[j >> 1], sc[nt][j]);
        }
      float alpha[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 1));
        mx[i] = fmaxf(mx[i], __shfl_xor_sync(0xffffffffu, mx[i], 2));
        const float top = fmaxf(m[i], mx[i]);
        alpha[i] = top == m[i] ? 1.f : fast_exp2(m[i] - top);
        m[i] = top;
        l[i] *= alpha[i];
      }
      if (__any_sync(0xffffffffu, alpha[0] != 1.f || alpha[1] != 1.f)) {
#pragma unroll
        for (int i = 0; i < D / 8; ++i) {
          o[i][0] *= alpha[0];
          o[i][1] *= alpha[0];
          o[i][2] *= alpha[1];
          o[i][3] *= alpha[1];
        }
      }
      uint32_t pa[4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float shift = m[i] == -INFINITY ? 0.f : m[i];
          const float e0 = fast_exp2(sc[nt][2 * i] - shift), e1 = fast_exp2(sc[nt][2 * i + 1] - shift);
          l[i] += e0 + e1;
          pa[2 * nt + i] = pack2<T>(e0, e1);
        }
#pragma unroll
      for (int k = 0; k < VC; ++k) {
        uint4 vr[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) vr[i] = lds16(src + (2 * KC + i * VC + k) * 512);
        const uint32_t v0[4] = {vr[0].x, vr[0].y, vr[0].z, vr[0].w}, v1[4] = {vr[1].x, vr[1].y, vr[1].z, vr[1].w};
        const uint32_t v2[4] = {vr[2].x, vr[2].y, vr[2].z, vr[2].w}, v3[4] = {vr[3].x, vr[3].y, vr[3].z, vr[3].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t pick = i & 1 ? 0x7632u : 0x5410u;
          mma_16816<T>(o[8 * k + i], pa[0], pa[1], pa[2], pa[3], __byte_perm(v0[i >> 1], v1[i >> 1], pick),
                       __byte_perm(v2[i >> 1], v3[i >> 1], pick));
        }
      }
    }
    copy_wait<0>();
    // The warps' statistics and sums.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      if (t == 0) sml[warp][g + 8 * i] = make_float2(m[i], l[i]);
    }
    __syncwarp();  // (the ring's slots belong to lanes, the sums do not)
#pragma unroll
    for (int k = 0; k < VC; ++k)
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int i = 0; i < 8; i += 4) {  // column 2t + e of product i is d = 64 k + 8 (2t + e) + i
          float* dst = so(warp) + g * (D + 4) + 64 * k + 16 * t + 8 * e + i;
          const float(*x)[4] = o + 8 * k + i;
          *reinterpret_cast<float4*>(dst) = make_float4(x[0][e], x[1][e], x[2][e], x[3][e]);
          *reinterpret_cast<float4*>(dst + 8 * (D + 4)) = make_float4(x[0][2 + e], x[1][2 + e], x[2][2 + e], x[3][2 + e]);
        }
    __syncthreads();
    // Groups of 4 values of the tile's rows.
    const int live_rows = min(kPrRows, rows - row0);
    for (int at = threadIdx.x; at < live_rows * (D / 4); at += 32 * kPrWarps) {
      const int r = at / (D / 4), d = (at - r * (D / 4)) * 4;
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kPrWarps; ++w) top = fmaxf(top, sml[w][r].x);
      float sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kPrWarps; ++w) {
        const float2 ml = sml[w][r];
        const float4 x = *reinterpret_cast<const float4*>(so(w) + r * (D + 4) + d);
        // (a warp without a key has the sums 0; a NaN maximum does not occur, a NaN sum stays one)
        const float wgt = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - top);
        sum += wgt * ml.y;
        acc.x += wgt * x.x;
        acc.y += wgt * x.y;
        acc.z += wgt * x.z;
        acc.w += wgt * x.w;
      }
      if (to - from < length) {
        const long long slot = static_cast<long long>(part_slot(p, share, from == 0, head)) * kPrRows + r;
        *reinterpret_cast<float4*>(p.part_o + slot * D + d) = acc;
        if (d == 0) p.part_ml[slot] = make_float2(top, sum);
      } else {
        const int token = (row0 + r) / p.group, h = (row0 + r) - token * p.group;
        const float inv = sum != 0.f ? 1.f / sum : 0.f;
        T* dst = static_cast<T*>(p.out) + (s.q0 + token) * p.ldo + (static_cast<long long>(head) * p.group + h) * p.hso + d;
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
      }
    }
    __syncthreads();  // the shared buffers are used again for the next tile
   }
  }
}

// Joins the parts of every tile that lies in several shares: with part i holding (m_i, l_i) and O_i,
// out = sum 2^(m_i - M) O_i / sum 2^(m_i - M) l_i.  A block looks at the cut between two shares, for
// one key head, and takes the tile there if it is the tile's first cut; a thread joins 4 values of a
// row, kPcAhead parts' loads at a time.  All but the parts is read before the wait for packed_rows:
// that kernel lets this one start after its own wait, when everything before it is complete.
constexpr int kPcAhead = 8;
template <typename T, int D>
__global__ void __launch_bounds__(128) packed_combine_kernel(const PkParams p) {
  const int lane = threadIdx.x & 31;
  const Line line = the_line(p, lane);
  bool waited = false;
  for (int block = blockIdx.x; block < (line.shares - 1) * p.hk; block += gridDim.x) {
    const int cut = block / p.hk + 1, head = block - (cut - 1) * p.hk;
    const long long at = line.total * cut / line.shares;
    long long before = 0;
    const int b = find_seq(p.batch, at, lane, [&](int i) { return seq_length(p, i); }, &before);
    if (b < 0) break;
    const Seq s = load_seq(p, b);
    const int length = tile_length(s), tile = static_cast<int>((at - before) / length);
    const long long tile_at = before + static_cast<long long>(tile) * length;
    // (a share may be longer than the tile: then the cut before this one is outside it)
    if (tile_at == at || line.total * (cut - 1) / line.shares > tile_at) continue;
    int parts = 2;  // the part before the cut and those after it
    while (cut + parts - 1 < line.shares && line.total * (cut + parts - 1) / line.shares < tile_at + length) ++parts;
    const int rows = s.lq * p.group, row0 = tile * kPrRows, live_rows = min(kPrRows, rows - row0);
    const long long first = static_cast<long long>(part_slot(p, cut - 1, 1, head)) * kPrRows;
    const long long second = static_cast<long long>(part_slot(p, cut, 0, head)) * kPrRows;
    const long long step = 2ll * p.hk * kPrRows;
    if (!waited) griddep_wait();
    waited = true;
    for (int at4 = threadIdx.x; at4 < live_rows * (D / 4); at4 += 128) {
      const int r = at4 / (D / 4), d = (at4 - r * (D / 4)) * 4;
      float top = -INFINITY, sum = 0.f;
      float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int i0 = 0; i0 < parts; i0 += kPcAhead) {
        float2 ml[kPcAhead];
        float4 x[kPcAhead];
#pragma unroll
        for (int i = 0; i < kPcAhead; ++i) {
          const bool in = i0 + i < parts;
          const long long slot = (i0 + i == 0 ? first : second + (i0 + i - 1) * step) + r;
          ml[i] = in ? __ldcg(p.part_ml + slot) : make_float2(-INFINITY, 0.f);
          x[i] = in ? __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float next = top;
#pragma unroll
        for (int i = 0; i < kPcAhead; ++i) next = fmaxf(next, ml[i].x);
        const float alpha = top == next ? 1.f : fast_exp2(top - next);
        top = next;
        sum *= alpha;
        acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
#pragma unroll
        for (int i = 0; i < kPcAhead; ++i) {
          const float wgt = ml[i].x == -INFINITY ? (ml[i].y == 0.f ? 0.f : 1.f) : fast_exp2(ml[i].x - top);
          sum += wgt * ml[i].y;
          acc.x += wgt * x[i].x;
          acc.y += wgt * x[i].y;
          acc.z += wgt * x[i].z;
          acc.w += wgt * x[i].w;
        }
      }
      const int token = (row0 + r) / p.group, h = (row0 + r) - token * p.group;
      const float inv = sum != 0.f ? 1.f / sum : 0.f;
      T* dst = static_cast<T*>(p.out) + (s.q0 + token) * p.ldo + (static_cast<long long>(head) * p.group + h) * p.hso + d;
      *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
    }
  }
  if (!waited) griddep_wait();  // (this kernel's end stands for packed_rows' end too)
}

// ---------------------------------------------------------------------------- host side

// Average queries per sequence up to which packed_rows takes a call.
constexpr int64_t kPrQueries = 16;
// What a call runs, from its sizes alone (the offsets are on the device).
struct PkPlan {
  bool rows = false;       // packed_rows (+ packed_combine), else packed_tiles
  int shares = 0;
  size_t o_bytes = 0, bytes = 0;
};

PkPlan plan(const b2g_attention_packed_desc* d, int sms) {
  PkPlan r;
  const int64_t group = d->n_head / d->n_kv_head;
  // Up to kPrQueries queries per sequence on average.  Measured on 64 sequences of their own 8 / 16 / 30
  // tokens, 32 and 8 heads: packed_rows 24 / 35 / 66 us, packed_tiles 39 us; with 24 and 24 heads of
  // 64 values, 128 sequences of 24: 66 and 54 us.  Long keys favour packed_rows, which shares them out.
  r.rows = d->total_q <= kPrQueries * d->batch || d->total_k == 0;
  if (!r.rows) return r;
  // A block per share and key head, as many as run at the same time; no more shares than the
  // longest line possible has pieces of kPrMinShare.
  const int64_t tiles = d->total_q * group / kPrRows + d->batch;
  const int64_t blocks = static_cast<int64_t>(kPrBlocksPerSm) * sms;
  int64_t shares = blocks / d->n_kv_head;
  const int64_t per_tile = (d->total_k + kPrKeys - 1) / kPrKeys + kPrTileCost;
  const int64_t line = tiles <= (1ll << 31) / per_tile ? tiles * per_tile : (1ll << 31);
  if (shares > (line + kPrMinShare - 1) / kPrMinShare) shares = (line + kPrMinShare - 1) / kPrMinShare;
  if (shares < 1) shares = 1;
  r.shares = static_cast<int>(shares);
  if (shares == 1) return r;
  const int64_t slots = 2 * shares * d->n_kv_head;
  r.o_bytes = static_cast<size_t>(round_up(slots * kPrRows * d->d_head * 4, 256));
  r.bytes = r.o_bytes + static_cast<size_t>(slots) * kPrRows * sizeof(float2);
  return r;
}

template <typename T, int D>
b2g_status launch_rows(const PkParams& p, int sms, cudaStream_t st) {
  const int64_t most = static_cast<int64_t>(kPrBlocksPerSm) * sms, blocks = static_cast<int64_t>(p.shares) * p.hk;
  auto kern = packed_rows_kernel<T, D>;
  b2g_status s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kPrSmem<D>),
                            "cudaFuncSetAttribute(packed_rows)");
  if (s != B2G_OK) return s;
  s = launch_pdl(kern, dim3(static_cast<unsigned>(blocks < most ? blocks : most)), dim3(32 * kPrWarps), kPrSmem<D>, st,
                 "packed_rows launch", p);
  if (s != B2G_OK || p.shares == 1) return s;
  return launch_pdl(packed_combine_kernel<T, D>, dim3(static_cast<unsigned>(blocks - p.hk < most ? blocks - p.hk : most)),
                    dim3(128), 0, st, "packed_combine launch", p);
}

template <typename T, int D>
b2g_status run_packed(const b2g_attention_packed_desc* d, PkParams p, void* ws, const PkPlan& pl, int sms,
                      cudaStream_t st) {
  if (pl.rows) {
    p.shares = pl.shares;
    p.part_o = static_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + pl.o_bytes);
    return launch_rows<T, D>(p, sms, st);
  }
  CUtensorMap tq, tk, tv;
  b2g_status s;
  const b2g_dtype dt = d->dtype;
  if ((s = make_operand_map(&tq, p.q, dt, D, p.total_q, p.ldq, p.hq, p.hsq, kPtRows)) != B2G_OK) return s;
  if ((s = make_operand_map(&tk, p.k, dt, D, p.total_k, p.ldk, p.hk, p.hsk, kPtKeys)) != B2G_OK) return s;
  if ((s = make_operand_map(&tv, p.v, dt, D, p.total_k, p.ldv, p.hk, p.hsv, kPtKeys)) != B2G_OK) return s;
  p.item_heads = 2;
  // Where every tile finds an SM of its own, two tiles in turn only slow each other: 8 heads of 128, 2048 tokens: 37.6
  // and 42.2 us; 2 heads, 612 causal: 14.9 and 17.7; 18 heads, 1024 (half as many tiles more than SMs): 26.1 in pairs.
  if ((static_cast<int64_t>(p.total_q) / kPtRows + p.batch) * p.hq <= sms) {
    p.item_heads = 1;
    return launch_tiles<T, D, kHeadsApart>(p, tq, tk, tv, sms, st);
  }
  if (p.group % 2 == 0) return launch_tiles<T, D, kHeadsOfGroup>(p, tq, tk, tv, sms, st);
  if (p.total_q <= kPtApartRows * static_cast<int64_t>(p.batch))
    return launch_tiles<T, D, kHeadsApart>(p, tq, tk, tv, sms, st);
  return launch_tiles<T, D, kTilesOfHead>(p, tq, tk, tv, sms, st);
}

b2g_status check_packed(const b2g_attention_packed_desc* d) {
  if (!d) return set_error(B2G_ERR_INVALID, "b2g_attention_packed: null descriptor");
  if (d->batch < 0 || d->total_q < 0 || d->total_k < 0 || d->n_head < 0 || d->n_kv_head < 0)
    return set_error(B2G_ERR_INVALID, "b2g_attention_packed: negative size");
  if (d->dtype != B2G_BF16 && d->dtype != B2G_F16)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_packed: BF16 or F16 operands");
  if (d->d_head != 64 && d->d_head != 128)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_packed: head dim must be 64 or 128");
  if (d->n_head > 0 && (d->n_kv_head < 1 || d->n_head % d->n_kv_head != 0))
    return set_error(B2G_ERR_INVALID, "b2g_attention_packed: n_head must be a multiple of n_kv_head");
  if (!(d->scale > 0.f) || !std::isfinite(d->scale))
    return set_error(B2G_ERR_INVALID, "b2g_attention_packed: scale must be positive");
  if (d->batch > 65536 || d->total_q > (1ll << 30) || d->total_k > (1ll << 30) || d->n_head > 65535)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_packed: size");
  return B2G_OK;
}

}  // namespace

size_t attention_packed_workspace(const b2g_attention_packed_desc* d) {
  DeviceInfo* dev = nullptr;
  if (check_packed(d) != B2G_OK || d->batch == 0 || d->total_q == 0 || d->n_head == 0 || device_info(&dev) != B2G_OK)
    return 0;
  return plan(d, dev->num_sms).bytes;
}

b2g_status attention_packed(const b2g_attention_packed_desc* d, void* workspace, size_t workspace_bytes,
                            cudaStream_t st) {
  b2g_status s = check_packed(d);
  if (s != B2G_OK) return s;
  if (d->batch == 0 || d->total_q == 0 || d->n_head == 0) return B2G_OK;
  if (!d->q || !d->out || !d->cu_q || !d->cu_k || (d->total_k > 0 && (!d->k || !d->v)))
    return set_error(B2G_ERR_INVALID, "b2g_attention_packed: null operand");
  const int64_t D = d->d_head;
  PkParams p{};
  p.ldq = used(d->ldq, d->total_q, d->n_head * D); p.hsq = used(d->hsq, d->n_head, D);
  p.ldk = used(d->ldk, d->total_k, d->n_kv_head * D); p.hsk = used(d->hsk, d->n_kv_head, D);
  p.ldv = used(d->ldv, d->total_k, d->n_kv_head * D); p.hsv = used(d->hsv, d->n_kv_head, D);
  p.ldo = used(d->ldo, d->total_q, d->n_head * D); p.hso = used(d->hso, d->n_head, D);
  const int64_t strides[8] = {p.ldq, p.hsq, p.ldk, p.hsk, p.ldv, p.hsv, p.ldo, p.hso};
  for (int64_t x : strides) {
    if (x < D) return set_error(B2G_ERR_INVALID, "b2g_attention_packed: a token or head stride is below the head dim");
    if (x % 8 != 0 || x >= (1ll << 38))
      return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_packed: strides must be multiples of 8 elements");
  }
  if ((reinterpret_cast<uintptr_t>(d->q) | reinterpret_cast<uintptr_t>(d->k) | reinterpret_cast<uintptr_t>(d->v) |
       reinterpret_cast<uintptr_t>(d->out)) & 15u)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_packed: 16-byte aligned operands required");
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  p.cu_q = d->cu_q; p.cu_k = d->cu_k; p.k_lens = d->k_lens;
  p.batch = static_cast<int>(d->batch);
  p.total_q = static_cast<int>(d->total_q); p.total_k = static_cast<int>(d->total_k);
  p.hq = d->n_head; p.hk = d->n_kv_head; p.group = d->n_head / d->n_kv_head;
  p.causal = d->causal ? 1 : 0;
  p.scale_log2 = d->scale * 1.4426950408889634f;
  p.q = d->q; p.k = d->k; p.v = d->v; p.out = d->out;
  p.err = dev->err_word;
  PkPlan pl = plan(d, dev->num_sms);
  void* ws = workspace;
  if (pl.bytes > 0) {
    if (!ws && (s = workspace_get(pl.bytes, &ws, kWsAttnSplit)) != B2G_OK) return s;
    if (workspace && (workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
      return set_error(B2G_ERR_INVALID, "b2g_attention_packed: the workspace is too small or not 256-byte aligned");
  }
  if (d->dtype == B2G_F16)
    return D == 128 ? run_packed<__half, 128>(d, p, ws, pl, dev->num_sms, st)
                    : run_packed<__half, 64>(d, p, ws, pl, dev->num_sms, st);
  return D == 128 ? run_packed<__nv_bfloat16, 128>(d, p, ws, pl, dev->num_sms, st)
                  : run_packed<__nv_bfloat16, 64>(d, p, ws, pl, dev->num_sms, st);
}

}  // namespace b2g
