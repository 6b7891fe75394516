// attention_blocks.cu — attention over packed sequences, of which every tile of queries sees some key
// blocks only, and what chooses the blocks.
//
// The keys of a sequence lie in blocks of 128, its queries in tiles of 128 (a single query is a tile of one).
//
//   block_means       m[j, g] = mean over the keys of block j of k[., g]
//   select_blocks     s[j] = (sum of the tile's queries, all heads of key head g's group) . m[j, g];
//                     bit j is set for the first and the last few blocks in sight, for blocks that some query of the
//                     tile sees in part, and for the `top` largest s[j] of the others (of equals the lowest j)
//   attention_blocks  out[i, h] = sum_j softmax_j(scale * q[i, h] . k[j, g]) v[j, g] over the keys of the set blocks
//
// Offsets are read on the device and clamped to the buffers, as in attention_packed.cu.
//
// The keys' sums, the statistics (row maximum and sum) and the output's sums are fp32, the blocks' scores 64 bits.  P is rounded
// to the operands' 16-bit type, as the tensor cores take it, at most 2^-8 (bf16) or 2^-11 (fp16) of a weight; the row's sum
// is taken before that.
//
//   packed_tiles (attention_packed.cuh)  long queries: tensor cores through TMEM, K and V by chosen block
//   chosen_rows, chosen_combine          few query rows per key head: equal shares of all that is chosen
#include "attention_packed.cuh"

namespace b2g {

namespace {

// ---------------------------------------------------------------------------- means of blocks
//
// Bound by memory: k is read once (16384 keys of 24 heads of 128: 20.1 us, 5.1 TB/s).  A warp reads 512 bytes of a key's row (8 values a lane) for 32 of the block's
// keys, kMnAhead loads at a time; the four warps' sums meet in shared memory in a fixed order.
constexpr int kMnWarps = 4;
constexpr int kMnAhead = 8;
constexpr int kMnPerSm = 12;  // CTAs an SM (the compiler's own choice is 10: 23.8 us; 16: 20.7)
constexpr int kMnCols = 256;  // values of a row that a block takes

struct MnParams {
  PkParams p;            // k, cu_k, k_lens
  const int* since;      // [batch] or NULL: all blocks
  float* means;          // [blocks, hk, D]
  int blocks, D;
};

__device__ __forceinline__ int key_blocks(const PkParams& p, int b) {  // with room left for more keys
  const int lo = clampi(__ldg(p.cu_k + b), 0, p.total_k);
  return (clampi(__ldg(p.cu_k + b + 1), lo, p.total_k) - lo + kPtKeys - 1) / kPtKeys;
}
// Blocks before sequence b's first (the whole warp).
__device__ __forceinline__ int blocks_before(const PkParams& p, int b, int lane) {
  int sum = 0;
#pragma unroll 4
  for (int i = lane; i < b; i += 32) sum = add_count(sum, key_blocks(p, i));
  return __reduce_add_sync(0xffffffffu, sum);
}

// Two values of a word.
template <typename T>
__device__ __forceinline__ float2 two(uint32_t w) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}
template <typename T>
__device__ __forceinline__ void add8(float (&sum)[8], uint4 v) {
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = two<T>(w[i]);
    sum[2 * i] += f.x;
    sum[2 * i + 1] += f.y;
  }
}

template <typename T>
__global__ void __launch_bounds__(32 * kMnWarps, kMnPerSm) block_means_kernel(const MnParams a) {
  __shared__ float4 sums[kMnWarps][2][32];
  const PkParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = blockIdx.y * kMnCols + lane * 8, cols = p.hk * a.D;
  griddep_wait();
  griddep_launch_dependents();
  int b, j, stop, base;
  const int step = a.since ? static_cast<int>(gridDim.z) : 1;
  if (a.since) {  // sequence blockIdx.x, its blocks from the one of key since[b] on
    b = blockIdx.x;
    const int since = __ldg(a.since + b);
    const Seq s = load_seq(p, b);
    base = blocks_before(p, b, lane);
    j = clampi(since, 0, s.lk) / kPtKeys + static_cast<int>(blockIdx.z);
    stop = (s.lk + kPtKeys - 1) / kPtKeys;
  } else {        // row blockIdx.x of the means
    base = 0;
    b = find_seq(p.batch, static_cast<int>(blockIdx.x), lane, [&](int i) { return key_blocks(p, i); }, &base);
    j = static_cast<int>(blockIdx.x) - base;
    stop = j + 1;
  }
  const Seq s = b >= 0 ? load_seq(p, b) : Seq{};
  const T* k = static_cast<const T*>(p.k) + (col < cols ? (col / a.D) * p.hsk + col % a.D : 0);
  for (; j < stop && base + j < a.blocks; j += step) {
    const int key0 = j * kPtKeys, n = b >= 0 ? clampi(s.lk - key0, 0, kPtKeys) : 0;
    float sum[8] = {};
    if (col < cols)
#pragma unroll
      for (int r0 = 0; r0 < 32; r0 += kMnAhead) {
        uint4 v[kMnAhead];
#pragma unroll
        for (int i = 0; i < kMnAhead; ++i) {
          const int r = warp * 32 + r0 + i;
          v[i] = make_uint4(0, 0, 0, 0);
          if (r < n) v[i] = __ldg(reinterpret_cast<const uint4*>(k + static_cast<long long>(s.k0 + key0 + r) * p.ldk));
        }
#pragma unroll
        for (int i = 0; i < kMnAhead; ++i) add8<T>(sum, v[i]);
      }
    sums[warp][0][lane] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    sums[warp][1][lane] = make_float4(sum[4], sum[5], sum[6], sum[7]);
    __syncthreads();
    if (warp < 2) {  // values 4 warp to 4 warp + 3 of each lane's 8
      const float4 x = sums[0][warp][lane], y = sums[1][warp][lane], z = sums[2][warp][lane], w = sums[3][warp][lane];
      const float count = static_cast<float>(max(n, 1));
      if (col < cols)
        *reinterpret_cast<float4*>(a.means + static_cast<long long>(base + j) * cols + col + 4 * warp) =
            make_float4(((x.x + y.x) + (z.x + w.x)) / count, ((x.y + y.y) + (z.y + w.y)) / count,
                        ((x.z + y.z) + (z.z + w.z)) / count, ((x.w + y.w) + (z.w + w.w)) / count);
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------- choice of blocks
//
// Bound by instructions, not by q's bytes (16384 queries of 24 heads: 46.7 us, floor 15.6): the summing of the queries and the
// scores after it do not overlap.  Scores are sums of 64 bits: a choice compares neighbours, and any rounding of theirs in 32 bits would decide
// the choice where two are close; in 64 bits the order of a sum moves one in some 10^12.
constexpr int kSlThreads = 256;
constexpr int kSlMostWords = 256;

struct SlParams {
  PkParams p;           // q, cu_q, cu_k, k_lens, causal
  const float* means;   // [blocks, hk, D]
  int blocks, D;
  int top, first, last;
  uint32_t* chosen;     // [tiles, hk, words]
  int tiles, words;
};

// Order of scores as that of whole numbers: NaN as -inf, -0 as 0; 0 is below every score.
__device__ __forceinline__ unsigned long long score_order(double s) {
  if (isnan(s)) s = -INFINITY;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(s + 0.0));
  return u >> 63 ? ~u : u | (1ull << 63);
}

// hi + lo += x exactly, up to lo's own rounding (2^-48 of the sum), for two values at a time.
__device__ __forceinline__ uint64_t f2_sub(uint64_t a, uint64_t b) { return f2_fma(b, f2_splat(-1.f), a); }
__device__ __forceinline__ void add_pair(uint64_t& hi, uint64_t& lo, uint64_t x) {
  const uint64_t sum = f2_add(hi, x), part = f2_sub(sum, hi);
  lo = f2_add(lo, f2_add(f2_sub(hi, f2_sub(sum, part)), f2_sub(x, part)));
  hi = sum;
}

// c += a b, 8 x 8 x 4 in 64 bits.
__device__ __forceinline__ void mma_884(double (&c)[2], double a, double b) {
  asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};" : "+d"(c[0]), "+d"(c[1]) : "d"(a), "d"(b));
}

template <typename T, int D, int NT>  // NT neighbouring tiles a CTA
__global__ void __launch_bounds__(kSlThreads) select_blocks_kernel(const SlParams a) {
  constexpr int kPieces = D / 8, kGroups = kSlThreads / kPieces;  // 16-byte pieces of a row, rows at a time
  constexpr int kWarps = kSlThreads / 32, kPitch = D + 4;         // (values from sum to sum, for the banks)
  static_assert(NT <= 8 && NT <= kWarps, "tiles");
  extern __shared__ __align__(16) unsigned char smem_sl[];
  double* part = reinterpret_cast<double*>(smem_sl);                                                    // [warp][NT][kPitch]
  unsigned long long* order = reinterpret_cast<unsigned long long*>(part + NT * kWarps * kPitch);             // [NT][32 words]: scores
  const PkParams& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.x % p.hk, tile0 = static_cast<int>(blockIdx.x / p.hk) * NT;
  const int most = 32 * a.words;
  griddep_wait();
  griddep_launch_dependents();
  // The tiles: rows, blocks in sight, the first and the last query's keys, where the sequence's means begin.
  struct Tile {
    int rows, q0, sees_first, sees_last, nb, base;
  };
  __shared__ Tile tiles[NT];
  if (warp < NT) {
    Tile t{};
    int before = 0;
    const int tile = tile0 + warp;
    const int b = tile < a.tiles ? find_seq(p.batch, tile, lane, [&](int i) {
      const int lo = clampi(__ldg(p.cu_q + i), 0, p.total_q);
      return (clampi(__ldg(p.cu_q + i + 1), lo, p.total_q) - lo + kPtRows - 1) / kPtRows;
    }, &before) : -1;
    if (b >= 0) {
      const Seq s = load_seq(p, b);
      const int row0 = (tile - before) * kPtRows;
      t.base = blocks_before(p, b, lane);
      t.rows = min(kPtRows, s.lq - row0);
      t.q0 = s.q0 + row0;
      t.sees_first = p.causal ? clampi(row0 + 1 + s.lk - s.lq, 0, s.lk) : s.lk;
      t.sees_last = p.causal ? clampi(row0 + t.rows + s.lk - s.lq, 0, s.lk) : s.lk;
      t.nb = min((t.sees_last + kPtKeys - 1) / kPtKeys, most);
    }
    if (lane == 0) tiles[warp] = t;
  }
  __syncthreads();
  // The tiles' queries, summed: in pairs of fp32 by a thread, in 64 bits after that.
  const int piece = threadIdx.x % kPieces, from = threadIdx.x / kPieces;
#pragma unroll 1
  for (int n = 0; n < NT; ++n) {
    const Tile t = tiles[n];
    const T* q = static_cast<const T*>(p.q) + static_cast<long long>(t.q0) * p.ldq + static_cast<long long>(g) * p.group * p.hsq + piece * 8;
    uint64_t hi[4], lo[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) hi[x] = lo[x] = 0;
    const int items = t.nb > 0 ? t.rows * p.group : 0;
    constexpr int kAheadQ = 8;
    for (int i0 = from; i0 < items; i0 += kAheadQ * kGroups) {
      uint4 v[kAheadQ];
#pragma unroll
      for (int u = 0; u < kAheadQ; ++u) {
        const int i = i0 + u * kGroups, row = p.group == 1 ? i : i / p.group, h = i - row * p.group;
        v[u] = i < items ? __ldg(reinterpret_cast<const uint4*>(q + row * p.ldq + h * p.hsq)) : make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int u = 0; u < kAheadQ; ++u) {
        if (i0 - from + u * kGroups >= items) break;  // (for the whole CTA)
        const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float2 f = two<T>(w[x]);
          add_pair(hi[x], lo[x], f2_pack(__float_as_uint(f.x), __float_as_uint(f.y)));
        }
      }
    }
    double sum[8];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const float2 h = f2_unpack(hi[x]), l = f2_unpack(lo[x]);
      // (the second is no number where the first is infinite)
      sum[2 * x] = isfinite(h.x) ? static_cast<double>(h.x) + static_cast<double>(l.x) : static_cast<double>(h.x);
      sum[2 * x + 1] = isfinite(h.y) ? static_cast<double>(h.y) + static_cast<double>(l.y) : static_cast<double>(h.y);
    }
#pragma unroll
    for (int o = 16; o >= kPieces; o >>= 1)
#pragma unroll
      for (int x = 0; x < 8; ++x) sum[x] += __shfl_xor_sync(0xffffffffu, sum[x], o);
    if (lane < kPieces)
#pragma unroll
      for (int x = 0; x < 8; ++x) part[(warp * NT + n) * kPitch + piece * 8 + x] = sum[x];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < NT * D; c += kSlThreads) {
    double* at = part + c / D * kPitch + c % D;
    double sum = at[0];
#pragma unroll
    for (int i = 1; i < kWarps; ++i) sum += at[i * NT * kPitch];
    at[0] = sum;
  }
  __syncthreads();
  // Scores, by products of 8 tiles x 8 blocks x 4 values in 64 bits: lane (r, t) holds the values 16 c + 4 t + e of tile r and
  // of block r for the products e of the 16 values c, and gets the scores of tile r for blocks 2 t and 2 t + 1.
  int nb_most = 0, base = 0;
  bool one = true;  // one sequence (the others see nothing), whose means are read once for all tiles
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (tiles[n].nb > 0) {
      one = one && (nb_most == 0 || base == tiles[n].base);
      base = tiles[n].base;
      nb_most = max(nb_most, tiles[n].nb);
    }
  const int r = lane >> 2, t4 = lane & 3;
  auto scores = [&](int nb, int mean0, int n0, int n1) {  // blocks below nb of tiles n0 to n1
    for (int j0 = warp * 8; j0 < nb; j0 += kWarps * 8) {
      __syncwarp();  // (the products are the whole warp's, the end of a round is not)
      float4 m[D / 16];
      const int at = mean0 + j0 + r;
      const bool in = j0 + r < nb && at < a.blocks;
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
        m[c] = in ? __ldg(reinterpret_cast<const float4*>(a.means + (static_cast<long long>(at) * p.hk + g) * D + 16 * c + 4 * t4))
                  : make_float4(0.f, 0.f, 0.f, 0.f);
      double s[2][2] = {};  // (two sums side by side)
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        double2 q01 = make_double2(0.0, 0.0), q23 = q01;
        if (NT == 8 || r < NT) {
          const double* q = part + r * kPitch + 16 * c + 4 * t4;
          q01 = *reinterpret_cast<const double2*>(q);
          q23 = *reinterpret_cast<const double2*>(q + 2);
        }
        mma_884(s[0], q01.x, m[c].x);
        mma_884(s[1], q01.y, m[c].y);
        mma_884(s[0], q23.x, m[c].z);
        mma_884(s[1], q23.y, m[c].w);
      }
      if (r < n0 || r >= n1) continue;
      const Tile& tile = tiles[r];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = j0 + 2 * t4 + e;
        const bool sure = j < a.first || j >= tile.nb - a.last || min((j + 1) * kPtKeys, tile.sees_last) > tile.sees_first;
        if (j < tile.nb) order[r * most + j] = sure ? 0 : score_order(s[0][e] + s[1][e]);
      }
    }
  };
  if (one) scores(nb_most, base, 0, NT);
  else
    for (int n = 0; n < NT; ++n) scores(tiles[n].nb, tiles[n].base, n, n + 1);
  __syncthreads();
  // A warp takes a tile: the largest threshold that `top` scores reach, bit by bit from above (fewer scores: 1, all of
  // them), looked for until it parts them; then the words.
  if (warp >= NT || tile0 + warp >= a.tiles) return;
  const unsigned long long* mine = order + warp * most;
  const int nb = tiles[warp].nb;
  uint32_t* out = a.chosen + (static_cast<long long>(tile0 + warp) * p.hk + g) * a.words;
  constexpr int kHeld = 8;  // scores in a lane's registers, as they come first
  unsigned long long held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i) held[i] = 32 * i + lane < nb ? mine[32 * i + lane] : 0;
  auto reach = [&](unsigned long long least) {
    int n = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) n += held[i] >= least;
    for (int j = 32 * kHeld + lane; j < nb; j += 32) n += mine[j] >= least;
    return __reduce_add_sync(0xffffffffu, n);
  };
  unsigned long long least = 0;
  int reached = reach(1), bit = -1;  // (no more than are to be taken: all of them)
  if (reached > a.top) {
    // The upper words' common bits need no search.
    uint32_t low = 0xFFFFFFFFu, high = 0;
    auto extend = [&](unsigned long long x) {
      const uint32_t word = static_cast<uint32_t>(x >> 32);
      if (x) {
        low = min(low, word);
        high = max(high, word);
      }
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) extend(held[i]);
    for (int j = 32 * kHeld + lane; j < nb; j += 32) extend(mine[j]);
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    const int same = __clz(low ^ high);
    bit = 63 - same;
    if (same > 0) least = static_cast<unsigned long long>(high & ~(same >= 32 ? 0u : 0xFFFFFFFFu >> same)) << 32;
  }
  for (; bit >= 0 && reached > a.top; --bit) {
    const unsigned long long next = least | (1ull << bit);
    const int n = reach(next);
    if (n >= a.top) {
      least = next;
      reached = n;
    }
  }
  if (least == 0) least = 1;
  int room = 0;  // of the scores that equal the threshold, as many as are still to be taken
  if (reached > a.top) room = a.top - (least == ~0ull ? 0 : reach(least + 1));
  else room = nb;
  for (int w = 0; w < a.words; ++w) {
    const int j = 32 * w + lane;
    const unsigned long long x = j < nb ? mine[j] : 0;
    const uint32_t equal = __ballot_sync(0xffffffffu, j < nb && x == least);
    const bool take = j < nb && (x == 0 || x > least || (x == least && __popc(equal & ((1u << lane) - 1u)) < room));
    const uint32_t bits = __ballot_sync(0xffffffffu, take);
    room -= __popc(equal);
    if (lane == 0) out[w] = bits;
  }
}

// ---------------------------------------------------------------------------- few rows over chosen blocks
//
// Bound by memory where caches are long, by round trips otherwise (48 single queries, 32 heads on 8, 18 blocks: 38.3 us for
// 97 MB with the join).  The query rows of one key head (lq tokens x group heads) in tiles of 16.  The products, the lanes' layout and the
// copies are those of packed_rows_kernel (attention_packed.cu): in a CTA the warps take 16 keys of the chosen blocks in turn.
//
// Pairs of a sequence and a key head choose different numbers of blocks (an empty cache none, a long one all that it
// may).  Their tiles lie end to end on a line, each as long as its chunks of 16 chosen keys and kCrTileCost more; the line
// is cut into equal shares, one a CTA, and a tile that lies in several is joined by chosen_combine.  A CTA finds its
// share in sums over the pairs that it takes itself, from the words of `chosen`: up to kCrPairs pairs; with more of
// them a CTA takes a tile.
constexpr int kCrWarps = 4;
constexpr int kCrRows = 16;
constexpr int kCrKeys = 16;
constexpr int kCrBlocksPerSm = 2;
constexpr int kCrListed = 256;  // chosen blocks that are listed at a time
constexpr int kCrPairs = 1024;
// What a tile costs beside its chunks, in chunks.  (64 caches of up to 700 keys: 4 50.1 us, 12 43.2, 24 45.8; 48 of up to 16383:
// 94.1, 92.7, 93.7)
constexpr int kCrTileCost = 12;
constexpr int kCrMinShare = 16;  // a share is at least so long
template <int D>
constexpr int kCrPieces = D / 8;
template <int D>
constexpr int kCrStages = D == 128 ? 3 : 6;
template <int D>
constexpr uint32_t kCrSmem = kCrWarps * kCrStages<D> * kCrPieces<D> * 512u;

// A tile of 16 rows of a sequence and key head, and its row of `chosen`.
struct CrTile {
  Seq s;
  int head, rows, row0, sees;  // rows of the sequence; the keys that any of the tile's rows sees
  const uint32_t* words;
  int nb;                      // blocks in sight
  __device__ __forceinline__ uint32_t word(int w) const {
    if (32 * w >= nb) return 0u;
    const uint32_t bits = __ldg(words + w);
    return nb - 32 * w >= 32 ? bits : bits & ((1u << (nb - 32 * w)) - 1u);
  }
  // Chunks: a block has 8; of the last one in sight, where it is chosen, only those with keys.
  __device__ __forceinline__ int less() const {
    const bool last = nb > 0 && (word((nb - 1) >> 5) >> ((nb - 1) & 31) & 1u) != 0;
    return last ? 8 - (min(sees - (nb - 1) * kPtKeys, kPtKeys) + kCrKeys - 1) / kCrKeys : 0;
  }
};
// mask_tiles: rows of `chosen` before sequence b's.
__device__ __forceinline__ CrTile chosen_tile(const PkParams& p, const Seq& s, int head, int tile, int mask_tiles) {
  CrTile r;
  r.s = s;
  r.head = head;
  r.rows = s.lq * p.group;
  r.row0 = tile * kCrRows;
  const int first_token = r.row0 / p.group, last_token = (min(r.row0 + kCrRows, r.rows) - 1) / p.group;
  r.sees = p.causal ? clampi(last_token + 1 + s.lk - s.lq, 0, s.lk) : s.lk;
  const int at = mask_tiles + first_token / kPtRows;  // (128 / 16 * group tiles of rows share one)
  r.words = p.chosen + (static_cast<long long>(at) * p.hk + head) * p.chosen_words;
  r.nb = at < p.chosen_tiles ? min((r.sees + kPtKeys - 1) / kPtKeys, 32 * p.chosen_words) : 0;
  return r;
}
__device__ __forceinline__ int chosen_tiles_of(const PkParams& p, int lq) {
  return static_cast<int>((static_cast<long long>(lq) * p.group + kCrRows - 1) / kCrRows);
}
// One thread's count of a tile's length on the line.
__device__ __forceinline__ int chosen_length(const CrTile& c) {
  int count = 0;
  for (int w = 0; 32 * w < c.nb; ++w) count += __popc(c.word(w));
  return 8 * count - c.less() + kCrTileCost;
}

// The line: sums over the pairs (sequence b, key head g) at b * hk + g, taken by all threads of the CTA.
struct CrLine {
  const long long* ends;  // shared memory [pairs]: the line's length up to the pair's end
  const int* mask_tiles;  // shared memory [batch]: rows of `chosen` up to the sequence's end
  long long total;
  int shares;
};
// Inclusive sums of the n values in `ends`.
template <int kThreads, typename I>
__device__ __forceinline__ void sums_of(int n, I* ends, long long* carry) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __syncthreads();
  I base = 0;
  for (int i0 = 0; i0 < n; i0 += kThreads) {
    const int i = i0 + threadIdx.x;
    I sum = i < n ? ends[i] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const I up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (lane == 31) carry[warp] = sum;
    __syncthreads();
    I before = base;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      before += w < warp ? static_cast<I>(carry[w]) : 0;
      base += static_cast<I>(carry[w]);
    }
    if (i < n) ends[i] = before + sum;
    __syncthreads();
  }
}
template <int kThreads>
__device__ __forceinline__ CrLine chosen_line(const PkParams& p, long long* ends, int* mask_tiles, long long* carry) {
  for (int b = threadIdx.x; b < p.batch; b += kThreads) {
    const int lo = clampi(__ldg(p.cu_q + b), 0, p.total_q);
    mask_tiles[b] = (clampi(__ldg(p.cu_q + b + 1), lo, p.total_q) - lo + kPtRows - 1) / kPtRows;
  }
  sums_of<kThreads>(p.batch, mask_tiles, carry);
  // A thread takes kAhead pairs, whose loads go out together: of sequences with one tile of rows (most of them) four
  // words at a time.
  constexpr int kAhead = 4;
  const int pairs = p.batch * p.hk, words = p.chosen_words;
  for (int i0 = threadIdx.x; i0 < pairs; i0 += kAhead * kThreads) {
    const uint32_t* from[kAhead];
    int tiles[kAhead], nb[kAhead], keys[kAhead], count[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = min(i0 + u * kThreads, pairs - 1), b = i / p.hk;
      const Seq s = load_seq(p, b);
      const int before = mask_tiles[b] - (s.lq + kPtRows - 1) / kPtRows;
      tiles[u] = chosen_tiles_of(p, s.lq);
      keys[u] = s.lk;  // (a sequence's last query sees every key)
      nb[u] = tiles[u] == 1 && before < p.chosen_tiles ? min((s.lk + kPtKeys - 1) / kPtKeys, 32 * words) : 0;
      from[u] = p.chosen + (static_cast<long long>(before) * p.hk + i - b * p.hk) * words;
      count[u] = 0;
    }
    for (int w0 = 0; w0 < words; w0 += 4) {
      uint32_t bits[kAhead][4];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) bits[u][w] = 32 * (w0 + w) < nb[u] ? __ldg(from[u] + w0 + w) : 0u;
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int left = nb[u] - 32 * (w0 + w);  // of the word's blocks in sight
          const uint32_t in = left >= 32 ? bits[u][w] : left > 0 ? bits[u][w] & ((1u << left) - 1u) : 0u;
          count[u] += 8 * __popc(in);
          if (left > 0 && left <= 32 && (in >> (left - 1) & 1u))  // the last block, of which only chunks with keys count
            count[u] -= 8 - (min(keys[u] - (nb[u] - 1) * kPtKeys, kPtKeys) + kCrKeys - 1) / kCrKeys;
        }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * kThreads;
      if (i < pairs) ends[i] = tiles[u] == 1 ? count[u] + kCrTileCost : -tiles[u];
    }
  }
  __syncthreads();
  // Pairs with more tiles of rows (less than 0: as many): each by a lane, or by the whole warp, one pair after the other, where
  // that takes fewer rounds, as it does for a long sequence among short ones.
  const int lane = threadIdx.x & 31;
  for (int i0 = threadIdx.x - lane; i0 < pairs; i0 += kThreads) {
    const int n = i0 + lane < pairs ? static_cast<int>(max(-ends[i0 + lane], 0ll)) : 0;
    const uint32_t many = __ballot_sync(0xffffffffu, n > 0);
    if (!many) continue;
    const bool shared = 2 * __reduce_add_sync(0xffffffffu, (n + 31) / 32) < __reduce_max_sync(0xffffffffu, n);
    auto sum_of = [&](int i, int first, int step, int tiles) {
      const int b = i / p.hk;
      const Seq s = load_seq(p, b);
      const int before = mask_tiles[b] - (s.lq + kPtRows - 1) / kPtRows;
      long long sum = 0;
      for (int tile = first; tile < tiles; tile += step) sum += chosen_length(chosen_tile(p, s, i - b * p.hk, tile, before));
      return sum;
    };
    if (!shared) {
      if (n > 0) ends[i0 + lane] = sum_of(i0 + lane, 0, 1, n);
      continue;
    }
    for (uint32_t left = many; left; left &= left - 1) {
      const int at = __ffs(left) - 1;
      long long sum = sum_of(i0 + at, lane, 32, __shfl_sync(0xffffffffu, n, at));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (lane == 0) ends[i0 + at] = sum;
    }
  }
  sums_of<kThreads>(pairs, ends, carry);
  const long long total = ends[pairs - 1], most = (total + kCrMinShare - 1) / kCrMinShare;
  return {ends, mask_tiles, total, static_cast<int>(min(static_cast<long long>(p.shares), most))};
}
// Where share i begins.
__device__ __forceinline__ long long cut_at(const CrLine& line, int i) { return line.total * i / line.shares; }
// Where a search left off: tile `tile` of pair `pair` begins at `start`.
struct CrPlace {
  int pair, tile;
  long long start;
};
// The tile that holds place `at` of the line: the tile, its start and length.  Whole warps search; of a pair with many tiles 32 at
// a time, from `from` on where it is in the same pair (a share's tiles follow one another).
__device__ __forceinline__ CrTile chosen_at(const PkParams& p, const CrLine& line, long long at, long long* start, int* length,
                                            CrPlace* from) {
  int lo = 0, hi = p.batch * p.hk - 1;  // the first pair that ends past `at`
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (line.ends[mid] > at) hi = mid;
    else lo = mid + 1;
  }
  const int b = lo / p.hk;
  const Seq s = load_seq(p, b);
  const int before = line.mask_tiles[b] - (s.lq + kPtRows - 1) / kPtRows, tiles = chosen_tiles_of(p, s.lq);
  if (from->pair != lo) *from = {lo, 0, lo > 0 ? line.ends[lo - 1] : 0};
  *start = from->start;
  int tile = from->tile;
  if (tiles == 1) {
    *length = static_cast<int>(line.ends[lo] - *start);
  } else {
    const int lane = threadIdx.x & 31;
    for (;; tile += 32) {
      const int mine = tile + lane < tiles ? chosen_length(chosen_tile(p, s, lo - b * p.hk, tile + lane, before)) : 0;
      long long sum = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long up = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += up;
      }
      const uint32_t past = __ballot_sync(0xffffffffu, *start + sum > at || tile + lane >= tiles - 1);
      if (past) {
        const int in = __ffs(past) - 1;
        *start += __shfl_sync(0xffffffffu, sum - mine, in);
        *length = __shfl_sync(0xffffffffu, mine, in);
        tile += in;
        break;
      }
      *start += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  *from = {lo, tile, *start};
  return chosen_tile(p, s, lo - b * p.hk, tile, before);
}

// With part i holding (m_i, l_i) and O_i: O = sum 2^(m_i - M) O_i, l = sum 2^(m_i - M) l_i.  (A part without a key has
// the sums 0; a NaN maximum does not occur, a NaN sum stays one.)
__device__ __forceinline__ float part_weight(float2 ml, float top) {
  return ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : 1.f) : fast_exp2(ml.x - top);
}
__device__ __forceinline__ void add_part(float4& acc, float w, float4 x) {
  acc.x += w * x.x;
  acc.y += w * x.y;
  acc.z += w * x.z;
  acc.w += w * x.w;
}
template <typename T>
__device__ __forceinline__ void store_row(const PkParams& p, const CrTile& c, int r, int d, float sum, float4 acc) {
  const int token = (c.row0 + r) / p.group, h = (c.row0 + r) - token * p.group;
  const float inv = sum != 0.f ? 1.f / sum : 0.f;
  T* dst = static_cast<T*>(p.out) + (c.s.q0 + token) * p.ldo + (static_cast<long long>(c.head) * p.group + h) * p.hso + d;
  *reinterpret_cast<uint2*>(dst) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
}

// Chunks [c_from, c_to) of a tile: its rows of `out` if slot < 0, else a part there.
template <typename T, int D>
__device__ __forceinline__ void chosen_part(const PkParams& p, const CrTile& tile, int c_from, int c_to, int slot, uint8_t* smem_rows,
                                            float2 (*sml)[kCrRows], int* list) {
  constexpr int KC = D / 32, VC = D / 64, NS = kCrStages<D>;
  constexpr uint32_t kStage = kCrPieces<D> * 512u;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = smem_u32(smem_rows) + warp * NS * kStage + lane * 16;
  auto so = [&](int w) { return reinterpret_cast<float*>(smem_rows + w * NS * kStage); };
  static_assert(kCrRows * (D + 4) * 4 <= NS * kStage, "sums fit a ring");
  const Seq& s = tile.s;
  const int head = tile.head, rows = tile.rows, row0 = tile.row0, tile_sees = tile.sees, nb = tile.nb;
  const T* kbase = static_cast<const T*>(p.k) + s.k0 * p.ldk + head * p.hsk + 8 * t;
  const T* vbase = static_cast<const T*>(p.v) + s.k0 * p.ldv + head * p.hsv + 8 * g;
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

  for (int block0 = c_from / 8; block0 * 8 < c_to; block0 += kCrListed) {
    // The chosen blocks block0 to block0 + kCrListed, in order.
    __syncthreads();
    if (warp == 0) {
      int seen = 0;
      for (int w0 = 0; 32 * w0 < nb && seen < block0 + kCrListed; w0 += 32) {
        uint32_t bits = tile.word(w0 + lane);
        int sum = __popc(bits);
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, sum, x);
          if (lane >= x) sum += up;
        }
        int at = seen + sum - __popc(bits) - block0;
        for (; bits; bits &= bits - 1, ++at)
          if (at >= 0 && at < kCrListed) list[at] = (w0 + lane) * 32 + __ffs(bits) - 1;
        seen += __shfl_sync(0xffffffffu, sum, 31);
      }
    }
    __syncthreads();
    const int c0 = max(c_from, block0 * 8), c1 = min(c_to, (block0 + kCrListed) * 8);
    auto first_key = [&](int c) { return list[(c >> 3) - block0] * kPtKeys + (c & 7) * kCrKeys; };
    // Copies chunk c into stage st: keys that no row of the tile sees are zeros.
    auto fetch = [&](int c, int st) {
      const uint32_t dst = ring + st * kStage;
      const int key0 = first_key(c);
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int key = key0 + nt * 8 + g;
        const bool live = key < tile_sees;
        const T* src = live ? kbase + key * p.ldk : kbase;
#pragma unroll
        for (int i = 0; i < KC; ++i) copy16(dst + (nt * KC + i) * 512, src + 32 * i, live);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int key = key0 + 2 * t + (i & 1) + 8 * (i >> 1);
        const bool live = key < tile_sees;
        const T* src = live ? vbase + key * p.ldv : vbase;
#pragma unroll
        for (int k = 0; k < VC; ++k) copy16(dst + (2 * KC + i * VC + k) * 512, src + 64 * k, live);
      }
    };
    // The first NS - 1 rounds only copy.  (One place in the code for all copies: a kernel begins with its instructions far away.)
    int ahead = c0 + warp, ahead_st = 0, st = 0;
#pragma unroll 1
    for (int c = c0 + warp - (NS - 1) * kCrWarps; c < c1; c += kCrWarps) {
      if (ahead < c1) fetch(ahead, ahead_st);  // (the stage used up in the last round)
      copy_commit();
      ahead += kCrWarps;
      ahead_st = ahead_st + 1 == NS ? 0 : ahead_st + 1;
      if (c < c0) continue;
      copy_wait<NS - 1>();
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
      // Scores in log2 units; sc[nt][2i + e] is row g + 8i, key 8nt + 2t + e of the chunk.
      const int key0 = first_key(c);
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = key0 + nt * 8 + 2 * t + (j & 1);
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
  }
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
  const int live_rows = min(kCrRows, rows - row0);
  for (int at = threadIdx.x; at < live_rows * (D / 4); at += 32 * kCrWarps) {
    const int r = at / (D / 4), d = (at - r * (D / 4)) * 4;
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kCrWarps; ++w) top = fmaxf(top, sml[w][r].x);
#pragma unroll
    for (int w = 0; w < kCrWarps; ++w) {
      const float wgt = part_weight(sml[w][r], top);
      sum += wgt * sml[w][r].y;
      add_part(acc, wgt, *reinterpret_cast<const float4*>(so(w) + r * (D + 4) + d));
    }
    if (slot < 0) store_row<T>(p, tile, r, d, sum, acc);
    else {
      const long long to = static_cast<long long>(slot) * kCrRows + r;
      *reinterpret_cast<float4*>(p.part_o + to * D + d) = acc;
      if (d == 0) p.part_ml[to] = make_float2(top, sum);
    }
  }
  __syncthreads();  // the shared buffers are used again
}

template <typename T, int D, bool kLine>
__global__ void __launch_bounds__(32 * kCrWarps, kCrBlocksPerSm) chosen_rows_kernel(const PkParams p) {
  extern __shared__ __align__(16) uint8_t smem_rows[];
  __shared__ float2 sml[kCrWarps][kCrRows];
  __shared__ int list[kCrListed];
  griddep_wait();
  griddep_launch_dependents();
  if constexpr (kLine) {
    __shared__ int mask_tiles[kCrPairs];
    __shared__ long long ends[kCrPairs], carry[kCrWarps];
    const CrLine line = chosen_line<32 * kCrWarps>(p, ends, mask_tiles, carry);
    const int share = blockIdx.x;
    if (share >= line.shares) return;
    const long long end = cut_at(line, share + 1);
    CrPlace place{-1, 0, 0};
    for (long long at = cut_at(line, share); at < end;) {
      long long start;
      int length;
      const CrTile tile = chosen_at(p, line, at, &start, &length, &place);
      const int from = static_cast<int>(at - start), to = static_cast<int>(min(static_cast<long long>(length), end - start));
      at = max(start + to, at + 1);  // (further on also where the words change under the kernel)
      const int slot = to - from < length ? 2 * share + (from == 0 ? 1 : 0) : -1;
      chosen_part<T, D>(p, tile, max(0, from - kCrTileCost), max(0, to - kCrTileCost), slot, smem_rows, sml, list);
    }
  } else {
    const int lane = threadIdx.x & 31;
    const int at_tile = static_cast<int>(blockIdx.x) / p.hk, head = static_cast<int>(blockIdx.x) - at_tile * p.hk;
    int before = 0;
    const int b = find_seq(p.batch, at_tile, lane, [&](int i) {
      const int lo = clampi(__ldg(p.cu_q + i), 0, p.total_q);
      return chosen_tiles_of(p, clampi(__ldg(p.cu_q + i + 1), lo, p.total_q) - lo);
    }, &before);
    if (b < 0) return;
    int mask_tiles = 0;
    for (int i = lane; i < b; i += 32) {
      const int lo = clampi(__ldg(p.cu_q + i), 0, p.total_q);
      mask_tiles = add_count(mask_tiles, (clampi(__ldg(p.cu_q + i + 1), lo, p.total_q) - lo + kPtRows - 1) / kPtRows);
    }
    const CrTile tile = chosen_tile(p, load_seq(p, b), head, at_tile - before, __reduce_add_sync(0xffffffffu, mask_tiles));
    chosen_part<T, D>(p, tile, 0, chosen_length(tile) - kCrTileCost, -1, smem_rows, sml, list);
  }
}

// Joins the parts of every tile that lies in several shares.  A CTA looks at the cut between two shares and takes the
// tile there if it is the tile's first cut; a thread joins 4 values of a row, kCcAhead parts' loads at a time.  All but the
// parts is read before the wait for chosen_rows, which lets this kernel start after its own wait.
constexpr int kCcAhead = 8;
constexpr int kCcThreads = 128;
template <typename T, int D>
__global__ void __launch_bounds__(kCcThreads) chosen_combine_kernel(const PkParams p) {
  __shared__ int mask_tiles[kCrPairs];
  __shared__ long long ends[kCrPairs], carry[kCcThreads / 32];
  const CrLine line = chosen_line<kCcThreads>(p, ends, mask_tiles, carry);
  const int cut = static_cast<int>(blockIdx.x) + 1;
  CrTile tile{};
  int parts = 0;
  if (cut < line.shares) {
    long long start;
    int length;
    CrPlace place{-1, 0, 0};
    tile = chosen_at(p, line, cut_at(line, cut), &start, &length, &place);
    // (a share may be longer than the tile: then the cut before this one is outside it)
    if (start != cut_at(line, cut) && cut_at(line, cut - 1) <= start)
      for (parts = 2; cut + parts - 1 < line.shares && cut_at(line, cut + parts - 1) < start + length;) ++parts;
  }
  griddep_wait();  // (this kernel's end stands for chosen_rows' end too)
  if (parts == 0) return;
  const int live_rows = min(kCrRows, tile.rows - tile.row0);
  const long long first = static_cast<long long>(2 * (cut - 1) + 1) * kCrRows, second = 2ll * cut * kCrRows, step = 2ll * kCrRows;
  for (int at4 = threadIdx.x; at4 < live_rows * (D / 4); at4 += kCcThreads) {
    const int r = at4 / (D / 4), d = (at4 - r * (D / 4)) * 4;
    float top = -INFINITY, sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int i0 = 0; i0 < parts; i0 += kCcAhead) {
      float2 ml[kCcAhead];
      float4 x[kCcAhead];
#pragma unroll
      for (int i = 0; i < kCcAhead; ++i) {
        const bool in = i0 + i < parts;
        const long long slot = (i0 + i == 0 ? first : second + (i0 + i - 1) * step) + r;
        ml[i] = in ? __ldcg(p.part_ml + slot) : make_float2(-INFINITY, 0.f);
        x[i] = in ? __ldcg(reinterpret_cast<const float4*>(p.part_o + slot * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
      float next = top;
#pragma unroll
      for (int i = 0; i < kCcAhead; ++i) next = fmaxf(next, ml[i].x);
      const float alpha = top == next ? 1.f : fast_exp2(top - next);
      top = next;
      sum *= alpha;
      acc.x *= alpha; acc.y *= alpha; acc.z *= alpha; acc.w *= alpha;
#pragma unroll
      for (int i = 0; i < kCcAhead; ++i) {
        const float wgt = part_weight(ml[i], top);
        sum += wgt * ml[i].y;
        add_part(acc, wgt, x[i]);
      }
    }
    store_row<T>(p, tile, r, d, sum, acc);
  }
}

// ---------------------------------------------------------------------------- host side

// Which form takes a call.  chosen_rows costs by tiles of 16 rows of a key head's group, each of which reads its keys,
// packed_tiles by heads of q.  us, rows and tiles, d 128, 48 sequences with 18 of 32 blocks or 4 with 26 of 128:
//   q heads, key heads    1 query      8 queries    16 queries
//   32, 8    48           -            210, 242     391, 242
//   16, 8    48           106, 124     115, 127     210, 127
//   32, 4    4            20.7, 58.1   44.4, 58.2   71.5, 58.3
//   8, 8     4            26.5, 57.6   28.0, 57.8   31.4, 57.9
// Heads of their own leave nothing to share, and tiles of many long caches stream faster (8 heads: 128 of 4096 keys
// 253, 202; 64: 135, 110; 48: 106, 103; 24 heads: 64 of 1500 249, 206, but 64 of 300 69, 72 and of 40 30, 47; short keys of more
// sequences are on the wrong side: 256 of 300 261, 225).
// One form takes a call, by its average: a prompt among single tokens reads its keys once for every 16 of its rows (95 single
// queries and a prompt of 512, 32 heads on 8, caches of 4096: 445 us; apart 194 and 51).
bool few_queries(const b2g_attention_packed_desc* d, int sms) {
  const int64_t group = d->n_head / d->n_kv_head;
  if (d->total_q > 8 * d->batch && d->total_q * group > kCrRows * d->batch) return false;
  return group > 1 || d->batch * d->n_kv_head < 3ll * sms || d->total_k < 8 * kPtKeys * d->batch;
}

// What a call runs, from its sizes alone.
struct CrPlan {
  bool rows = false;  // chosen_rows (+ chosen_combine), else packed_tiles
  int shares = 0;     // 0: a CTA a tile
  size_t o_bytes = 0, bytes = 0;
};
CrPlan chosen_plan(const b2g_attention_packed_desc* d, int64_t words, int sms) {
  CrPlan r;
  r.rows = d->total_k == 0 || few_queries(d, sms);
  if (!r.rows || d->batch * d->n_kv_head > kCrPairs) return r;
  // A share a CTA, as many as run at the same time; no more than the longest line possible has pieces of kCrMinShare.
  const int64_t tiles = (d->total_q * (d->n_head / d->n_kv_head) / kCrRows + d->batch) * d->n_kv_head;
  const int64_t blocks = d->total_k / kPtKeys + 1, length = 8 * (blocks < 32 * words ? blocks : 32 * words) + kCrTileCost;
  const int64_t most = tiles < (1ll << 30) / length ? (tiles * length + kCrMinShare - 1) / kCrMinShare : 1ll << 30;
  int64_t shares = static_cast<int64_t>(kCrBlocksPerSm) * sms;
  r.shares = static_cast<int>(shares < most ? shares : most);
  r.o_bytes = static_cast<size_t>(round_up(2 * static_cast<int64_t>(r.shares) * kCrRows * d->d_head * 4, 256));
  r.bytes = r.o_bytes + 2 * static_cast<size_t>(r.shares) * kCrRows * sizeof(float2);
  return r;
}

template <typename T, int D>
b2g_status launch_chosen_rows(const PkParams& p, cudaStream_t st) {
  const int64_t items = (static_cast<int64_t>(p.total_q) * p.group / kCrRows + p.batch) * p.hk;
  if (p.shares == 0 && items > (1ll << 31) - 1) return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_blocks: size");
  auto kern = p.shares ? chosen_rows_kernel<T, D, true> : chosen_rows_kernel<T, D, false>;
  b2g_status s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kCrSmem<D>)),
                            "cudaFuncSetAttribute(chosen_rows)");
  if (s != B2G_OK) return s;
  s = launch_pdl(kern, dim3(static_cast<unsigned>(p.shares ? p.shares : items)), dim3(32 * kCrWarps), kCrSmem<D>, st,
                 "chosen_rows launch", p);
  if (s != B2G_OK || p.shares <= 1) return s;
  return launch_pdl(chosen_combine_kernel<T, D>, dim3(static_cast<unsigned>(p.shares - 1)), dim3(kCcThreads), 0, st,
                    "chosen_combine launch", p);
}

template <typename T, int D>
b2g_status run_chosen(const b2g_attention_packed_desc* d, PkParams p, const CrPlan& pl, int sms, cudaStream_t st) {
  if (pl.rows) return launch_chosen_rows<T, D>(p, st);
  CUtensorMap tq, tk, tv;
  b2g_status s;
  if ((s = make_operand_map(&tq, p.q, d->dtype, D, p.total_q, p.ldq, p.hq, p.hsq, kPtRows)) != B2G_OK) return s;
  if ((s = make_operand_map(&tk, p.k, d->dtype, D, p.total_k, p.ldk, p.hk, p.hsk, kPtKeys)) != B2G_OK) return s;
  if ((s = make_operand_map(&tv, p.v, d->dtype, D, p.total_k, p.ldv, p.hk, p.hsv, kPtKeys)) != B2G_OK) return s;
  p.item_heads = 2;
  // A head a CTA where every tile finds an SM of its own (512 tokens of 24 heads 16.1 us against 17.9 with two; twice 512,
  // where they do not, 26.9 and 19.3).
  if ((static_cast<int64_t>(p.total_q) / kPtRows + p.batch) * p.hq <= sms) {
    p.item_heads = 1;
    return launch_tiles<T, D, kHeadsApart, true>(p, tq, tk, tv, sms, st);
  }
  // Two heads of a group have the same blocks and share their stages; others have their own.
  if (p.group % 2 == 0) return launch_tiles<T, D, kHeadsOfGroup, true>(p, tq, tk, tv, sms, st);
  return launch_tiles<T, D, kHeadsApart, true>(p, tq, tk, tv, sms, st);
}

// The checks that the three operators have in common, and the parameters; uses_q: q and cu_q, uses_v: v and out.
b2g_status blocks_params(const b2g_attention_packed_desc* d, const char* who, bool uses_q, bool uses_v, PkParams* p) {
  auto fail = [&](b2g_status st, const char* why) { return set_error(st, std::string(who) + ": " + why); };
  if (!d) return fail(B2G_ERR_INVALID, "null descriptor");
  if (d->batch < 0 || d->total_q < 0 || d->total_k < 0 || d->n_head < 0 || d->n_kv_head < 0)
    return fail(B2G_ERR_INVALID, "negative size");
  if (d->dtype != B2G_BF16 && d->dtype != B2G_F16) return fail(B2G_ERR_UNSUPPORTED, "BF16 or F16 operands");
  if (d->d_head != 64 && d->d_head != 128) return fail(B2G_ERR_UNSUPPORTED, "head dim must be 64 or 128");
  if (uses_q && d->n_head > 0 && (d->n_kv_head < 1 || d->n_head % d->n_kv_head != 0))
    return fail(B2G_ERR_INVALID, "n_head must be a multiple of n_kv_head");
  if (uses_v && (!(d->scale > 0.f) || !std::isfinite(d->scale))) return fail(B2G_ERR_INVALID, "scale must be positive");
  if (d->batch > 65536 || d->total_q > (1ll << 30) || d->total_k > (1ll << 30) || d->n_head > 65535 || d->n_kv_head > 65535)
    return fail(B2G_ERR_UNSUPPORTED, "size");
  const int64_t D = d->d_head;
  p->ldq = used(d->ldq, d->total_q, d->n_head * D); p->hsq = used(d->hsq, d->n_head, D);
  p->ldk = used(d->ldk, d->total_k, d->n_kv_head * D); p->hsk = used(d->hsk, d->n_kv_head, D);
  p->ldv = used(d->ldv, d->total_k, d->n_kv_head * D); p->hsv = used(d->hsv, d->n_kv_head, D);
  p->ldo = used(d->ldo, d->total_q, d->n_head * D); p->hso = used(d->hso, d->n_head, D);
  const bool uses_k = uses_v || !uses_q;
  struct { bool in_use; const void* at; int64_t ld, hs, rows; } ops[4] = {{uses_q, d->q, p->ldq, p->hsq, d->total_q * d->n_head},
                                                                       {uses_k, d->k, p->ldk, p->hsk, d->total_k * d->n_kv_head},
                                                                       {uses_v, d->v, p->ldv, p->hsv, d->total_k * d->n_kv_head},
                                                                       {uses_v, d->out, p->ldo, p->hso, d->total_q * d->n_head}};
  for (const auto& o : ops) {
    if (!o.in_use || o.rows == 0) continue;
    if (!o.at) return fail(B2G_ERR_INVALID, "null operand");
    if (o.ld < D || o.hs < D) return fail(B2G_ERR_INVALID, "a token or head stride is below the head dim");
    if (o.ld % 8 != 0 || o.hs % 8 != 0 || o.ld >= (1ll << 38) || o.hs >= (1ll << 38))
      return fail(B2G_ERR_UNSUPPORTED, "strides must be multiples of 8 elements");
    if (reinterpret_cast<uintptr_t>(o.at) & 15u) return fail(B2G_ERR_UNSUPPORTED, "16-byte aligned operands required");
  }
  if (d->batch > 0 && (!d->cu_k || (uses_q && !d->cu_q))) return fail(B2G_ERR_INVALID, "null operand");
  p->cu_q = d->cu_q; p->cu_k = d->cu_k; p->k_lens = d->k_lens;
  p->batch = static_cast<int>(d->batch);
  p->total_q = static_cast<int>(d->total_q); p->total_k = static_cast<int>(d->total_k);
  p->hq = d->n_head; p->hk = d->n_kv_head; p->group = uses_q && d->n_kv_head > 0 ? d->n_head / d->n_kv_head : 1;
  p->causal = d->causal ? 1 : 0;
  p->scale_log2 = d->scale * 1.4426950408889634f;
  p->q = d->q; p->k = d->k; p->v = d->v; p->out = d->out;
  return B2G_OK;
}

}  // namespace

b2g_status block_means(const b2g_attention_packed_desc* d, const int32_t* since, float* means, int64_t blocks,
                       cudaStream_t st) {
  MnParams a{};
  b2g_status s = blocks_params(d, "b2g_block_means", false, false, &a.p);
  if (s != B2G_OK) return s;
  if (blocks < 0) return set_error(B2G_ERR_INVALID, "b2g_block_means: negative size");
  if (blocks == 0 || d->n_kv_head == 0) return B2G_OK;
  if (!means) return set_error(B2G_ERR_INVALID, "b2g_block_means: null operand");
  if (reinterpret_cast<uintptr_t>(means) & 15u)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_block_means: 16-byte aligned operands required");
  if (blocks > (1ll << 30)) return set_error(B2G_ERR_UNSUPPORTED, "b2g_block_means: size");
  if (since && d->batch == 0) return B2G_OK;
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  a.since = since;
  a.means = means;
  a.blocks = static_cast<int>(blocks);
  a.D = d->d_head;
  const int64_t parts = (static_cast<int64_t>(d->n_kv_head) * d->d_head + kMnCols - 1) / kMnCols;
  if (parts > 65535) return set_error(B2G_ERR_UNSUPPORTED, "b2g_block_means: size");
  int64_t z = 1;
  if (since) {  // as many blocks of a sequence side by side as the SMs have room for
    z = 2ll * dev->num_sms / (d->batch * parts);
    z = z < 1 ? 1 : z > blocks ? blocks : z;
    if (z > 65535) z = 65535;
  }
  const dim3 grid(static_cast<unsigned>(since ? d->batch : blocks), static_cast<unsigned>(parts), static_cast<unsigned>(z));
  const dim3 block(32 * kMnWarps);
  if (d->dtype == B2G_F16) return launch_pdl(block_means_kernel<__half>, grid, block, 0, st, "block_means launch", a);
  return launch_pdl(block_means_kernel<__nv_bfloat16>, grid, block, 0, st, "block_means launch", a);
}

b2g_status select_blocks(const b2g_attention_packed_desc* d, const float* means, int64_t blocks, int64_t top, int64_t first,
                         int64_t last, int32_t* chosen, int64_t tiles, int64_t words, cudaStream_t st) {
  SlParams a{};
  b2g_status s = blocks_params(d, "b2g_select_blocks", true, false, &a.p);
  if (s != B2G_OK) return s;
  if (blocks < 0 || tiles < 0 || words < 0 || top < 0 || first < 0 || last < 0)
    return set_error(B2G_ERR_INVALID, "b2g_select_blocks: negative size");
  if (tiles == 0 || words == 0 || d->n_kv_head == 0) return B2G_OK;
  if (!chosen || (blocks > 0 && !means)) return set_error(B2G_ERR_INVALID, "b2g_select_blocks: null operand");
  if (words > kSlMostWords) return set_error(B2G_ERR_UNSUPPORTED, "b2g_select_blocks: at most 2^20 keys a sequence");
  if ((reinterpret_cast<uintptr_t>(means) & 15u) || (reinterpret_cast<uintptr_t>(chosen) & 3u))
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_select_blocks: 16-byte aligned means required");
  if (blocks > (1ll << 30) || tiles * d->n_kv_head > (1ll << 31) - 1)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_select_blocks: size");
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  const int64_t most = 32 * words;  // (more of them take every block just the same)
  a.means = means;
  a.blocks = static_cast<int>(blocks);
  a.top = static_cast<int>(top < most ? top : most);
  a.first = static_cast<int>(first < most ? first : most);
  a.last = static_cast<int>(last < most ? last : most);
  a.chosen = reinterpret_cast<uint32_t*>(chosen);
  a.tiles = static_cast<int>(tiles);
  a.words = static_cast<int>(words);
  // Four tiles a CTA, which share the means, where that leaves CTAs for all SMs and their scores fit.  (24 heads, us, one and
  // four: 16384 tokens 62.5, 46.0; 4096 16.1, 16.6; 2048 10.5, 12.5; 16 x 512 22.7, 21.4; 32 x 300 28.8, 30.9)
  const bool four = tiles / 4 * d->n_kv_head >= dev->num_sms && d->total_q >= 512 * d->batch && words <= kSlMostWords / 4;
  auto run = [&](auto kern, int nt) {
    const size_t sums = static_cast<size_t>(nt) * kSlThreads / 32 * (d->d_head + 4) * 8, smem = sums + static_cast<size_t>(nt) * words * 32 * 8;
    b2g_status st2 = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 100 * 1024),
                                "cudaFuncSetAttribute(select_blocks)");
    return st2 != B2G_OK ? st2
                         : launch_pdl(kern, dim3(static_cast<unsigned>((tiles + nt - 1) / nt * d->n_kv_head)), dim3(kSlThreads), smem, st,
                                      "select_blocks launch", a);
  };
  auto pick = [&](auto type) {
    using T = decltype(type);
    if (d->d_head == 128) return four ? run(select_blocks_kernel<T, 128, 4>, 4) : run(select_blocks_kernel<T, 128, 1>, 1);
    return four ? run(select_blocks_kernel<T, 64, 4>, 4) : run(select_blocks_kernel<T, 64, 1>, 1);
  };
  return d->dtype == B2G_F16 ? pick(__half()) : pick(__nv_bfloat16());
}

size_t attention_blocks_workspace(const b2g_attention_packed_desc* d, int64_t words) {
  PkParams p{};
  DeviceInfo* dev = nullptr;
  if (blocks_params(d, "b2g_attention_blocks_workspace", true, true, &p) != B2G_OK || words < 0 || words > (1ll << 20) ||
      d->batch == 0 || d->total_q == 0 || d->n_head == 0 || device_info(&dev) != B2G_OK)
    return 0;
  return chosen_plan(d, words, dev->num_sms).bytes;
}

b2g_status attention_blocks(const b2g_attention_packed_desc* d, const int32_t* chosen, int64_t tiles, int64_t words,
                            void* workspace, size_t workspace_bytes, cudaStream_t st) {
  PkParams p{};
  b2g_status s = blocks_params(d, "b2g_attention_blocks", true, true, &p);
  if (s != B2G_OK) return s;
  if (tiles < 0 || words < 0) return set_error(B2G_ERR_INVALID, "b2g_attention_blocks: negative size");
  if (d->batch == 0 || d->total_q == 0 || d->n_head == 0) return B2G_OK;
  if (tiles > 0 && words > 0 && !chosen) return set_error(B2G_ERR_INVALID, "b2g_attention_blocks: null operand");
  if (reinterpret_cast<uintptr_t>(chosen) & 3u)
    return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_blocks: 4-byte aligned words required");
  if (tiles > (1ll << 30) || words > (1ll << 20)) return set_error(B2G_ERR_UNSUPPORTED, "b2g_attention_blocks: size");
  DeviceInfo* dev = nullptr;
  if ((s = device_info(&dev)) != B2G_OK) return s;
  p.chosen = reinterpret_cast<const uint32_t*>(chosen);
  p.chosen_tiles = words > 0 ? static_cast<int>(tiles) : 0;
  p.chosen_words = static_cast<int>(words);
  p.err = dev->err_word;
  const CrPlan pl = chosen_plan(d, words, dev->num_sms);
  void* ws = workspace;
  if (pl.bytes > 0) {
    if (!ws && (s = workspace_get(pl.bytes, &ws, kWsAttnSplit)) != B2G_OK) return s;
    if (workspace && (workspace_bytes < pl.bytes || (reinterpret_cast<uintptr_t>(workspace) & 255u)))
      return set_error(B2G_ERR_INVALID, "b2g_attention_blocks: the workspace is too small or not 256-byte aligned");
  }
  p.shares = pl.shares;
  p.part_o = static_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(static_cast<char*>(ws) + pl.o_bytes);
  const int sms = dev->num_sms;
  if (d->dtype == B2G_F16)
    return d->d_head == 128 ? run_chosen<__half, 128>(d, p, pl, sms, st) : run_chosen<__half, 64>(d, p, pl, sms, st);
  return d->d_head == 128 ? run_chosen<__nv_bfloat16, 128>(d, p, pl, sms, st)
                          : run_chosen<__nv_bfloat16, 64>(d, p, pl, sms, st);
}

}  // namespace b2g
