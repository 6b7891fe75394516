// attention_packed.cuh — what the attentions over packed sequences share: offsets and searches, the tile
// kernel for long queries over all keys or over chosen key blocks, 16-row products and copies.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cmath>
#include <cstdint>
#include <type_traits>
#include "engine.cuh"
#include "ptx_sm100.cuh"

namespace b2g {

namespace {

struct PkParams {
  const int* cu_q;
  const int* cu_k;
  const int* k_lens;       // [batch] or NULL
  int batch;
  int total_q, total_k;    // rows of q and of k, v
  int hq, hk, group;       // query heads, key heads, hq / hk
  int item_heads;          // kHeadsApart: heads per work item, 1 or 2
  int causal;
  float scale_log2;        // scale * log2(e)
  const void *q, *k, *v;
  long long ldq, hsq, ldk, hsk, ldv, hsv;  // token and head strides, elements
  void* out;
  long long ldo, hso;
  int* err;
  // packed_rows
  int shares;              // most shares that the work is cut into
  float* part_o;           // [slot][16][D]
  float2* part_ml;         // [slot][16]: row maximum (log2 units), row sum
  // chosen key blocks (attention_blocks.cu): bit j % 32 of word j / 32 of (tile of 128 queries, key head)
  const uint32_t* chosen;
  int chosen_tiles, chosen_words;
};

// Rows of sequence b, clamped to the buffers.
struct Seq {
  int q0, lq, k0, lk;
};
__device__ __forceinline__ int clampi(int v, int lo, int hi) { return min(max(v, lo), hi); }
__device__ __forceinline__ Seq load_seq(const PkParams& p, int b) {
  Seq s;
  s.q0 = clampi(__ldg(p.cu_q + b), 0, p.total_q);
  s.lq = clampi(__ldg(p.cu_q + b + 1), s.q0, p.total_q) - s.q0;
  s.k0 = clampi(__ldg(p.cu_k + b), 0, p.total_k);
  s.lk = clampi(__ldg(p.cu_k + b + 1), s.k0, p.total_k) - s.k0;
  if (p.k_lens) s.lk = clampi(__ldg(p.k_lens + b), 0, s.lk);
  return s;
}
// A lane's sum of sequences' tiles or blocks.  Rising offsets give at most 2^30 / 128 + 65536; those that jump back and forth
// count rows again and again, and their sum stops where 32 lanes' sums and a sequence's blocks still fit 32 bits: what such a sum
// is compared with (rows of `means`, of `chosen`) then bounds it, as no wrapped one could be.
__device__ __forceinline__ int add_count(int sum, int n) { return min(sum + n, 1 << 25); }

// The sequence that holds unit `want` when sequence b holds count(b) units, and the number of units
// before it; -1 if there are not so many.  A whole warp searches, 32 sequences at a time, from
// sequence `first` on, before which there are *before units.
template <typename I, typename Count>
__device__ __forceinline__ int find_seq(int batch, I want, int lane, Count count, I* before, int first = 0) {
  I base = *before;
  for (int b0 = first; b0 < batch; b0 += 32) {
    const int b = b0 + lane;
    const I n = b < batch ? count(b) : 0;
    I sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const I up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    const uint32_t past = __ballot_sync(0xffffffffu, base + sum > want);
    if (past) {
      const int at = __ffs(past) - 1;
      *before = base + __shfl_sync(0xffffffffu, sum - n, at);
      return b0 + at;
    }
    base += __shfl_sync(0xffffffffu, sum, 31);
  }
  return -1;
}

// A shared-memory int read afresh at every use, so that it occupies no register in between.
__device__ __forceinline__ int ld_shared_int(const int* p) {
  int v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(smem_u32(p)) : "memory");
  return v;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
    __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  } else {
    __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&h);
  }
}

// ---------------------------------------------------------------------------- long queries
//
// A persistent CTA per SM works on two 128-row query tiles at a time, in one of three ways:
//   kTilesOfHead   consecutive tiles of one head, which share the keys' shared-memory stages
//   kHeadsOfGroup  the same rows of two query heads that share a key head: shared stages, finer steps
//   kHeadsApart    the same rows of two heads with their own keys: twice the key traffic, but no idle
//                  second tile where sequences are short; or of one head, where there are few tiles
// Roles: warp 3 finds the work items and hands them round in a ring, warp 0 loads Q and K, warp 2 V, one
// thread of warp 1 issues the MMAs, warps 4-7 and 8-11 are the softmax of tiles A and B with one thread
// per row.  S (fp32) and O live in TMEM, P (16-bit) overwrites S and is the A operand of P.V.  Per key
// block j, for A then B:
//   O += P(j) V_j, S(j+1)
// so the tensor core works for one tile while the other's softmax runs.  The roles run through the
// work items without stopping: S of the next item's first block is issued behind the last P.V, Q, K and V
// are loaded ahead as their stages come free, and only the tile's own softmax warps pause to write O.
// (With a CTA per item, its start and end cost 8 us beside 2.3 us per key block.)
//
// Bound by the chain of a tile: S, softmax (128 exponentials a row on 16 units a clock and SM), P.V; with
// two tiles in turn the tensor core is busy some 60 % of the time at d = 128, 35 % at d = 64, whose
// products take half as long beside the same softmax.  d = 128, 24 heads, sequences of 4608: 1050 TFLOP/s; 7
// images of 300 to 4608: 700 us.  Short sequences pay for whole 128 x 128 blocks, of which a
// sequence of 1 to 509 tokens sees half, and for what a tile costs once (at d = 64 1.35 us an SM, beside 0.81 us per key
// block: 96 sequences of 128 and of 256 tokens take 90 and 247 us): 96 of them, 64 heads of 64: 228 us; 40 causal prompts
// of 1 to 2047: 206 us.
//
// Items that see no key (causal rows before the first key, empty caches) are written as zeros by warp 3 and stay
// out of the ring: the MMA thread looks one item ahead, and so many in a row that the ring ends before the next one
// with keys would leave it waiting for a place that its own tile holds.
//
// Items: sequences by falling key count (up to kPtSorted of them; else as they come), tiles from the
// last, which see most keys; dealt to the CTAs back and forth.  That evens out many short sequences without a mask (96 short
// prompts: the busiest CTA has 140 tile blocks, the mean is 139), a few long ones less (7 images: 604, 562).  Causal tiles
// fall from many blocks to one within each sequence, so that the order is not by size (40 causal prompts: 148, 120).
//
// The last key block may reach into the next sequence's rows, whose values may be anything: those
// scores are replaced by -inf, and those rows of V are zeroed in shared memory before the MMA
// reads them (0 times a NaN would be a NaN).  Within a sequence, V is expected to be finite: a
// non-finite row of V reaches the query rows of its tile that do not see it.
constexpr int kPtThreads = 384;
constexpr int kPtRegsIdle = 88;      // producers and MMA issuer
constexpr int kPtRegsSoftmax = 208;  // a 128-key row of scores in registers
static_assert(4 * 32 * kPtRegsIdle + 8 * 32 * kPtRegsSoftmax <= kPtThreads * 168, "register split");
constexpr int kPtRows = 128;
constexpr int kPtKeys = 128;
constexpr uint32_t kPtBox = 128 * 128;  // bytes of one 128-row x 128-byte swizzled box
constexpr float kPtRescaleLog2 = 8.0f;
constexpr int kPtSorted = 512;
constexpr int kPtItems = 4;      // items in the ring
constexpr int kPtReaders = 11;   // Q/K, V, MMA, 8 softmax warps
enum { kTilesOfHead = 0, kHeadsOfGroup = 1, kHeadsApart = 2 };

template <int D>
struct PtLayout {
  static constexpr int KS = D == 128 ? 2 : 6, VS = D == 128 ? 2 : 4;
  static constexpr uint32_t kTileBytes = 128 * D * 2;  // Q tile, K block, V block: D / 64 boxes
  static constexpr uint32_t kQ = 0;
  static constexpr uint32_t kK = kQ + 2 * kTileBytes;
  static constexpr uint32_t kV = kK + KS * kTileBytes;
  static constexpr uint32_t kOut = kV + VS * kTileBytes;   // 32 rows x 64 columns of output per softmax warp
  static constexpr uint32_t kBars = kOut + 8 * 4096;
  static constexpr uint32_t kOrder = kBars + 384;      // sequences in working order, uint16 [kPtSorted]
  static constexpr uint32_t kItems = kOrder + 2 * kPtSorted;
  static constexpr uint32_t kSmem = 1024 + kItems + 32 * kPtItems;
  static constexpr uint32_t kSmemChosen = 1024 + kItems + 64 * kPtItems;
};

// One work item: rows [row0, row0 + 128) of tile A and B (B's 128 further on in kTilesOfHead).
struct PtItem {
  int q0, lq, k0, lk;
  int row0, head;  // of tile A; head -1: no more items
  int blocks[2];   // key blocks of each tile (0: nothing to see, or no rows)
};
static_assert(sizeof(PtItem) == 32, "two 16-byte words");
// The same with chosen key blocks: its row of `chosen`, and per tile how many of its blocks, the first ones,
// are seen whole by every row; the others, two at most, are part_block and its neighbour.
struct PtChosenItem : PtItem {
  int tile;
  int whole[2], part_block[2];
  int unused[3];
};
static_assert(sizeof(PtChosenItem) == 64, "four 16-byte words");

// The set bits of a row of `chosen`, in order.  (Past the last word, which a row changed under the kernel could
// reach, it gives block 0.)
struct ChosenWalk {
  const uint32_t* words;
  int at, end;
  uint32_t bits;
  __device__ __forceinline__ void start(const PkParams& p, int tile, int kv_head) {
    words = p.chosen + (static_cast<long long>(tile) * p.hk + kv_head) * p.chosen_words;
    at = -1;
    end = p.chosen_words;
    bits = 0;
  }
  __device__ __forceinline__ int next() {
    while (bits == 0) {
      if (++at >= end) return 0;
      bits = __ldg(words + at);
    }
    const int j = at * 32 + __ffs(bits) - 1;
    bits &= bits - 1;
    return j;
  }
};

// A place in a ring of n stages: the stage and the parity of its use.
template <int n>
struct Turn {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next() {
    if (++stage == n) {
      stage = 0;
      parity ^= 1u;
    }
  }
  __device__ __forceinline__ void back() {
    if (stage-- == 0) {
      stage = n - 1;
      parity ^= 1u;
    }
  }
};

template <typename T, int D, int kMode, bool kChosen = false>
__global__ void __launch_bounds__(kPtThreads, 1)
    packed_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const PkParams p) {
  using Ly = PtLayout<D>;
  constexpr int KS = Ly::KS, VS = Ly::VS;
  constexpr bool kApart = kMode == kHeadsApart;
  static_assert(!kChosen || kMode != kTilesOfHead, "two tiles of a head choose blocks of their own");
  using Item = std::conditional_t<kChosen, PtChosenItem, PtItem>;
  constexpr uint32_t kFmt = std::is_same<T, __half>::value ? kFmtF16 : kFmtBF16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sQ = smem + Ly::kQ;
  uint8_t* sK = smem + Ly::kK;
  uint8_t* sV = smem + Ly::kV;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + Ly::kBars);
  uint64_t* q_full = bars;          // [tile] Q landed
  uint64_t* q_empty = bars + 2;     // [tile] the item's last S is computed
  uint64_t* s_full = bars + 4;      // [tile] S computed
  uint64_t* p_part = bars + 6;      // [tile] P of keys 0-95 written (4 softmax warps)
  uint64_t* p_full = bars + 8;      // [tile] all of P written
  uint64_t* pv_done = bars + 10;    // [tile] P.V added
  uint64_t* o_empty = bars + 12;    // [tile] O read (4 softmax warps)
  uint64_t* drain_bar = bars + 14;
  uint64_t* k_full = bars + 15;
  uint64_t* k_empty = k_full + KS;
  uint64_t* v_full = k_empty + KS;
  uint64_t* v_empty = v_full + VS;
  uint64_t* v_land = v_empty + VS;  // V blocks whose rows past the keys in sight are still to be zeroed
  uint64_t* item_full = v_land + VS;
  uint64_t* item_empty = item_full + kPtItems;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(item_empty + kPtItems);
  static_assert(8 * (15 + 2 * KS + 3 * VS + 2 * kPtItems) + 4 <= 384, "barriers");
  Item* items = reinterpret_cast<Item*>(smem + Ly::kItems);
  uint16_t* order = reinterpret_cast<uint16_t*>(smem + Ly::kOrder);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0 && lane == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&q_full[t], 1);
      mbar_init(&q_empty[t], 1);
      mbar_init(&s_full[t], 1);
      mbar_init(&p_part[t], 4);
      mbar_init(&p_full[t], 4);
      mbar_init(&pv_done[t], 1);
      mbar_init(&o_empty[t], 4);
    }
    mbar_init(drain_bar, 1);
    for (int i = 0; i < kPtItems; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], kPtReaders);
    }
    for (int i = 0; i < KS; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
    }
    for (int i = 0; i < VS; ++i) {
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
      mbar_init(&v_land[i], 1);
    }
    fence_mbar_init();
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  griddep_wait();  // the set-up above overlapped the previous kernel's tail
  griddep_launch_dependents();
  const bool sorted = p.batch <= kPtSorted;
  if (sorted) {
    // Rank of each sequence by its keys (the counts pass through Q's space, still unused).
    int* count = reinterpret_cast<int*>(sQ);
    for (int b = threadIdx.x; b < p.batch; b += kPtThreads) count[b] = load_seq(p, b).lk;
    __syncthreads();
    for (int b = threadIdx.x; b < p.batch; b += kPtThreads) {
      int rank = 0;
      for (int i = 0; i < p.batch; ++i) rank += count[i] > count[b] || (count[i] == count[b] && i < b);
      order[rank] = static_cast<uint16_t>(b);
    }
    fence_proxy_async_smem();  // (Q arrives there by the async proxy)
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  constexpr int kSpan = kMode == kTilesOfHead ? 2 * kPtRows : kPtRows;  // sequence rows per item
  // Keys that either tile sees: V rows from there on are zeroed.
  auto keys_seen = [&](const Item& w) {
    const int last = w.row0 + (kMode == kTilesOfHead && w.blocks[1] > 0 ? 2 : 1) * kPtRows;
    return p.causal ? clampi(min(last, w.lq) + w.lk - w.lq, 0, w.lk) : w.lk;
  };

  auto wait = [&](uint64_t* bar, uint32_t parity, int code) { return mbar_wait_short(bar, parity, p.err, code); };
  if (warp < 4) {
    regs_dec<kPtRegsIdle>();
    if (warp == 3) {
      // ---------------------------------------------------------- work items
      const int item_heads = kApart ? p.item_heads : kMode == kTilesOfHead ? 1 : 2;
      const int head_units = (p.hq + item_heads - 1) / item_heads;
      const int most_units = p.total_q / kSpan + p.batch;  // (offsets that jump back and forth have more: they end here)
      const int grid = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
      int units_before = 0, i = 0;
      [[maybe_unused]] int tiles_of = -1, tiles_before = 0;  // kChosen: tiles in front of sequence tiles_of
      Turn<kPtItems> at;
      for (int round = 0; i >= 0; ++round) {
        const long long index = static_cast<long long>(round) * grid + (round & 1 ? grid - 1 - cta : cta);
        const int unit = static_cast<int>(index / head_units);
        const int head_unit = static_cast<int>(index - static_cast<long long>(unit) * head_units);
        auto seq_of = [&](int j) { return sorted ? static_cast<int>(order[j]) : j; };
        i = unit >= most_units ? -1 : find_seq(p.batch, unit, lane, [&](int j) {
          const int b = seq_of(j), lo = clampi(__ldg(p.cu_q + b), 0, p.total_q);
          return (clampi(__ldg(p.cu_q + b + 1), lo, p.total_q) - lo + kSpan - 1) / kSpan;
        }, &units_before, i);
        Item w{};
        w.head = -1;
        if (i >= 0) {
          const Seq s = load_seq(p, seq_of(i));
          if constexpr (kChosen) {
            if (tiles_of != seq_of(i)) {
              tiles_of = seq_of(i);
              int sum = 0;
              for (int b = lane; b < tiles_of; b += 32) {
                const int lo = clampi(__ldg(p.cu_q + b), 0, p.total_q);
                sum = add_count(sum, (clampi(__ldg(p.cu_q + b + 1), lo, p.total_q) - lo + kPtRows - 1) / kPtRows);
              }
              tiles_before = __reduce_add_sync(0xffffffffu, sum);
            }
          }
          w.q0 = s.q0;
          w.lq = s.lq;
          w.k0 = s.k0;
          w.lk = s.lk;
          w.row0 = ((s.lq + kSpan - 1) / kSpan - 1 - (unit - units_before)) * kSpan;
          w.head = item_heads * head_unit;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int row = w.row0 + (kMode == kTilesOfHead ? t * kPtRows : 0);
            int n = row < s.lq && (!kApart || (t < item_heads && w.head + t < p.hq)) ? s.lk : 0;
            if (p.causal) n = clampi(min(row + kPtRows, s.lq) + s.lk - s.lq, 0, n);
            w.blocks[t] = (n + kPtKeys - 1) / kPtKeys;
            if constexpr (kChosen) {
              w.tile = tiles_before + w.row0 / kPtRows;
              const int nb = w.tile < p.chosen_tiles ? min(w.blocks[t], 32 * p.chosen_words) : 0;
              const uint32_t* words =
                  p.chosen + (static_cast<long long>(w.tile) * p.hk + min((w.head + t) / p.group, p.hk - 1)) * p.chosen_words;
              int count = 0;
              for (int i = lane; 32 * i < nb; i += 32) {
                const uint32_t bits = __ldg(words + i);
                count += __popc(nb - 32 * i >= 32 ? bits : bits & ((1u << (nb - 32 * i)) - 1u));
              }
              w.blocks[t] = __reduce_add_sync(0xffffffffu, count);
              const int whole = (p.causal ? clampi(row + 1 + s.lk - s.lq, 0, s.lk) : s.lk) / kPtKeys;
              auto taken = [&](int j) { return j < nb && ((__ldg(words + (j >> 5)) >> (j & 31)) & 1u) != 0; };
              const int first = taken(whole), second = taken(whole + 1);
              w.whole[t] = w.blocks[t] - first - second;
              w.part_block[t] = first ? whole : whole + 1;
            }
          }
          if ((w.blocks[0] | w.blocks[1]) == 0) {
            // Rows that see no key are 0, written here: no other role has to find its way past such items.
            const int rows = min(s.lq - w.row0, kSpan), heads = min(item_heads, p.hq - w.head);
            T* to = static_cast<T*>(p.out) + static_cast<long long>(s.q0 + w.row0) * p.ldo +
                    static_cast<long long>(w.head) * p.hso;
            for (int h = 0; h < heads; ++h, to += p.hso)
              for (int x = lane; x < rows * (D / 8); x += 32)
                *reinterpret_cast<uint4*>(to + static_cast<long long>(x / (D / 8)) * p.ldo + x % (D / 8) * 8) =
                    make_uint4(0, 0, 0, 0);
            continue;
          }
        }
        bool ok = true;
        if (lane == 0) {
          ok = mbar_wait_short(&item_empty[at.stage], at.parity ^ 1u, p.err, kErrWaitProducer);
          if (ok) {
            items[at.stage] = w;
            mbar_arrive(&item_full[at.stage]);
          }
        }
        if (!__shfl_sync(0xffffffffu, ok, 0)) break;
        at.next();
      }
    } else if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- Q and K
      const uint64_t shared_kv = policy_evict_last(), once = policy_evict_first();
      Turn<kPtItems> at;
      Turn<KS> k_at;
      uint32_t q_parity[2] = {0, 0};
      int k_used = 0;
      bool ok = true, q_used[2] = {false, false};
      for (; ok; at.next()) {
        if (!(ok = mbar_wait_short(&item_full[at.stage], at.parity, p.err, kErrWaitProducer))) break;
        const Item w = items[at.stage];
        mbar_arrive(&item_empty[at.stage]);
        if (w.head < 0) break;
        const int nkb = max(w.blocks[0], w.blocks[1]);
        const int kv_head = w.head / p.group, kv_head_b = kApart ? (w.head + 1) / p.group : kv_head;
        ChosenWalk walk[kApart ? 2 : 1];
        if constexpr (kChosen) {
          walk[0].start(p, w.tile, kv_head);
          if constexpr (kApart) walk[1].start(p, w.tile, kv_head_b);
        }
        for (int j = 0; j < nkb && ok; ++j) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && j == 0 && w.blocks[t] > 0) {  // this tile's Q
              ok = mbar_wait_short(&q_empty[t], q_parity[t] ^ 1u, p.err, kErrWaitProducer);
              if (!ok) break;
              q_parity[t] ^= 1u;
              q_used[t] = true;
              mbar_arrive_expect_tx(&q_full[t], Ly::kTileBytes);
#pragma unroll
              for (int c = 0; c < D / 64; ++c)
                tma_load_3d(sQ + t * Ly::kTileBytes + c * kPtBox, &tmQ, &q_full[t], c * 64,
                            w.q0 + w.row0 + (kMode == kTilesOfHead ? t * kPtRows : 0),
                            w.head + (kMode == kTilesOfHead ? 0 : t), once);
            }
            if (kApart ? j >= w.blocks[t] : t != 0) continue;
            ok = mbar_wait_short(&k_empty[k_at.stage], k_at.parity ^ 1u, p.err, kErrWaitProducer);
            if (!ok) break;
            int block = j;
            if constexpr (kChosen) block = walk[kApart ? t : 0].next();
            mbar_arrive_expect_tx(&k_full[k_at.stage], Ly::kTileBytes);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_3d(sK + k_at.stage * Ly::kTileBytes + c * kPtBox, &tmK, &k_full[k_at.stage], c * 64,
                          w.k0 + block * kPtKeys, t ? kv_head_b : kv_head, shared_kv);
            k_at.next();
            ++k_used;
          }
        }
      }
      // This thread's copies land before the CTA's shared memory goes away (they have, unless
      // another role gave up early).
      for (int t = 0; t < 2; ++t)
        if (q_used[t]) mbar_wait_drain(&q_full[t], q_parity[t] ^ 1u);
      for (int i = min(k_used, KS); i > 0; --i) {
        k_at.back();
        mbar_wait_drain(&k_full[k_at.stage], k_at.parity);
      }
    } else if (warp == 2) {
      // ---------------------------------------------------------- V
      // A block that reaches past the keys in sight lands on v_land; its rows from there on are zeroed
      // before it is passed to the MMAs.  Loads go out ahead of that while stages are free.
      const uint64_t shared_kv = policy_evict_last();
      Turn<kPtItems> at;
      Turn<VS> v_at, tail_at;
      Item w{};
      int seen = 0;
      ChosenWalk walk[kApart ? 2 : 1];
      auto nkb = [](const Item& i) { return max(i.blocks[0], i.blocks[1]); };
      int key = 0, t = 0;              // the next load: this block of the item, and head
      bool have = false, more = true;  // there is a next load; there may be more items
      int used = 0;
      uint32_t tails = 0;              // a byte per stage: rows to keep of an unfinished tail (0: none)
      uint32_t land_parity = 0;        // bit per stage
      auto ready = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_test_wait(smem_u32(bar), parity)); };
      bool ok = true;
#pragma unroll 1
      while (ok) {
        if (!have && more && (tails == 0 || ready(&item_full[at.stage], at.parity))) {
          ok = __all_sync(0xffffffffu, wait(&item_full[at.stage], at.parity, kErrWaitProducer));
          if (!ok) break;
          w = items[at.stage];
          __syncwarp();
          more = w.head >= 0;
          if (more && lane == 0) mbar_arrive(&item_empty[at.stage]);
          at.next();
          key = 0;
          t = kApart && w.blocks[0] == 0 ? 1 : 0;
          seen = keys_seen(w);
          if constexpr (kChosen) {
            walk[0].start(p, w.tile, max(w.head, 0) / p.group);
            if constexpr (kApart) walk[1].start(p, w.tile, (w.head + 1) / p.group);
          }
          have = more;
          continue;
        }
        if (have && (tails == 0 || ready(&v_empty[v_at.stage], v_at.parity ^ 1u))) {
          const int st = v_at.stage;
          ok = __all_sync(0xffffffffu, wait(&v_empty[st], v_at.parity ^ 1u, kErrWaitProducer));
          if (!ok) break;
          int from = key;
          if constexpr (kChosen) from = (kApart && t ? walk[kApart].next() : walk[0].next()) * kPtKeys;
          // Rows of this block that are seen (chosen blocks begin in sight; no row of `chosen` makes it 0).
          const int valid = kChosen ? max(seen - from, 1) : seen - from;
          if (lane == 0) {
            uint64_t* bar = valid < kPtKeys ? &v_land[st] : &v_full[st];
            mbar_arrive_expect_tx(bar, Ly::kTileBytes);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_3d(sV + st * Ly::kTileBytes + c * kPtBox, &tmV, bar, c * 64, w.k0 + from, (w.head + t) / p.group,
                          shared_kv);
          }
          if (valid < kPtKeys) tails |= static_cast<uint32_t>(valid) << (8 * st);
          v_at.next();
          ++used;
          if (kApart && t == 0 && key < w.blocks[1] * kPtKeys) t = 1;
          else {
            key += kPtKeys;
            t = kApart && key >= w.blocks[0] * kPtKeys ? 1 : 0;
            have = key < nkb(w) * kPtKeys;
          }
          continue;
        }
        if (tails == 0) break;  // nothing left to do
        const uint32_t valid = (tails >> (8 * tail_at.stage)) & 0xFFu;
        if (valid) {  // the oldest tail
          const int st = tail_at.stage;
          ok = __all_sync(0xffffffffu, wait(&v_land[st], (land_parity >> st) & 1u, kErrWaitProducer));
          if (!ok) break;
          land_parity ^= 1u << st;
          const int zeros = kPtKeys - static_cast<int>(valid);
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            uint4* z = reinterpret_cast<uint4*>(sV + st * Ly::kTileBytes + c * kPtBox + valid * 128);
            for (int i = lane; i < zeros * 8; i += 32) z[i] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_full[st]);
          tails &= ~(0xFFu << (8 * st));
        }
        tail_at.next();
      }
      if (lane == 0) {
        // Loads of an abandoned run land before the shared memory goes away.
#pragma unroll 1
        for (int i = min(used, VS); i > 0; --i) {
          v_at.back();
          if ((tails >> (8 * v_at.stage)) & 0xFFu) mbar_wait_drain(&v_land[v_at.stage], (land_parity >> v_at.stage) & 1u);
          else mbar_wait_drain(&v_full[v_at.stage], v_at.parity);
        }
      }
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------- MMA issuer
      constexpr uint32_t idesc_s = idesc_make(kFmt, kPtRows, kPtKeys);
      constexpr uint32_t idesc_o = idesc_make(kFmt, kPtRows, D) | kIdescBMajorMN;
      Turn<kPtItems> at;
      Turn<KS> k_at;
      Turn<VS> v_at;
      // Parities of the tiles' barriers: q_full, P (one use per block), o_empty.
      uint32_t q_parity[2] = {0, 0}, p_parity[2] = {0, 0}, o_parity[2] = {0, 0};
      bool ok = true;
      // The next item's blocks; no more items: blocks 0, 0.
      auto next_blocks = [&](int (&blocks)[2]) {
        blocks[0] = blocks[1] = 0;
        if (!(ok = mbar_wait_short(&item_full[at.stage], at.parity, p.err, kErrWaitMma))) return;
        if (ld_shared_int(&items[at.stage].head) < 0) return;  // (not handed back: asked again, it says the same)
        blocks[0] = ld_shared_int(&items[at.stage].blocks[0]);
        blocks[1] = ld_shared_int(&items[at.stage].blocks[1]);
        mbar_arrive(&item_empty[at.stage]);
        at.next();
      };
      // S of the key block at k_at, of tile t; first: of its item (Q), last: Q is free afterwards.
      auto issue_s = [&](int t, bool first, bool last) {
        if (first) {
          if (!(ok = mbar_wait_short(&q_full[t], q_parity[t], p.err, kErrWaitMma))) return;
          q_parity[t] ^= 1u;
        }
        if (!(ok = mbar_wait_short(&k_full[k_at.stage], k_at.parity, p.err, kErrWaitMma))) return;
        tc_fence_after();
        const uint32_t q0 = smem_u32(sQ + t * Ly::kTileBytes), k0 = smem_u32(sK + k_at.stage * Ly::kTileBytes);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f16(tmem + t * 256, smem_desc_k_sw128(q0 + c * kPtBox + k * 32),
                     smem_desc_k_sw128(k0 + c * kPtBox + k * 32), idesc_s, (c | k) != 0 ? 1u : 0u);
        umma_commit(&s_full[t]);
        if (last) umma_commit(&q_empty[t]);
        if constexpr (kApart) {
          umma_commit(&k_empty[k_at.stage]);
          k_at.next();
        }
      };
      int cur[2], then[2];
      next_blocks(cur);
      for (int t = 0; t < 2; ++t)
        if (ok && cur[t] > 0) issue_s(t, true, cur[t] == 1);
      if (!kApart && ok && (cur[0] | cur[1]) != 0) {
        umma_commit(&k_empty[k_at.stage]);
        k_at.next();
      }
      while (ok && (cur[0] | cur[1]) != 0) {
        const int nkb = max(cur[0], cur[1]);
        for (int j = 0; j < nkb && ok; ++j) {
          if (j + 1 == nkb) next_blocks(then);
          bool more = false;  // some tile's next S was issued
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok) break;
            if (j < cur[t]) {
              const uint32_t v0 = smem_u32(sV + v_at.stage * Ly::kTileBytes);
              if (j == 0) {  // O is overwritten: the last item's has been read
                if (!(ok = mbar_wait_short(&o_empty[t], o_parity[t] ^ 1u, p.err, kErrWaitMma))) break;
                o_parity[t] ^= 1u;
              }
              // 16 keys per MMA: keys 0-95 as soon as the softmax has written them, then 96-127.
              if (!(ok = mbar_wait_short(&p_part[t], p_parity[t], p.err, kErrWaitMma))) break;
              if (!(ok = mbar_wait_short(&v_full[v_at.stage], v_at.parity, p.err, kErrWaitMma))) break;
              tc_fence_after();
#pragma unroll
              for (int k = 0; k < 6; ++k)
                umma_f16_ts(tmem + t * 256 + 128, tmem + t * 256 + 8 * k, smem_desc_mn_sw128(v0 + k * 2048, kPtBox),
                            idesc_o, (j | k) != 0 ? 1u : 0u);
              if (!(ok = mbar_wait_short(&p_full[t], p_parity[t], p.err, kErrWaitMma))) break;
              tc_fence_after();
#pragma unroll
              for (int k = 6; k < 8; ++k)
                umma_f16_ts(tmem + t * 256 + 128, tmem + t * 256 + 8 * k, smem_desc_mn_sw128(v0 + k * 2048, kPtBox),
                            idesc_o, 1u);
              umma_commit(&pv_done[t]);
              p_parity[t] ^= 1u;
              if constexpr (kApart) {
                umma_commit(&v_empty[v_at.stage]);
                v_at.next();
              }
            }
            // The tile's next S, of this item or the next: over P, which the P.V issued before it
            // reads first (issue order).
            const bool same = j + 1 < cur[t], other = j + 1 == nkb && then[t] > 0;
            if (same || other) {
              issue_s(t, other, same ? j + 2 == cur[t] : then[t] == 1);
              more = true;
            }
          }
          if (!kApart && ok) {
            umma_commit(&v_empty[v_at.stage]);
            v_at.next();
            if (more) {
              umma_commit(&k_empty[k_at.stage]);
              k_at.next();
            }
          }
        }
        cur[0] = then[0];
        cur[1] = then[1];
      }
      if (!ok) {
        umma_commit(drain_bar);  // MMAs already issued retire before TMEM is released
        mbar_wait_drain(drain_bar, 0);
      }
    }
  } else {
    regs_inc<kPtRegsSoftmax>();
    // ------------------------------------------------------------ softmax
    const int t = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const uint32_t sbase = tmem + t * 256 + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t obase = sbase + 128;
    uint32_t s_parity = 0;  // of s_full and pv_done: one use per block
    Turn<kPtItems> at;
    bool good = true;
    for (;; at.next()) {
      good = __all_sync(0xffffffffu, mbar_wait_short(&item_full[at.stage], at.parity, p.err, kErrWaitEpilogue));
      if (!good || ld_shared_int(&items[at.stage].head) < 0) break;
      const int n = ld_shared_int(&items[at.stage].blocks[t]);
      int left;  // keys that this row sees, from the block at hand on
      bool idle;
      {
        const int lq = ld_shared_int(&items[at.stage].lq), lk = ld_shared_int(&items[at.stage].lk);
        const int row = ld_shared_int(&items[at.stage].row0) + (kMode == kTilesOfHead ? t * kPtRows : 0) + quarter * 32 + lane;
        left = p.causal ? min(lk, row + 1 + lk - lq) : lk;
        idle = row - lane >= lq;
      }
      if (idle) {
        // None of the warp's rows is in the sequence: what its P and O hold matters to no other row.
#pragma unroll 1
        for (int j = 0; j < n; ++j, s_parity ^= 1u) {
          good = __all_sync(0xffffffffu, mbar_wait_short(&s_full[t], s_parity, p.err, kErrWaitEpilogue));
          if (!good) break;
          if (lane == 0) {
            mbar_arrive(&p_part[t]);
            mbar_arrive(&p_full[t]);
          }
        }
        if (!good) break;
        if (lane == 0) {
          if (n > 0) mbar_arrive(&o_empty[t]);
          mbar_arrive(&item_empty[at.stage]);
        }
        __syncwarp();
        continue;
      }
      int whole = 0, left_part = 0;  // blocks that need no look at `left`; its value behind them
      if constexpr (kChosen) {
        whole = ld_shared_int(&items[at.stage].whole[t]);
        left_part = left - ld_shared_int(&items[at.stage].part_block[t]) * kPtKeys;
        left = kPtKeys;
      }
      float m_used = -INFINITY, l_sum = 0.f;
      for (int j = 0; j < n; ++j, s_parity ^= 1u, left -= kChosen && j <= whole ? 0 : kPtKeys) {
        if (kChosen && j == whole) left = left_part;
        good = __all_sync(0xffffffffu, mbar_wait_short(&s_full[t], s_parity, p.err, kErrWaitEpilogue));
        if (!good) break;
        tc_fence_after();
        uint32_t r[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(sbase + c * 32, r[c]);
        tmem_wait_ld();
        if (__any_sync(0xffffffffu, left < kPtKeys)) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= left) r[c][i] = 0xFF800000u;  // -inf
        }
        float m16[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) m16[i] = fmaxf(__uint_as_float(r[0][i]), __uint_as_float(r[0][i + 16]));
#pragma unroll
        for (int c = 1; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 16; ++i) m16[i] = max3f(m16[i], __uint_as_float(r[c][i]), __uint_as_float(r[c][i + 16]));
        float mx = m16[0];
#pragma unroll
        for (int i = 1; i < 15; i += 2) mx = max3f(mx, m16[i], m16[i + 1]);
        mx = fmaxf(mx, m16[15]) * p.scale_log2;  // scale > 0: the max commutes with it
        // The maximum in use is raised only when a block exceeds it by 2^8 (O is then rescaled).
        const bool raise = mx > m_used + kPtRescaleLog2;
        const float alpha = raise ? fast_exp2(m_used - mx) : 1.f;
        if (raise) m_used = mx;
        if (__any_sync(0xffffffffu, raise && j > 0)) {
          good = __all_sync(0xffffffffu, mbar_wait_short(&pv_done[t], s_parity ^ 1u, p.err, kErrWaitEpilogue));
          if (!good) break;
          tc_fence_after();
#pragma unroll
          for (int c = 0; c < D / 32; ++c) {
            uint32_t o[32];
            tmem_ld_32x32b_x32(obase + c * 32, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st_32x32b_x32(obase + c * 32, o);
          }
        }
        l_sum *= alpha;
        const uint64_t ua2 = f2_splat(p.scale_log2), nm2 = f2_splat(m_used == -INFINITY ? 0.f : -m_used);
        uint64_t ls2[2] = {f2_splat(0.f), f2_splat(0.f)};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            const float2 xx = f2_unpack(f2_fma(f2_pack(r[c][i], r[c][i + 1]), ua2, nm2));
            const float x0 = fast_exp2(xx.x), x1 = fast_exp2(xx.y);
            ls2[(i >> 1) & 1] = f2_add(ls2[(i >> 1) & 1], f2_pack(__float_as_uint(x0), __float_as_uint(x1)));
            pk[i >> 1] = pack2<T>(x0, x1);
          }
          tmem_st_32x32b_x16(sbase + c * 16, pk);
          if (c == 2) {
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_part[t]);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[t]);
        const float2 la = f2_unpack(ls2[0]), lb = f2_unpack(ls2[1]);
        l_sum += (la.x + la.y) + (lb.x + lb.y);
      }
      if (!good) break;
      if (n > 0) {
        good = __all_sync(0xffffffffu, mbar_wait_short(&pv_done[t], s_parity ^ 1u, p.err, kErrWaitEpilogue));
        if (!good) break;
        tc_fence_after();
      }
      const float inv = l_sum != 0.f ? __fdividef(1.f, l_sum) : 0.f;  // (a NaN sum stays a NaN)
      const Item w = items[at.stage];
      __syncwarp();
      if (lane == 0) mbar_arrive(&item_empty[at.stage]);
      const int warp_row = w.row0 + (kMode == kTilesOfHead ? t * kPtRows : 0) + quarter * 32;
      const int head = w.head + (kMode == kTilesOfHead ? 0 : t);
      const int rows = !kApart || (t < p.item_heads && head < p.hq) ? w.lq - warp_row : 0;  // of this warp's 32
      // 64 columns at a time through this warp's staging space: a row per lane in, four rows of
      // 128 bytes per instruction out (16-byte pieces swizzled by the row).  A row that sees nothing
      // has P = 0 and so O = 0; without any key O was not written, and counts as 0.
      uint8_t* stage = smem + Ly::kOut + (warp - 4) * 4096;
      const int out_row = lane >> 3, piece = lane & 7;
      T* dst = static_cast<T*>(p.out) + static_cast<long long>(w.q0 + warp_row + out_row) * p.ldo +
               static_cast<long long>(head) * p.hso + piece * 8;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(obase + c * 32, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) o[i] = 0u;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            x[k] = pack2<T>(__uint_as_float(o[8 * i + 2 * k]) * inv, __uint_as_float(o[8 * i + 2 * k + 1]) * inv);
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((((c & 1) * 4 + i) ^ (lane & 7)) << 4)) =
              make_uint4(x[0], x[1], x[2], x[3]);
        }
        if (c & 1) {
          __syncwarp();
          T* to = dst + (c >> 1) * 64;
#pragma unroll 1
          for (int row = out_row; row < 32; row += 4, to += 4 * p.ldo)
            if (row < rows)
              *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(stage + row * 128 + ((piece ^ (row & 7)) << 4));
          __syncwarp();
        }
      }
      if (n > 0) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&o_empty[t]);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------- pieces of the few-row kernels

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1) {
  if constexpr (std::is_same<T, __half>::value)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes, global to shared memory, or zeros where !live (src is not read then).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t src) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(src) : "memory");
  return v;
}

// ---------------------------------------------------------------------------- host side

// Average queries per sequence up to which two heads beat two tiles of one head (24 heads of 128, 64 x 128
// tokens: 51 and 53 us; 32 x 256: the same; 16 x 512: 92 and 89 us; 96 short prompts 237 and 301 us).
constexpr int64_t kPtApartRows = 256;

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

template <typename T, int D, int kMode, bool kChosen = false>
b2g_status launch_tiles(const PkParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, int sms,
                        cudaStream_t st) {
  constexpr uint32_t smem = kChosen ? PtLayout<D>::kSmemChosen : PtLayout<D>::kSmem;
  static_assert(smem <= 227 * 1024, "shared memory budget");
  auto kern = packed_tiles_kernel<T, D, kMode, kChosen>;
  b2g_status s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                            "cudaFuncSetAttribute(packed_tiles)");
  if (s != B2G_OK) return s;
  constexpr int kSpan = kMode == kTilesOfHead ? 2 * kPtRows : kPtRows;
  const int64_t items = (static_cast<int64_t>(p.total_q) / kSpan + p.batch) * (kMode == kTilesOfHead ? p.hq : (p.hq + p.item_heads - 1) / p.item_heads);
  return launch_pdl(kern, dim3(static_cast<unsigned>(items < sms ? items : sms)), dim3(kPtThreads), smem, st,
                    "packed_tiles launch", tq, tk, tv, p);
}

// A stride of a dimension that has one element says nothing: any valid one.
int64_t used(int64_t stride, int64_t extent, int64_t fallback) { return extent > 1 ? stride : fallback; }

}  // namespace

}  // namespace b2g
