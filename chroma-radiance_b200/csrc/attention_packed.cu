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
};

// One work item: rows [row0, row0 + 128) of tile A and B (B's 128 further on in kTilesOfHead).
struct PtItem {
  int q0, lq, k0, lk;
  int row0, head;  // of tile A; head -1: no more items
  int blocks[2];   // key blocks of each tile (0: nothing to see, or no rows)
};
static_assert(sizeof(PtItem) == 32, "two 16-byte words");

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

template <typename T, int D, int kMode>
__global__ void __launch_bounds__(kPtThreads, 1)
    packed_tiles_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                        const __grid_constant__ CUtensorMap tmV, const PkParams p) {
  using Ly = PtLayout<D>;
  constexpr int KS = Ly::KS, VS = Ly::VS;
  constexpr bool kApart = kMode == kHeadsApart;
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
  PtItem* items = reinterpret_cast<PtItem*>(smem + Ly::kItems);
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
  auto keys_seen = [&](const PtItem& w) {
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
      const int grid = static_cast<int>(gridDim.x), cta = static_cast<int>(blockIdx.x);
      int units_before = 0, i = 0;
      Turn<kPtItems> at;
      for (int round = 0; i >= 0; ++round) {
        const long long index = static_cast<long long>(round) * grid + (round & 1 ? grid - 1 - cta : cta);
        const int unit = static_cast<int>(index / head_units);
        const int head_unit = static_cast<int>(index - static_cast<long long>(unit) * head_units);
        auto seq_of = [&](int j) { return sorted ? static_cast<int>(order[j]) : j; };
        i = find_seq(p.batch, unit, lane, [&](int j) {
          const int b = seq_of(j), lo = clampi(__ldg(p.cu_q + b), 0, p.total_q);
          return (clampi(__ldg(p.cu_q + b + 1), lo, p.total_q) - lo + kSpan - 1) / kSpan;
        }, &units_before, i);
        PtItem w{};
        w.head = -1;
        if (i >= 0) {
          const Seq s = load_seq(p, seq_of(i));
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
        const PtItem w = items[at.stage];
        mbar_arrive(&item_empty[at.stage]);
        if (w.head < 0) break;
        const int nkb = max(w.blocks[0], w.blocks[1]);
        const int kv_head = w.head / p.group, kv_head_b = kApart ? (w.head + 1) / p.group : kv_head;
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
            mbar_arrive_expect_tx(&k_full[k_at.stage], Ly::kTileBytes);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_3d(sK + k_at.stage * Ly::kTileBytes + c * kPtBox, &tmK, &k_full[k_at.stage], c * 64,
                          w.k0 + j * kPtKeys, t ? kv_head_b : kv_head, shared_kv);
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
      PtItem w{};
      int seen = 0;
      auto nkb = [](const PtItem& i) { return max(i.blocks[0], i.blocks[1]); };
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
          have = more;
          continue;
        }
        if (have && (tails == 0 || ready(&v_empty[v_at.stage], v_at.parity ^ 1u))) {
          const int st = v_at.stage;
          ok = __all_sync(0xffffffffu, wait(&v_empty[st], v_at.parity ^ 1u, kErrWaitProducer));
          if (!ok) break;
          const int valid = seen - key;  // rows of this block that are seen
          if (lane == 0) {
            uint64_t* bar = valid < kPtKeys ? &v_land[st] : &v_full[st];
            mbar_arrive_expect_tx(bar, Ly::kTileBytes);
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_3d(sV + st * Ly::kTileBytes + c * kPtBox, &tmV, bar, c * 64, w.k0 + key, (w.head + t) / p.group,
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
      float m_used = -INFINITY, l_sum = 0.f;
      for (int j = 0; j < n; ++j, s_parity ^= 1u, left -= kPtKeys) {
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
      const PtItem w = items[at.stage];
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
// Average queries per sequence up to which two heads beat two tiles of one head (24 heads of 128, 64 x 128
// tokens: 51 and 53 us; 32 x 256: the same; 16 x 512: 92 and 89 us; 96 short prompts 237 and 301 us).
constexpr int64_t kPtApartRows = 256;

// What a call runs, from its sizes alone (the offsets are on the device).
struct PkPlan {
  bool rows = false;       // packed_rows (+ packed_combine), else packed_tiles
  int shares = 0;
  size_t o_bytes = 0, bytes = 0;
};

int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }

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

template <typename T, int D, int kMode>
b2g_status launch_tiles(const PkParams& p, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, int sms,
                        cudaStream_t st) {
  constexpr uint32_t smem = PtLayout<D>::kSmem;
  static_assert(smem <= 227 * 1024, "shared memory budget");
  auto kern = packed_tiles_kernel<T, D, kMode>;
  b2g_status s = check_cuda(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)),
                            "cudaFuncSetAttribute(packed_tiles)");
  if (s != B2G_OK) return s;
  constexpr int kSpan = kMode == kTilesOfHead ? 2 * kPtRows : kPtRows;
  const int64_t items = (static_cast<int64_t>(p.total_q) / kSpan + p.batch) * (kMode == kTilesOfHead ? p.hq : (p.hq + p.item_heads - 1) / p.item_heads);
  return launch_pdl(kern, dim3(static_cast<unsigned>(items < sms ? items : sms)), dim3(kPtThreads), smem, st,
                    "packed_tiles launch", tq, tk, tv, p);
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

// A stride of a dimension that has one element says nothing: any valid one.
int64_t used(int64_t stride, int64_t extent, int64_t fallback) { return extent > 1 ? stride : fallback; }

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
