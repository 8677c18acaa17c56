// Attention of many query rows on the tensor cores: packed prompts, and chunks of new tokens over
// the paged cache.
//
// A work item is two tiles of 128 query rows of one key/value head (rows: token x the query heads that
// share the head, so grouped heads read each key tile once), walked over the keys that they see in
// tiles of 128.  Per tile and key tile: S = Q K^T into TMEM, the softmax warps turn S into
// probabilities P, 16-bit pairs in TMEM, and O += P V with P as the TMEM operand.
// Two row tiles share every K and V tile, so that the tensor core works on one while the softmax
// warps work on the other.  S has one place in TMEM, which the tiles take in turn: a tile's scores leave it for
// registers at once, so the next product needs neither to wait for the exponentials nor for P to be consumed
// (with P in S's place each tile's P V, the next S and their latency, 1400 clocks, followed the 1850 of its
// softmax: 1040 TFLOP/s).  A thread owns a row, so the running maximum m and sum l need no exchange
// between threads.  O in TMEM is in units of a reference maximum that moves only when a row's true
// maximum has passed it by 2^8: P stays inside fp16 and the rescaling of O, a
// round trip through registers, is skipped for almost every tile.
//
// A 128 x 128 tile costs 1024 clocks of exp on the special-function units (16 a clock), as many as its
// two products at head size 128.  Taking a part of the powers by a polynomial on the multiply-add
// pipes instead made every size slower (8 of 32: 3 %, 16 of 32: 8 %): the softmax warps are not what the products wait for.
//
// Few items (and a workspace, with the paged cache): items longer than an SM's share of all key tiles
// are split into parts, which go out like items; each leaves its rows' unnormalised sums, and a second
// launch joins them.
//
// One CTA per SM stays for all its items: the loads, the score products and the search of the next
// item go on while the softmax warps write the last one's output.  Items go out in the order of their key tiles,
// the longest first, one to each CTA in turn and every other turn backwards, so that ragged batches
// and the causal triangle end evenly.
//
// Roles: warps 0-3 softmax of tile 0, warps 4-7 of tile 1, one thread each of warps 8 and 11 issues
// the MMAs of tile 0 and of tile 1 (one thread for both spent 93 clocks an MMA instead of the
// pipe's 64: it holds few MMAs, and ran dry whenever the thread looked at its barriers), warp 9
// loads, warp 10 finds the items and cleans V tiles.  Registers are split by warpgroup, 216 for a softmax thread (it
// holds a whole row of S) and 72 for the others, 2 * 216 + 72 = 3 * 168 as launched.
// TMEM columns: S 0-127, P0 128-191, P1 192-255, O0 256-, O1 384-.
//
// Rows of more than 16384 keys are summed in stretches (kSumKeys): O starts anew and the sums before go to fp32 ones in
// local memory, since the registers hold a row of S.
//
// Measured (32 heads over 8, head size 128, bf16, 1000 W limit; boxes and the length of the run differ): one prompt of
// 16384 tokens 1.69 ms (1305 TFLOP/s) in the first second, 1.95 to 1.97 ms in long runs at 1.55 GHz; 19 ragged prompts of
// 15001 tokens 213 to 226 us; 2 x 1024 tokens over 32768 cached keys 475 to 560 us.  In chunks and long prompts the
// tensor pipe is 64 % active; ragged ones lose 9000 clocks an item to the last product's latency and the output, which
// warps of their own did not win back (registers: 176 / 80 / 80; 260 -> 285 us).
#pragma once
#include <climits>

#include "attention_join.cuh"

namespace aexrt {

constexpr int kTcRows = 128;   // query rows of a tile
constexpr int kTcKeys = 128;   // keys of a tile
constexpr int kTcThreads = 384;
// Items of fewer key tiles stay whole: below, the joining costs more than the split saves (100 tokens over 300 cached
// keys: 19 us whole, 22 in parts of 2 tiles).
constexpr int kTcMinTiles = 6;
constexpr int kTcStretch = kSumKeys / kTcKeys;  // key tiles that O sums in TMEM

// Slots of the K / V ring: what 227 KB hold beside the two Q tiles and the output staging.
template <int DP>
constexpr int tc_slots() { return DP == 128 ? 4 : 8; }

template <int DP>
struct TcSmem {
  static constexpr int kTile = 128 * DP * 2;
  static constexpr int kQ = 0, kRing = 2 * kTile, kStage = kRing + tc_slots<DP>() * kTile;
  static constexpr int kBars = kStage + 8 * 4096;  // per softmax warp: 32 rows of 64 output columns
  // barriers, TMEM base, items; then, per item of two, the first keys with non-finite values of a column
  static constexpr int kFix = kBars + 640, kBytes = kFix + 2 * kFixInts * 4;
};

__device__ __forceinline__ uint64_t desc_sw128(uint32_t saddr, uint32_t lbo, uint32_t sbo) {
  return static_cast<uint64_t>((saddr >> 4) & 0x3FFFu) | static_cast<uint64_t>((lbo >> 4) & 0x3FFFu) << 16 |
         static_cast<uint64_t>((sbo >> 4) & 0x3FFFu) << 32 | 1ull << 46 | 2ull << 61;  // 128-byte swizzle
}

// kind::f16 instruction descriptor, M = 128: fp32 accumulator, 16-bit operands, B along N or along K.
template <typename T>
__device__ __forceinline__ uint32_t tc_idesc(int n, bool b_along_n) {
  constexpr uint32_t fmt = sizeof(T) == 2 && __is_same(T, __nv_bfloat16) ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (b_along_n ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         ((128u >> 4) << 24);
}

// D[tmem] (+)= A[tmem] * B[smem], one K step of 16.
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(acc)
      : "memory");
}

__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
      "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
      "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
      "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]),
      "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(taddr)
      : "memory");
}
// 16 columns: the rescaling runs beside a whole row of S in registers.
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::
          "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

struct TcWork {
  int head, seq, tile, len_q, rows_q, len_k, q0, k0;  // rows_q: query tokens taken (len_q, at most max_q); head -1: no more
  int begin, end;  // key tiles
  int part;        // part of the workspace that the rows go to, -1: the item is whole
};

// Splitting.  An item of more than T key tiles is split into ceil(tiles / T) parts.  T is a CTA's share of all key tiles,
// a little more when that leaves one part to a CTA (equal contexts); else, where it does not (ragged ones), two thirds of
// the share, for parts that even out over the CTAs.  So at most 1.5 * grid items are split, into at most 3 * grid
// parts.  Items are numbered by falling length, so those that have a part k are the first ones.  The parts go out part 0
// of every item first, then the parts 1, ...; part k of item r lies at bases[k] + r.
struct TcSplit {
  int* split_items; // of the call
  int* bases;       // [3 * grid]
  JoinHead* heads;  // [2 * grid]
  float* sums;      // [3 * grid][256][head_dim]
  float* stats;     // [3 * grid][256][2]
};

// Numbers the items of a call: descending in key tiles while a warp can hold every sequence's lengths
// (kHeld per lane), else by sequence.  Asked for ascending numbers, by a whole warp.  By length against by sequence, in
// us (32 heads over 8 of 128, causal): 19 ragged prompts of 15001 tokens 210-231 against 271-274, 8 of 13870 425-459
// against 439-449, 100 of 42775 490-520 against 492-501; but 40 short ones of 3867 tokens 50 against 47 and 32 of 512
// 153-168 against 140-153, where each search costs more than the order saves.
template <bool kPaged>
struct TcFinder {
  static constexpr int kHeld = 4;
  const AttnParams& p;
  int tokens;      // query tokens of an item
  float per_token; // 1 / tokens
  // of sequence 32 * h + lane: items, len_k - len_q, key tiles of the last item and what that counts for
  int items[kHeld], shift[kHeld], tiles[kHeld], last[kHeld];
  int total = 0, top = 0;  // of all sequences: items, key tiles at most
  int64_t volume = 0;      // items times their sequence's most key tiles
  int level = 0;           // of the item found last
  int base = 0;            // by sequence: the first sequence of the 32 looked at, and the items before it
  int64_t before = 0;

  __device__ __forceinline__ TcFinder(const AttnParams& params, int tokens_) : p(params), tokens(tokens_) {
    per_token = 1.f / static_cast<float>(tokens);
    if (p.num_seqs <= 32 * kHeld) {
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        const int s = 32 * h + (threadIdx.x & 31);
        items[h] = shift[h] = tiles[h] = 0;
        last[h] = -1;
        if (s < p.num_seqs) {
          const int len_q = q_len(p, s), len_k = k_len<kPaged>(p, s), rows = kPaged ? min(len_q, p.max_q) : len_q;
          items[h] = (rows + tokens - 1) / tokens;
          shift[h] = len_k - len_q;
          if (rows) {
            tiles[h] = (keys_seen(rows - 1, len_q, len_k, p.causal) + kTcKeys - 1) / kTcKeys;
            // the last item counts half its key tiles when it fills one row tile only
            last[h] = rows - (items[h] - 1) * tokens <= tokens / 2 ? (tiles[h] + 1) / 2 : tiles[h];
          }
        }
        total += items[h];
        volume += static_cast<int64_t>(items[h]) * tiles[h];
        top = max(top, tiles[h]);
      }
      total = __reduce_add_sync(~0u, total);
      top = __reduce_max_sync(~0u, top);
#pragma unroll
      for (int o = 16; o; o >>= 1) volume += __shfl_xor_sync(~0u, volume, o);
    }
  }
  __device__ __forceinline__ int rows_of(int s) const { return kPaged ? min(q_len(p, s), p.max_q) : q_len(p, s); }
  // Items of held sequence h of this lane with at least `level` key tiles, its last item aside.
  __device__ __forceinline__ int items_from(int h, int level) const {
    const int before_last = max(0, items[h] - 1);
    if (level <= 0) return before_last;
    if (level > tiles[h]) return 0;
    if (!p.causal) return before_last;
    // item t ends at token e = (t + 1) * tokens and sees e + shift keys: the first ceil(e / tokens) - 1 see too few
    const int e = (level - 1) * kTcKeys + 1 - shift[h];
    if (e <= 0) return before_last;
    int few = static_cast<int>(static_cast<float>(e - 1) * per_token);  // floor((e - 1) / tokens), then made exact
    while (few * tokens > e - 1) --few;
    while ((few + 1) * tokens <= e - 1) ++few;
    return max(0, before_last - few);
  }
  __device__ __forceinline__ int all_from(int level) const {
    int n = 0;
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
      if (32 * h < p.num_seqs) n += items_from(h, level) + (last[h] >= max(level, 0) ? 1 : 0);
    return __reduce_add_sync(~0u, n);
  }
  // Parts of at most `size` key tiles that all items make, each counted like its sequence's longest.
  __device__ __forceinline__ int64_t parts_at_most(int size) const {
    int n = 0;
#pragma unroll
    for (int h = 0; h < kHeld; ++h)
      if (32 * h < p.num_seqs) n += items[h] * ((tiles[h] + size - 1) / size);  // items of a split call: 1.5 for an SM at most
    return __reduce_add_sync(~0u, n);
  }
  __device__ __forceinline__ void fill(TcWork& w, int s, int tile) const {
    w.seq = s;
    w.tile = tile;
    w.rows_q = rows_of(s);
    w.len_q = q_len(p, s);
    w.q0 = q_start(p, s);
    w.len_k = k_len<kPaged>(p, s);
    w.k0 = k_start<kPaged>(p, s);
  }
  __device__ __forceinline__ bool find(int64_t item, TcWork& w) {
    const int lane = threadIdx.x & 31;
    if (p.num_seqs <= 32 * kHeld) {
      if (item >= total) return false;
      int lo = 0, hi = top;  // the highest level that has more than `item` items at or above it
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (all_from(mid) > item) lo = mid; else hi = mid - 1;
      }
      level = lo;
      int rank = static_cast<int>(item) - all_from(lo + 1);  // among the items of exactly this level
#pragma unroll
      for (int h = 0; h < kHeld; ++h) {
        if (32 * h >= p.num_seqs) break;
        const int above = items_from(h, lo + 1), here = items_from(h, lo) - above;
        const int n = here + (last[h] == lo ? 1 : 0);
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int z = __shfl_up_sync(~0u, sum, o);
          if (lane >= o) sum += z;
        }
        const uint32_t past = __ballot_sync(~0u, sum > rank);
        if (past) {
          const int src = __ffs(past) - 1;
          const int off = rank - (sum - n);
          // a sequence's later items see more keys: those above this level are the last ones before its last item
          const int tile = off < here ? items[h] - 2 - above - off : items[h] - 1;
          fill(w, 32 * h + src, __shfl_sync(~0u, tile, src));
          return true;
        }
        rank -= __shfl_sync(~0u, sum, 31);
      }
      return false;
    }
    for (; base < p.num_seqs; base += 32) {
      const int s = base + lane;
      const int n = s < p.num_seqs ? (rows_of(s) + tokens - 1) / tokens : 0;
      int sum = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int z = __shfl_up_sync(~0u, sum, o);
        if (lane >= o) sum += z;
      }
      const uint32_t past = __ballot_sync(~0u, before + sum > item);
      if (past) {
        const int src = __ffs(past) - 1;
        const int tile = n - 1 - static_cast<int>(item - before - (sum - n));
        fill(w, base + src, __shfl_sync(~0u, tile, src));
        return true;
      }
      before += __shfl_sync(~0u, sum, 31);
    }
    return false;
  }
};

// An item's two row tiles: first token, tokens, keys that the last one sees, key tiles from `begin` on.
template <bool kSplit>
struct TcTiles {
  int first[2], valid[2], keys[2], n[2];
  int key_end, nmax, common;  // keys at and above `common` are seen by some rows and not by others
  int unclean;                // from this one on (of all of the item's) V tiles are cleaned before their product
  __device__ __forceinline__ TcTiles(const AttnParams& p, const TcWork& w, int tokens) {
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      first[s] = (w.tile * 2 + s) * tokens;
      valid[s] = clampi(w.rows_q - first[s], 0, tokens);
      keys[s] = valid[s] ? keys_seen(first[s] + valid[s] - 1, w.len_q, w.len_k, p.causal) : 0;
      n[s] = (keys[s] + kTcKeys - 1) / kTcKeys;
      if (kSplit) n[s] = max(0, min(n[s], w.end) - w.begin);
    }
    key_end = max(keys[0], keys[1]);
    nmax = max(n[0], n[1]);
    common = min(keys_seen(first[0], w.len_q, w.len_k, p.causal), key_end);
    unclean = (common < key_end ? common : key_end) / kTcKeys;  // a whole last tile that all rows see: none
  }
};

__device__ __forceinline__ void mbar_arrive_count(uint64_t* bar, uint32_t count) {
  asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.shared::cta.b64 st, [%0], %1;\n\t}" ::"r"(smem_u32(bar)), "r"(count)
               : "memory");
}

// A wait that may last an item: it gives up when neither the barrier nor the loading warp (*beat, its ring items) has
// moved for the limit's clocks.  An item may take longer than any limit (40 million keys pass half a second).  The ring is
// finite, so a loading warp that goes on means products that go on.  Only where it is needed: the finding warp's waits, and
// the softmax warps' for an item or its first scores, whose tile may have no part in the item before.  All other waits are
// over within a few key tiles (in every wait of the kernel it made ragged prompts 9 % slower).
__device__ __forceinline__ bool mbar_wait_beat(uint64_t* bar, uint32_t parity, uint32_t* status, const volatile int* beat) {
  while (true) {
    const int seen = *beat;
    const long long t0 = clock64();
    do {
      if (mbar_try_wait(bar, parity)) return true;
    } while (clock64() - t0 <= kWaitLimitCycles);
    if (*beat == seen) {
      atomicOr(status, kAttnTimeout);
      return false;
    }
  }
}

// Quarters of 32 keys that a row tile needs of key tile j when its last row sees `keys` keys: products and
// softmax of the last tile stop there.
__device__ __forceinline__ int tc_quarters(int keys, int j) { return min(4, (keys - j * kTcKeys + 31) >> 5); }

template <int kRegs>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

template <typename T, bool kPaged, int DP, bool kSplit>
__global__ void __launch_bounds__(kTcThreads, 1)
    attention_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map, const AttnParams p, const TcSplit split) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using L = TcSmem<DP>;
  constexpr int NS = tc_slots<DP>(), kHalves = DP / 64;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t *q_empty = q_full + 2, *s_full = q_empty + 2, *p_full = s_full + 2, *o_done = p_full + 2, *w_full = o_done + 2,
           *w_empty = w_full + 2, *kv_full = w_empty + 2, *kv_empty = kv_full + NS, *raw = kv_empty + NS, *s_free = raw + NS,
           *drain = s_free + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
  int* fixed = reinterpret_cast<int*>(tmem_slot + 1);  // [2]
  volatile int* beat = fixed + 2;
  TcWork* work = reinterpret_cast<TcWork*>(fixed + 3);  // [2]
  int* fix = reinterpret_cast<int*>(smem + L::kFix);    // [2][kFixInts]
  static_assert((14 + 3 * tc_slots<DP>() + 4) * 8 + 16 + 2 * sizeof(TcWork) <= 640, "barriers and items fit");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(q_empty + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
      mbar_init(o_done + i, 1);
      mbar_init(w_full + i, 1);
      mbar_init(w_empty + i, 12);  // the loading and the cleaning warp, two MMA threads, eight softmax warps
      mbar_init(s_free + i, 128);
      mbar_init(drain + i, 1);
      fixed[i] = 0;
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 2);
      mbar_init(raw + i, 1);
    }
    *beat = 0;
    fence_mbar_init();
  }
  for (int i = threadIdx.x; i < 2 * kFixInts; i += kTcThreads) fix[i] = INT_MAX;
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_dep_wait();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int tokens = kTcRows / p.group;  // query tokens of a row tile
  auto wait = [&](uint64_t* bar, int phase) { return mbar_wait_bounded(bar, phase & 1, p.status, kAttnTimeout); };
  auto wait_long = [&](uint64_t* bar, int phase) { return mbar_wait_beat(bar, phase & 1, p.status, beat); };
  // Item number k of this CTA, once it is known; head -1 ends the roles (so does a wait that gave up).
  auto item = [&](int k, TcWork& w, bool may_last) {
    const bool ok = may_last ? wait_long(w_full + (k & 1), k >> 1) : wait(w_full + (k & 1), k >> 1);
    w = work[k & 1];
    return ok && w.head >= 0;
  };

  if (warp >= 8) {
    regs_down<72>();
    if (warp == 10) {
      // ---------------------------------------------------------------- items
      TcFinder<kPaged> finder(p, 2 * tokens);
      // splitting, when the finder numbers by length: key tiles of a part, and parts of the longest item
      const int64_t all = static_cast<int64_t>(finder.total) * p.kv_heads;
      const bool splits = kSplit && finder.total > 0;
      int size = 1, most = 1;
      // items and heads with a part k, of those that are split
      auto with_part = [&](int k) { return finder.all_from(max(1, k) * size + 1) * p.kv_heads; };
      if (splits) {
        const int grid = gridDim.x;
        const int share = max(kTcMinTiles, static_cast<int>((finder.volume * p.kv_heads + grid - 1) / grid));
        bool fits = false;
        for (size = share; all <= grid && 10 * size <= 13 * share; size += max(1, size / 16))
          if ((fits = finder.parts_at_most(size) * p.kv_heads <= grid)) break;
        if (!fits) size = max(kTcMinTiles, (2 * share + 2) / 3);
        most = max(1, (finder.top + size - 1) / size);
      }
      const int first = splits && most > 1 ? with_part(0) : 0;  // the items that are split
      int part = 0;             // of the numbers that are handed out now, their first, and how many there are
      int64_t part_start = 0, part_count = all;
      bool last = false;  // the item that ends the roles is out
      // Finds item number k of this CTA and puts it out, once every role has left item k - 2; false: that wait gave up.
      auto publish = [&](int k) {
        int64_t number = static_cast<int64_t>(k) * gridDim.x + ((k & 1) ? gridDim.x - 1 - blockIdx.x : blockIdx.x);
        if (splits) {
          while (number >= part_start + part_count && part + 1 < most) {
            part_start += part_count;
            part_count = with_part(++part);
          }
          number -= part_start;
        }
        TcWork w = {};
        w.end = INT_MAX;
        w.part = -1;
        const bool found = (!splits || number < part_count) && finder.find(number / p.kv_heads, w);
        w.head = found ? static_cast<int>(number % p.kv_heads) : -1;
        if (splits && found) {
          const int parts = (finder.level + size - 1) / size;
          if (parts > 1) {
            const TcTiles<false> t(p, w, tokens);
            if (part == 0 && lane == 0)
              split.heads[number] = JoinHead{parts, t.valid[0] + t.valid[1], w.q0 + t.first[0], w.head};
            w.begin = static_cast<int>(static_cast<int64_t>(t.nmax) * part / parts);
            w.end = static_cast<int>(static_cast<int64_t>(t.nmax) * (part + 1) / parts);
            w.part = static_cast<int>(number + (part ? first + part_start - all : 0));
          }
        }
        if (!__all_sync(~0u, wait_long(w_empty + (k & 1), (k >> 1) + 1))) return false;
        const bool used = fixed[k & 1] != 0;
        __syncwarp();
        if (used) {  // by item k - 2
          for (int i = lane; i < kFixInts; i += 32) fix[(k & 1) * kFixInts + i] = INT_MAX;
          if (lane == 0) fixed[k & 1] = 0;
          __syncwarp();
        }
        if (lane == 0) {
          work[k & 1] = w;
          mbar_arrive(w_full + (k & 1));
        }
        __syncwarp();
        last = !found;
        return true;
      };
      // V tiles that have to be cleaned before their product.  P is 0 where a row does not see a key, but
      // 0 * inf and 0 * NaN are not: rows behind the last key become zeros (as far as the product goes, a
      // quarter of the tile), and non-finite values of keys that only some rows see are taken out and put
      // back into the outputs of the rows that do.  Such a tile lands on a barrier of its own, and this warp
      // hands it on.
      uint32_t raws = 0;  // per slot, the phase of that barrier
      int it = 0;         // ring items of the items before
      auto clean = [&](int k, const TcWork& w) {
        const TcTiles<kSplit> t(p, w, tokens);
        int* fx = fix + (k & 1) * kFixInts;
        const int begin = kSplit ? w.begin : 0, sub = lane >> 3, piece = lane & 7;
        for (int j = max(t.unclean - begin, 0); j < t.nmax; ++j) {
          const int slot = (it + (j + 1 < t.nmax ? 2 * j + 2 : 2 * t.nmax - 1)) % NS, key = (begin + j) * kTcKeys;
          if (!__all_sync(~0u, wait_long(raw + slot, (raws >> slot) & 1))) return false;
          raws ^= 1u << slot;
          const int last = min(t.key_end - key, kTcKeys), from = max(0, min(t.common - key, last));
          for (int h = 0; h < kHalves; ++h) {
            // 16-byte piece c of row r lies at piece c ^ (r % 8): the 128-byte swizzle
            uint4* tile = reinterpret_cast<uint4*>(smem + L::kRing + slot * L::kTile + h * 16384) + piece;
#pragma unroll 4
            for (int r = last + sub; r < min(kTcKeys, (last + 31) & ~31); r += 4) tile[r * 8] = make_uint4(0, 0, 0, 0);
            for (int r = from + sub; r < last; r += 32) {
              uint32_t bits = 0;
#pragma unroll
              for (int i = 0; i < 8; ++i) {  // rows past the end look at this lane's first row again
                const uint4 x = tile[(r + 4 * i < last ? r + 4 * i : r) * 8];
                bits |= non_finite_bits<T>(x.x) | non_finite_bits<T>(x.y) | non_finite_bits<T>(x.z) | non_finite_bits<T>(x.w);
              }
              if (bits) {
                for (int row = r; row < min(r + 32, last); row += 4)
                  tile[row * 8] = take_non_finite<T>(tile[row * 8], key + row, h * 64 + (piece ^ (row & 7)) * 8, fx);
                fixed[k & 1] = 1;
              }
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(kv_full + slot);
        }
        it += 2 * t.nmax;
        __syncwarp();
        if (lane == 0) mbar_arrive(w_empty + (k & 1));
        return true;
      };
      // two items are out at a time; an item's tiles are cleaned once the next one is out
      bool ok = publish(0) && (last || publish(1));
      for (int k = 0; ok; ++k) {
        const TcWork w = work[k & 1];
        __syncwarp();
        if (w.head < 0 || !clean(k, w)) break;
        if (!last) ok = publish(k + 2);
      }
      if (kSplit && blockIdx.x == 0) {  // for the joining
        int base = 0;
        for (int k = 0; k < most && first; ++k) {
          if (lane == 0) split.bases[k] = base;
          base += with_part(k);
        }
        if (lane == 0) *split.split_items = first;
      }
    } else if (warp == 9) {
      // ---------------------------------------------------------------- loads
      const uint32_t q_bytes = static_cast<uint32_t>(tokens * p.group * 128 * kHalves);
      bool ok = true;
      int it = 0, qs[2] = {0, 0};        // ring items and Q tiles loaded
      uint32_t raws = 0, raw_last = 0;  // per slot: loads onto the barrier `raw`, modulo 2, and whether the last load was one
      TcWork w;
      for (int k = 0; ok; ++k) {
        ok = __all_sync(~0u, wait(w_full + (k & 1), k >> 1));
        w = work[k & 1];
        if (!ok || w.head < 0) break;
        const TcTiles<kSplit> t(p, w, tokens);
        auto load_q = [&](int s) {
          if (!t.n[s] || !ok) return;
          ok = __all_sync(~0u, wait(q_empty + s, qs[s] + 1));
          if (!ok) return;
          ++qs[s];
          if (lane == 0) {
            mbar_arrive_expect_tx(q_full + s, q_bytes);
            for (int h = 0; h < kHalves; ++h)
              tma_load_4d(smem + L::kQ + s * L::kTile + h * 16384, &q_map, q_full + s, h * 64, 0, w.head, w.q0 + t.first[s]);
          }
        };
        // The page of this lane's box of key tile j (no_page for what lies behind the last key)
        const int box_rows = kPaged ? min(1 << p.page_shift, kTcKeys) : kTcKeys;
        auto page_of = [&](int j) {
          const int key = j * kTcKeys + lane * box_rows;
          if (!kPaged || lane * box_rows >= kTcKeys || key >= t.key_end) return p.no_page;
          const int id = __ldg(p.block_table + w.seq * p.table_stride + (key >> p.page_shift));
          if (id >= 0 && id < p.kv_tokens) return id;
          atomicOr(p.status, kAttnBadPage);
          return p.no_page;
        };
        // one K or V tile; the bytes count whole boxes, what lies outside the tensor arrives as zeros
        auto load_kv = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* bar, int j, int page) {
          if (lane == 0) mbar_arrive_expect_tx(bar, L::kTile);
          __syncwarp();
          if constexpr (kPaged) {
            if (lane * box_rows < kTcKeys) {
              const int row = (j * kTcKeys + lane * box_rows) & ((1 << p.page_shift) - 1);
              for (int h = 0; h < kHalves; ++h)
                tma_load_4d(dst + h * 16384 + lane * box_rows * 128, map, bar, h * 64, w.head, row, page);
            }
          } else if (lane == 0) {
            for (int h = 0; h < kHalves; ++h) tma_load_3d(dst + h * 16384, map, bar, h * 64, w.head, w.k0 + j * kTcKeys);
          }
          __syncwarp();
        };
        // pages of the key tiles of the V before last K, of the last K, and of the next one, looked up a tile ahead
        int page_v = 0, page_k = 0, page_next = t.nmax ? page_of(kSplit ? w.begin : 0) : 0;
        load_q(0);
        for (int i = 0; i < 2 * t.nmax && ok; ++i, ++it) {  // K0 K1 V0 K2 V1 ... as the products take them
          const bool is_v = i + 1 == 2 * t.nmax || (i > 0 && !(i & 1));
          const int slot = it % NS, j = (kSplit ? w.begin : 0) + (is_v ? (i + 1 == 2 * t.nmax ? t.nmax : i >> 1) - 1 : (i + 1) >> 1);
          const bool dirty = is_v && j >= t.unclean;
          ok = __all_sync(~0u, wait(kv_empty + slot, it / NS + 1));
          if (!ok) break;
          if (!is_v) {
            page_v = page_k;
            page_k = page_next;
          }
          load_kv(is_v ? &v_map : &k_map, smem + L::kRing + slot * L::kTile, dirty ? raw + slot : kv_full + slot, j,
                  is_v && i + 1 < 2 * t.nmax ? page_v : page_k);
          raw_last = dirty ? raw_last | 1u << slot : raw_last & ~(1u << slot);
          if (dirty) raws ^= 1u << slot;
          if (lane == 0) *beat = it;
          if (kPaged && !is_v) page_next = page_of(j + 1);
          if (i == 0) load_q(1);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(w_empty + (k & 1));
      }
      if (!ok) {
        // a wait gave up: the loads in flight still have to land before the CTA may leave, which are at most the last
        // ones of each slot (a barrier that nothing is loaded onto would cost its whole limit)
        for (int slot = 0; slot < min(NS, it); ++slot)
          if ((raw_last >> slot) & 1) wait(raw + slot, static_cast<int>(raws >> slot) + 1);
          else wait(kv_full + slot, (it - 1 - slot) / NS);
        for (int s = 0; s < 2; ++s)
          if (qs[s]) wait(q_full + s, qs[s] - 1);
      }
    } else if (lane == 0) {
      // ---------------------------------------------------------------- MMA issue, one thread per row tile
      const int s = warp == 8 ? 0 : 1;
      const uint32_t id_s = tc_idesc<T>(kTcKeys, false), id_n = tc_idesc<T>(32, false) - tc_idesc<T>(0, false), id_o = tc_idesc<T>((p.head_dim + 15) / 16 * 16, true);
      const int steps = (p.head_dim + 15) / 16;
      // descriptors of the first K step; later steps and slots add to the address field
      const uint64_t q_desc = desc_sw128(smem_u32(smem + L::kQ + s * L::kTile), 16, 1024);
      const uint64_t k_desc = desc_sw128(smem_u32(smem + L::kRing), 16, 1024);
      const uint64_t v_desc = desc_sw128(smem_u32(smem + L::kRing), 16384, 1024);
      const uint32_t p_at = tmem + 128 + s * 64, o_at = tmem + 256 + s * 128;
      bool ok = true;
      int it = 0, qs = 0, ps = 0;
      auto full = [&](int i) { return wait(kv_full + i % NS, i / NS); };
      TcWork w;
      for (int k = 0; ok && item(k, w, false); ++k) {
        const TcTiles<kSplit> t(p, w, tokens);
        const int n = s ? t.n[1] : t.n[0], keys = s ? t.keys[1] : t.keys[0], begin = kSplit ? w.begin : 0;
        // every ring item in order, K0 K1 V0 K2 V1 ..., also those that only the other tile uses
        for (int j = -1; j < t.nmax && ok; ++j) {
          if (j + 1 < t.nmax) {  // S = Q K^T for key tile j + 1
            const int i = it + (j < 0 ? 0 : 2 * j + 1);
            ok = full(i);
            if (j < 0 && n && ok) ok = wait(q_full + s, qs++);
            // S's place goes tile 0, tile 1, tile 0 ...: it is this tile's once the other's scores have left it.  A
            // tile without this key tile passes its turn on, so that both count the same phases.
            const int turn = (it >> 1) + j + 1;
            if (ok && (s || turn)) ok = s ? wait(s_free, turn) : wait(s_free + 1, turn - 1);
            if (!ok) break;
            if (j + 1 < n) {
              tc_fence_after();
              const uint64_t b = k_desc + (i % NS) * (L::kTile >> 4);
              const uint32_t id = id_s - (4 - tc_quarters(keys, begin + j + 1)) * id_n;
#pragma unroll
              for (int c = 0; c < DP / 16; ++c) {
                const int off = ((c >> 2) * 16384 + (c & 3) * 32) >> 4;
                if (c < steps) tc_mma<true>(tmem, q_desc + off, b + off, id, c != 0);
              }
              tc_commit(s_full + s);
              tc_commit(kv_empty + i % NS);
              if (j + 2 == n) tc_commit(q_empty + s);  // the tile's last score product
            } else {
              mbar_arrive_count(s_free + s, 128);
              mbar_arrive(kv_empty + i % NS);
            }
          }
          if (j >= 0 && ok) {  // O += P V for key tile j
            const int i = it + (j + 1 < t.nmax ? 2 * j + 2 : 2 * t.nmax - 1);
            ok = full(i);
            if (j < n) {
              ok = ok && wait(p_full + s, ps++);
              if (!ok) break;
              tc_fence_after();
              const uint64_t b = v_desc + (i % NS) * (L::kTile >> 4);
              const int quarters = tc_quarters(keys, begin + j);
#pragma unroll
              for (int c = 0; c < kTcKeys / 16; ++c)
                if (c < quarters * 2) tc_mma_ts(o_at, p_at + c * 8, b + c * (2048 >> 4), id_o, (j % kTcStretch | c) != 0);
              tc_commit(o_done + s);
              tc_commit(kv_empty + i % NS);
            } else if (ok) {
              mbar_arrive(kv_empty + i % NS);
            }
          }
        }
        if (!ok) break;
        it += 2 * t.nmax;
        mbar_arrive(w_empty + (k & 1));
      }
      if (!ok) {  // a wait gave up: the products in flight end before TMEM is freed
        tc_commit(drain + s);
        mbar_wait_bounded(drain + s, 0, p.status, kAttnTimeout);
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax: one row per thread
    regs_up<216>();
    const int s = warp >> 2, row = threadIdx.x & 127;
    const int row_token = row / p.group, row_head = row % p.group;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's 32 TMEM lanes
    const uint32_t p_at = lanes + 128 + s * 64, o_at = lanes + 256 + s * 128;
    const float sl2 = p.scale * 1.4426950408889634f;
    bool ok = true;
    int done = 0;  // key tiles of this row tile so far, over all items
    TcWork w;
    for (int k = 0; ok && __all_sync(~0u, item(k, w, true)); ++k) {
      const TcTiles<kSplit> t(p, w, tokens);
      const int first = s ? t.first[1] : t.first[0], valid = s ? t.valid[1] : t.valid[0], n = s ? t.n[1] : t.n[0];
      const int token = first + row_token, begin = kSplit ? w.begin : 0;
      const bool mine = row_token < valid;  // rows behind the last whole token have row_token >= tokens
      const int seen = mine ? keys_seen(token, w.len_q, w.len_k, p.causal) : 0;
      const int all_see = valid ? keys_seen(first, w.len_q, w.len_k, p.causal) : 0;
      float m = -INFINITY, l = 0.f;
      // The stretches before the one in TMEM, against their own maximum.  In local memory (the loops that use it index
      // it), out of the way of the registers: a row of more than kSumKeys keys needs it once a stretch.
      float carry[DP], carry_m = -INFINITY;
      bool carried = false;
      int seen_beat = -1;
      for (int j = 0; j < n;) {
        const int start = j, stop = min(n, j + kTcStretch);
        for (; j < stop; ++j, ++done) {
          ok = __all_sync(~0u, mbar_wait_bounded(s_full + s, done & 1, p.status, j ? kAttnTimeout : 0u));
          if (!ok) break;
          tc_fence_after();
          uint32_t x[128];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32(lanes + c * 32, *reinterpret_cast<uint32_t(*)[32]>(x + c * 32));
          tmem_ld_wait();
          tc_fence_before();
          mbar_arrive(s_free + s);
          if ((begin + j + 1) * kTcKeys > all_see) {
            const int lim = seen - (begin + j) * kTcKeys;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              // bit i: the row sees column 32 c + i (columns that the product left out are never seen)
              const uint32_t sees = lim >= 32 * c + 32 ? ~0u : (lim <= 32 * c ? 0u : (1u << (lim - 32 * c)) - 1u);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(sees & (1u << e))) x[32 * c + e] = 0xff800000u;
            }
          }
          float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 128; c += 8)
#pragma unroll
            for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], __uint_as_float(x[c + 2 * e]), __uint_as_float(x[c + 2 * e + 1]));
          const float top = max3(mx[0], mx[1], max3(mx[2], mx[3], mx[3]));
          const bool move = (top - m) * sl2 > kLazyLog2;  // from -inf too
          if (__any_sync(~0u, move)) {
            const float old = m;
            if (move) m = top;
            const float f = move ? exp2_sfu((old - m) * sl2) : 1.f;
            l *= f;
            if (__any_sync(~0u, move && old != -INFINITY)) {
              ok = __all_sync(~0u, wait(o_done + s, done - 1));
              if (!ok) break;
              tc_fence_after();
              uint32_t o[16];
#pragma unroll 1
              for (int c = 0; c < DP; c += 16) {
                tmem_ld_32x16(o_at + c, o);
                tmem_ld_wait();
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                tmem_st_32x16(o_at + c, o);
              }
              tmem_st_wait();
            }
          }
          const float m0 = m == -INFINITY ? 0.f : m;
          const float top2 = m0 * sl2;
          float base = kProbLog2<T> - top2;
          const bool large = fabsf(top2) > kLargeLog2;  // row by row: no row's result depends on its neighbours
          if (__any_sync(~0u, large)) {
            const float first = large ? m0 : 0.f;
#pragma unroll
            for (int c = 0; c < 128; ++c) x[c] = __float_as_uint(__uint_as_float(x[c]) - first);
            if (large) base = kProbLog2<T>;
          }
          const uint64_t base2 = f2_pack(base, base), sl22 = f2_pack(sl2, sl2);
          uint64_t sum[2] = {0, 0};
#pragma unroll
          for (int c = 0; c < 128; c += 2) {
            float a, b;
            f2_unpack(f2_fma(f2_pack(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), sl22, base2), a, b);
            a = exp2_sfu(a);
            b = exp2_sfu(b);
            sum[(c >> 1) & 1] = f2_add(sum[(c >> 1) & 1], f2_pack(a, b));
            x[c >> 1] = pack16<T>(a, b);
          }
          if (j > start) {  // the last P has been consumed
            ok = __all_sync(~0u, wait(o_done + s, done - 1));
            if (!ok) break;
            tc_fence_after();
          }
          tmem_st_32x32(p_at, x);
          tmem_st_32x32(p_at + 32, x + 32);
          float a, b;
          f2_unpack(f2_add(sum[0], sum[1]), a, b);
          l += a + b;
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(p_full + s);
        }
        if (!ok && j == 0) {
          // The first scores, which may be an item away: as mbar_wait_beat, but out of the loop above (in it, or as a wait of
          // its own before it, 2 to 3 % slower at head size 64).
          const int now = __shfl_sync(~0u, *beat, 0);
          ok = now != seen_beat;
          seen_beat = now;
          if (ok) continue;
          atomicOr(p.status, kAttnTimeout);
        }
        if (!ok || j == n) break;
        ok = __all_sync(~0u, wait(o_done + s, done - 1));  // the next tile's product starts O anew
        if (!ok) break;
        tc_fence_after();
        const float f = moved(carry_m, m, sl2);
        uint32_t o[16];
#pragma unroll 1
        for (int c = 0; c < DP; c += 16) {
          tmem_ld_32x16(o_at + c, o);
          tmem_ld_wait();
#pragma unroll
          for (int e = 0; e < 16; ++e) carry[c + e] = carried ? fmaf(carry[c + e], f, __uint_as_float(o[e])) : __uint_as_float(o[e]);
      }
      carry_m = m;
      carried = true;
      }
      if (ok && n) ok = __all_sync(~0u, wait(o_done + s, done - 1));
      if (ok && valid) {
        tc_fence_after();
        const bool part = kSplit && w.part >= 0;
        const float inv = part ? 1.f : (l == 0.f ? 0.f : 1.f / l);
        const float carry_f = moved(carry_m, m, sl2);
        const int64_t tok = w.q0 + token;
        const int qh = w.head * p.group + row_head;
        const uint64_t dst = reinterpret_cast<uint64_t>(static_cast<T*>(p.out) + tok * p.o_ts + qh * p.o_hs);
        const uint32_t owned = __ballot_sync(~0u, mine);
        const bool patch = *reinterpret_cast<volatile int*>(fixed + (k & 1)) != 0;
        const int* fx = fix + (k & 1) * kFixInts;
        // 64 columns at a time through shared memory (16-byte piece c of row r at c ^ (r % 8)): a store
        // instruction then writes whole 128-byte lines of four rows instead of 16 bytes of 32
        uint8_t* stage = smem + L::kStage + warp * 4096;
        for (int c0 = 0; c0 < p.head_dim && !part; c0 += 64) {
          for (int c = c0; c < min(c0 + 64, p.head_dim); c += 32) {
            uint32_t o[32];
            if (n) {
              tmem_ld_32x32(o_at + c, o);
              tmem_ld_wait();
            } else {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0;
            }
            if (carried) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(fmaf(carry[c + e], carry_f, __uint_as_float(o[e])));
            }
            if (seen == 0) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = 0;
            }
            if (patch) {
#pragma unroll 1
              for (int e = 0; e < 32; ++e) {
                // a loop over registers by number: every value moves up by one place
                const float y = put_back(__uint_as_float(o[0]) * inv, fx, c + e, seen);
#pragma unroll
                for (int i = 0; i < 31; ++i) o[i] = o[i + 1];
                o[31] = __float_as_uint(y);
              }
            }
            float f = patch ? 1.f : inv;
            if constexpr (__is_same(T, __half)) {  // 32 at a time: 90.0 us for 16 maps of 1600 positions, value by value 91.2
              float big = 0.f;
#pragma unroll
              for (int e = 0; e < 32; e += 2) big = max3(big, fabsf(__uint_as_float(o[e])), fabsf(__uint_as_float(o[e + 1])));
              if (big * f > 65504.f) {
#pragma unroll
                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(in_range<T>(__uint_as_float(o[e]) * f));
                f = 1.f;
              }
            }
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                y[e] = pack16<T>(__uint_as_float(o[8 * v + 2 * e]) * f, __uint_as_float(o[8 * v + 2 * e + 1]) * f);
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((((c - c0) / 8 + v) ^ (lane & 7)) << 4)) =
                  make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
          __syncwarp();
          const int piece = lane & 7;
          uint4 y[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
            y[i] = *reinterpret_cast<const uint4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
          }
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int r = 4 * i + (lane >> 3);
            const uint64_t row_dst = __shfl_sync(~0u, dst, r);
            if (((owned >> r) & 1) && c0 + piece * 8 < p.head_dim)
              *reinterpret_cast<uint4*>(row_dst + (c0 + piece * 8) * sizeof(T)) = y[i];
          }
          __syncwarp();
        }
        if (kSplit && part) {  // fp32 sums, 32 columns at a time through the same staging
          float* sums = split.sums + (static_cast<int64_t>(w.part) * 256 + s * 128 + (warp & 3) * 32) * p.head_dim;
          for (int c = 0; c < p.head_dim; c += 32) {
            uint32_t o[32];
            if (n) {
              tmem_ld_32x32(o_at + c, o);
              tmem_ld_wait();
            }
            if (carried) {
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(fmaf(carry[c + e], carry_f, __uint_as_float(o[e])));
            }
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = n && seen ? o[e] : 0u;
            if (patch) {
#pragma unroll 1
              for (int e = 0; e < 32; ++e) {
                const float y = put_back(__uint_as_float(o[0]), fx, c + e, seen);
#pragma unroll
                for (int i = 0; i < 31; ++i) o[i] = o[i + 1];
                o[31] = __float_as_uint(y);
              }
            }
#pragma unroll
            for (int v = 0; v < 8; ++v)
              *reinterpret_cast<uint4*>(stage + lane * 128 + ((v ^ (lane & 7)) << 4)) =
                  make_uint4(o[4 * v], o[4 * v + 1], o[4 * v + 2], o[4 * v + 3]);
            __syncwarp();
            const int piece = lane & 7;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const int r = 4 * i + (lane >> 3);
              if (((owned >> r) & 1) && c + piece * 4 < p.head_dim)
                *reinterpret_cast<uint4*>(sums + r * p.head_dim + c + piece * 4) =
                    *reinterpret_cast<const uint4*>(stage + r * 128 + ((piece ^ (r & 7)) << 4));
            }
            __syncwarp();
          }
          if (mine) *reinterpret_cast<float2*>(split.stats + (static_cast<int64_t>(w.part) * 256 + s * 128 + row) * 2) = make_float2(m, l);
        } else if (mine && p.lse) {
          p.lse[tok * p.q_heads + qh] = l == 0.f ? -INFINITY : fmaf(m, p.scale, logf(l * kProbUnit<T>));
        }
        tc_fence_before();  // these reads of O before the next item's first product into it
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(w_empty + (k & 1));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the split items: a block takes 16 of an item's 256 rows, a thread 8 columns of a row.
constexpr int kTcJoinThreads = 256, kTcJoinRows = 16;
template <typename T>
__global__ void __launch_bounds__(kTcJoinThreads) attention_tc_join_kernel(const AttnParams p, const TcSplit split) {
  grid_dep_launch();
  grid_dep_wait();
  const int tokens = kTcRows / p.group, vecs = p.head_dim / 8, items = *split.split_items;
  for (int n = blockIdx.x; n < items; n += gridDim.x) {
    const JoinHead item = split.heads[n];
    for (int i = threadIdx.x; i < kTcJoinRows * vecs; i += kTcJoinThreads) {
      const int r = blockIdx.y * kTcJoinRows + i / vecs, in_tile = r & 127, row_token = in_tile / p.group;
      const int token = (r >> 7) * tokens + row_token;
      if (row_token >= tokens || token >= item.rows) continue;
      auto row_of = [&](int k) { return (static_cast<int64_t>(split.bases[k]) + n) * 256 + r; };
      join_row<T>(p, split.sums, split.stats, item.parts, row_of, i % vecs * 8, item.q0 + token,
                  item.head * p.group + in_tile % p.group);
    }
  }
}

}  // namespace aexrt
