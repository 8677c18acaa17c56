// Attention of a few query rows per sequence over the paged cache: one new token, or some drafted ones.
//
// The rows of a sequence that share a key/value head (new tokens x query heads of the head, at most
// 64) form MT tiles of 16 for the warp-level tensor instructions; each cached K and V row is read once from
// memory, which is what bounds the kernel.  Work is a list of units, one per sequence, head and 64 keys, cut into
// equal runs over a fixed grid: any mix of lengths fills the GPU, with one long sequence as with
// many short ones.  A (sequence, head) that lies inside one run is finished there; one that is cut
// leaves each part's unnormalised sum with its maximum and normaliser in the workspace, and a second
// launch joins the parts in a fixed order, so results do not depend on timing.
//
// Four warps compute: MT over the row tiles, 4 / MT over the keys of a stage; each keeps its own
// running maximum and the accumulators of its keys, joined once per (sequence, head) through shared
// memory.  A fifth warp loads, one TMA box per page, ahead across the sequences' borders: with the
// loads and their page lookups in the computing warps (cp.async), those spent 945 instructions a unit and
// the kernel reached 3.1 TB/s at 64 x 4096 keys, 8 heads of 128; now 174 to 181 us, 5.9 to 6.2 TB/s, which is what the
// loads alone reach.  With 33 to 64 rows the warps' products bound it, at 3.1 to 3.5 TB/s.
#pragma once
#include <climits>

#include "attention_join.cuh"

namespace aexrt {

constexpr int kRowsCompute = 128, kRowsThreads = kRowsCompute + 32;
constexpr int kRowsKeys = 64;     // keys of a unit
constexpr int kRowsMinUnits = 2;  // units of a run at least: shorter runs cost more in the joining than they save

template <int DP>
constexpr int rows_stages() { return DP == 128 ? 3 : 6; }

template <int DP>
struct RowsSmem {
  static constexpr int kHalf = kRowsKeys * DP * 2, kStage = 2 * kHalf;  // K, V
  static_assert(kStage == 4 * 16 * DP * 4, "a stage holds the four warps' accumulators");
  static constexpr int kStat = rows_stages<DP>() * kStage;              // m, l of each warp's rows
  static constexpr int kPrev = kStat + 4 * 16 * 2 * 4;                  // m, l of each row's stretches before, in turn
  static constexpr int kFix = kPrev + 2 * 64 * 2 * 4;
  static constexpr int kBars = kFix + kFixInts * 4 + 16;
  static constexpr int kBytes = kBars + 2 * rows_stages<DP>() * 8;
};

struct RowsParams {
  AttnParams a;
  JoinHead* runs;   // [grid]: of the (sequence, head) that run c goes on with, when it is the first to do so
  float* parts;     // [grid][2][rows][head_dim]: first a run's part of a (sequence, head) begun before it, then of one that goes on behind it
  float* stats;     // [grid][2][rows][2]: maximum (raw score units), normaliser
  int rows;         // max_q * group
};

template <bool kTrans>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Tiles of a sequence per head: one at least when it has query rows, so that empty rows are written too.
__device__ __forceinline__ int rows_tiles(const AttnParams& p, int s) {
  if (min(q_len(p, s), p.max_q) == 0) return 0;
  return max(1, (k_len<true>(p, s) + kRowsKeys - 1) / kRowsKeys);
}

// A place in the list of units, with what its sequence needs.
struct RowsPlace {
  int seq, head, tile, tiles, len_k;
  __device__ __forceinline__ void enter(const AttnParams& p) {  // the first sequence from seq on that has units
    tiles = 0;
    while (seq < p.num_seqs && (tiles = rows_tiles(p, seq)) == 0) ++seq;
    len_k = seq < p.num_seqs ? k_len<true>(p, seq) : 0;
  }
  __device__ __forceinline__ void advance(const AttnParams& p) {
    if (++tile < tiles) return;
    tile = 0;
    if (++head < p.kv_heads) return;
    head = 0;
    ++seq;
    enter(p);
  }
};

// `units` cut into `runs`: the first units % runs of them are one longer.
struct RowsCut {
  int64_t per;
  int runs, more;
  __device__ __forceinline__ RowsCut(int64_t units, int grid) {
    runs = static_cast<int>(min(static_cast<int64_t>(grid), (units + kRowsMinUnits - 1) / kRowsMinUnits));
    if (units >> 31) {
      per = units / max(runs, 1);
      more = static_cast<int>(units % max(runs, 1));
    } else {  // the usual case: a 32-bit division
      const uint32_t n = static_cast<uint32_t>(units), r = static_cast<uint32_t>(max(runs, 1));
      per = n / r;
      more = static_cast<int>(n % r);
    }
  }
  __device__ __forceinline__ int64_t start(int c) const { return c * per + min(c, more); }
};

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(kRowsThreads, 2)
    attention_rows_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                          const RowsParams rp) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using L = RowsSmem<DP>;
  constexpr int kStages = rows_stages<DP>(), kKeyWarps = 4 / MT, kWarpKeys = kRowsKeys / kKeyWarps;
  constexpr int kHalves = DP / 64, kHalfBytes = kRowsKeys * 128;  // a tile: [column half][key][128 bytes], swizzled
  const AttnParams& p = rp.a;
  float* stat = reinterpret_cast<float*>(smem + L::kStat);
  float2* prev = reinterpret_cast<float2*>(smem + L::kPrev);
  int* fix = reinterpret_cast<int*>(smem + L::kFix);
  int* fixed = fix + kFixInts;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t* empty = full + kStages;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = warp % MT, wk = warp / MT;
  if (tid == 0) {
    for (int i = 0; i < kStages; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 4);
    }
    fence_mbar_init();
  }
  grid_dep_wait();

  // ---- this CTA's run: the units of every sequence are summed, then the one that holds the first unit found
  for (int i = tid; i < kFixInts; i += kRowsThreads) fix[i] = INT_MAX;
  if (tid == 0) *fixed = 0;
  constexpr int kWarps = kRowsThreads / 32;
  __shared__ int64_t sums[kWarps];
  __shared__ RowsPlace found;
  auto up_to = [&](int64_t n) {  // inclusive sum over the warp
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t z = __shfl_up_sync(~0u, n, o);
      if (lane >= o) n += z;
    }
    return n;
  };
  // one sequence per thread, or one block of sequences when there are more of them than threads
  const int each = (p.num_seqs + kRowsThreads - 1) / kRowsThreads, s0 = min(tid * each, p.num_seqs);
  const int s1 = min(s0 + each, p.num_seqs);
  int64_t mine = 0;
  for (int s = s0; s < s1; ++s) mine += rows_tiles(p, s);
  const int64_t incl = up_to(mine);
  if (lane == 31) sums[warp] = incl;
  __syncthreads();
  int64_t units = 0, before = incl - mine;  // tiles, of all sequences and of those before this thread's
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    if (i < warp) before += sums[i];
    units += sums[i];
  }
  units *= p.kv_heads;
  before *= p.kv_heads;
  const RowsCut cut(units, gridDim.x);
  const int64_t start = cut.start(blockIdx.x);
  const int count = static_cast<int>(cut.start(blockIdx.x + 1) - start);
  if (static_cast<int>(blockIdx.x) >= cut.runs) {
    if (tid == 0) rp.runs[blockIdx.x].parts = 0;
    return;
  }
  if (start >= before && start < before + mine * p.kv_heads) {
    for (int s = s0; s < s1; ++s) {
      const int n = rows_tiles(p, s);
      const int64_t here = static_cast<int64_t>(n) * p.kv_heads;
      if (start < before + here) {
        const int64_t off = start - before;
        found.seq = s;
        if (off >> 31) {
          found.head = static_cast<int>(off / n);
          found.tile = static_cast<int>(off % n);
        } else {
          found.head = static_cast<int>(static_cast<uint32_t>(off) / static_cast<uint32_t>(n));
          found.tile = static_cast<int>(static_cast<uint32_t>(off) % static_cast<uint32_t>(n));
        }
        found.tiles = n;
        found.len_k = k_len<true>(p, s);
        break;
      }
      before += here;
    }
  }
  __syncthreads();
  RowsPlace at = found;

  if (warp == 4) {
    // ---- loads: a lane has one box, a page's rows of one column half of K or V
    const int box_rows = min(1 << p.page_shift, kRowsKeys), boxes = kRowsKeys / box_rows;
    const int box = lane % boxes, half = (lane / boxes) % kHalves, is_v = lane / (boxes * kHalves);
    const bool on = is_v < 2;
    bool ok = true;
    const RowsPlace begin = at;
    int u = 0;
    for (; u < count; ++u) {
      const int stage = u % kStages;
      int page = p.no_page;
      const int key = at.tile * kRowsKeys + box * box_rows;
      if (on && key < at.len_k) {
        const int id = __ldg(p.block_table + at.seq * p.table_stride + (key >> p.page_shift));
        if (id >= 0 && id < p.kv_tokens) page = id; else atomicOr(p.status, kAttnBadPage);
      }
      ok = __all_sync(~0u, mbar_wait_bounded(empty + stage, ((u / kStages) & 1) ^ 1, p.status, kAttnTimeout));
      if (!ok) break;
      if (lane == 0) mbar_arrive_expect_tx(full + stage, L::kStage);
      __syncwarp();
      if (on)
        tma_load_4d(smem + stage * L::kStage + is_v * L::kHalf + half * kHalfBytes + box * box_rows * 128,
                    is_v ? &v_map : &k_map, full + stage, half * 64, at.head, key & ((1 << p.page_shift) - 1), page);
      at.advance(p);
    }
    if (lane == 0) {
      // is this run the first that goes on with its first (sequence, head)?  Then it heads the joining.
      const int c = blockIdx.x;
      const int64_t first = start - begin.tile, end = first + begin.tiles;
      JoinHead r = {};
      if (begin.tile > 0 && cut.start(c - 1) <= first) {
        r.parts = 1;
        while (c + r.parts - 1 < cut.runs && cut.start(c + r.parts - 1) < end) ++r.parts;
        r.rows = min(q_len(p, begin.seq), p.max_q) * p.group;
        r.q0 = q_start(p, begin.seq);
        r.head = begin.head;
      }
      rp.runs[c] = r;
    }
    // after a wait that gave up, the loads in flight land before the block ends: the last ones of each stage
    for (int i = max(0, u - kStages); i < u && !ok; ++i)
      mbar_wait_bounded(full + i % kStages, (i / kStages) & 1, p.status, kAttnTimeout);
    grid_dep_launch();
    return;
  }

  const float sl2 = p.scale * 1.4426950408889634f;
  const int steps = (p.head_dim + 15) / 16;
  const int g = lane >> 2, quad = lane & 3;

  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];
  constexpr int kStretch = kSumKeys / kWarpKeys;  // units that a warp sums at a time
  int seen[2], common = 0, rows = 0, q0 = 0, len_q = 0;
  bool fresh = true, dead = false;
  int part_first = at.tile;  // first tile of the current (sequence, head) that this run takes

  for (int u = 0; u < count; ++u) {
    if (fresh) {  // a new (sequence, head): its rows of q into registers
      len_q = q_len(p, at.seq);
      q0 = q_start(p, at.seq);
      rows = min(len_q, p.max_q) * p.group;
      common = keys_seen(0, len_q, at.len_k, p.causal);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = wr * 16 + g + 8 * e, token = r / p.group;
        const bool on = r < rows;
        seen[e] = on ? keys_seen(token, len_q, at.len_k, p.causal) : 0;
        // rows and columns that are not there read the first ones and count 0: no branch between the loads
        const int64_t from = on ? token * p.q_ts + (r % p.group) * p.q_hs : 0;
        const T* src = static_cast<const T*>(p.q) + q0 * p.q_ts + at.head * p.group * p.q_hs + from;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const int d = k * 16 + f * 8 + quad * 2;
            const uint32_t x = __ldg(reinterpret_cast<const uint32_t*>(src + (d < p.head_dim ? d : 0)));
            qf[k][e + 2 * f] = on && d < p.head_dim ? x : 0u;
          }
        m[e] = -INFINITY;
        l[e] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
      fresh = false;
    }
    // after a wait that gave up, the warp goes on without waiting (the status tells): the barriers between the
    // warps still see all of them
    if (!dead) dead = !mbar_wait_bounded(full + u % kStages, (u / kStages) & 1, p.status, kAttnTimeout);
    __syncwarp();
    uint8_t* stage = smem + (u % kStages) * L::kStage;
    const uint32_t ks = smem_u32(stage), vs = ks + L::kHalf;
    const int key0 = at.tile * kRowsKeys;
    const int last = at.len_k - key0;
    const bool clean = last < kRowsKeys || common - key0 < kRowsKeys;
    if (clean) {
      // P is 0 where a row does not see a key, but 0 * inf and 0 * NaN are not: rows behind the last key
      // become zeros, and non-finite values of keys that only some rows see are taken out and put back
      // into the outputs of the rows that do
      for (int i = tid; i < kRowsKeys * 8 * kHalves; i += kRowsCompute) {
        const int r = (i >> 3) % kRowsKeys, half = i / (kRowsKeys * 8);
        uint4* v = reinterpret_cast<uint4*>(stage + L::kHalf + half * kHalfBytes + r * 128) + (i & 7);
        if (r >= last) {
          *v = make_uint4(0, 0, 0, 0);
        } else if (r >= common - key0) {
          const uint4 x = *v;
          if (non_finite_bits<T>(x.x) | non_finite_bits<T>(x.y) | non_finite_bits<T>(x.z) | non_finite_bits<T>(x.w)) {
            *v = take_non_finite<T>(x, key0 + r, half * 64 + ((i & 7) ^ (r & 7)) * 8, fix);
            *fixed = 1;
          }
        }
      }
      fence_proxy_async_smem();  // before a later TMA write of this stage
      named_bar_sync(1, kRowsCompute);
    }

    // ---- S = Q K^T for this warp's keys, 16 at a time: all of their K first, then two sums over
    // the even and the odd steps, so that neither the loads nor the sums wait for one another
    float s[kWarpKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kWarpKeys / 16; ++n) {
      const int key = wk * kWarpKeys + n * 16 + ((lane >> 4) << 3) + (lane & 7);
      uint32_t b[DP / 16][4];
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const int c = 2 * k + ((lane >> 3) & 1);
        ldmatrix4<false>(ks + (c >> 3) * kHalfBytes + key * 128 + (((c & 7) ^ (key & 7)) << 4), b[k]);
      }
      float t[2][2][4] = {};
#pragma unroll
      for (int k = 0; k < DP / 16; ++k)
        if (k < steps) {
          mma_16816<T>(t[k & 1][0], qf[k], b[k][0], b[k][1]);
          mma_16816<T>(t[k & 1][1], qf[k], b[k][2], b[k][3]);
        }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[2 * n][e] = t[0][0][e] + t[1][0][e];
        s[2 * n + 1][e] = t[0][1][e] + t[1][1][e];
      }
    }
    const int keyw = key0 + wk * kWarpKeys;
    if (keyw + kWarpKeys > common) {
#pragma unroll
      for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (keyw + n * 8 + quad * 2 + (e & 1) >= seen[e >> 1]) s[n][e] = -INFINITY;
    }
    // ---- running maximum and probabilities
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 1));
      top[e] = fmaxf(top[e], __shfl_xor_sync(~0u, top[e], 2));
    }
    const bool move0 = (top[0] - m[0]) * sl2 > kLazyLog2, move1 = (top[1] - m[1]) * sl2 > kLazyLog2;
    if (__any_sync(~0u, move0 || move1)) {
      float f[2] = {1.f, 1.f};
      if (move0) { f[0] = exp2_sfu((m[0] - top[0]) * sl2); m[0] = top[0]; }
      if (move1) { f[1] = exp2_sfu((m[1] - top[1]) * sl2); m[1] = top[1]; }
      l[0] *= f[0];
      l[1] *= f[1];
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] *= f[e >> 1];
    }
    const float m0[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2_sfu(fmaf(s[n][e] - m0[e >> 1], sl2, kProbLog2<T>));  // the difference first: finite for any finite scores
        l[e >> 1] += s[n][e];
      }
    // ---- O += P V
#pragma unroll
    for (int k = 0; k < kWarpKeys / 16; ++k) {
      const uint32_t a[4] = {pack16<T>(s[2 * k][0], s[2 * k][1]), pack16<T>(s[2 * k][2], s[2 * k][3]),
                             pack16<T>(s[2 * k + 1][0], s[2 * k + 1][1]), pack16<T>(s[2 * k + 1][2], s[2 * k + 1][3])};
      const int key = wk * kWarpKeys + k * 16 + (((lane >> 3) & 1) << 3) + (lane & 7);
#pragma unroll
      for (int n = 0; n < DP / 16; ++n) {
        if (n < steps) {
          uint32_t b[4];
          const int c = 2 * n + (lane >> 4);
          ldmatrix4<true>(vs + (c >> 3) * kHalfBytes + key * 128 + (((c & 7) ^ (key & 7)) << 4), b);
          mma_16816<T>(o[2 * n], a, b[0], b[1]);
          mma_16816<T>(o[2 * n + 1], a, b[2], b[3]);
        }
      }
    }


    // ---- the end of a (sequence, head), of the run or of a stretch: join the key warps, write
    if (at.tile + 1 == at.tiles || u + 1 == count || (at.tile + 1 - part_first) % kStretch == 0) {
      const bool whole = part_first == 0 && at.tile + 1 == at.tiles;
      const int slot = 2 * blockIdx.x + (part_first == 0 ? 1 : 0);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        l[e] += __shfl_xor_sync(~0u, l[e], 1);
        l[e] += __shfl_xor_sync(~0u, l[e], 2);
        if (quad == 0) {
          stat[(warp * 16 + g + 8 * e) * 2] = m[e];
          stat[(warp * 16 + g + 8 * e) * 2 + 1] = l[e];
        }
      }
      named_bar_sync(1, kRowsCompute);  // no warp reads the stage's K and V any more: it holds the accumulators now
      const bool patch = *fixed != 0;
      // A stretch that is not the end goes to the workspace as a part does, its maxima and normalisers to one half of
      // `prev`; the next one is added to it there, from that half to the other.  (As sums that the warps keep beside o this
      // made 20 rows 17 % and 64 rows 29 % slower.)
      const int ends = (at.tile - part_first) / kStretch;  // of stretches before
      const bool more = at.tile + 1 < at.tiles && u + 1 < count;
      // [warp][row][DP] floats, columns swizzled by the row so that a warp's stores spread over the banks
      float* join = reinterpret_cast<float*>(stage);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (wr * 16 + g + 8 * e < rows) {
          float all = -INFINITY;  // the row's maximum over the key warps
#pragma unroll
          for (int w = 0; w < kKeyWarps; ++w) all = fmaxf(all, stat[((w * MT + wr) * 16 + g + 8 * e) * 2]);
          const float f = moved(m[e], all, sl2);
          float* row = join + (warp * 16 + g + 8 * e) * DP;
#pragma unroll
          for (int n = 0; n < DP / 8; ++n)
            *reinterpret_cast<float2*>(row + ((n * 8 + quad * 2) ^ (g << 3))) = make_float2(o[n][2 * e] * f, o[n][2 * e + 1] * f);
        }
      }
      named_bar_sync(1, kRowsCompute);
      constexpr int kVecs = DP / 8;
      for (int i = tid; i < rows * kVecs; i += kRowsCompute) {  // 8 columns of one row
        const int r = i / kVecs, c = i % kVecs * 8;
        if (c >= p.head_dim) continue;
        float y[8] = {}, all = -INFINITY, norm = 0.f;
#pragma unroll
        for (int w = 0; w < kKeyWarps; ++w) all = fmaxf(all, stat[((w * MT + (r >> 4)) * 16 + (r & 15)) * 2]);
#pragma unroll
        for (int w = 0; w < kKeyWarps; ++w) {
          const int at_row = (w * MT + (r >> 4)) * 16 + (r & 15);
          const float2 st = *reinterpret_cast<const float2*>(stat + at_row * 2);
          norm += st.y * moved(st.x, all, sl2);  // NaN from a warp whose scores are all NaN (maximum -inf) too
          const float4* src = reinterpret_cast<const float4*>(join + at_row * DP + (c ^ ((r & 7) << 3)));
          const float4 a = src[0], b = src[1];
          y[0] += a.x, y[1] += a.y, y[2] += a.z, y[3] += a.w, y[4] += b.x, y[5] += b.y, y[6] += b.z, y[7] += b.w;
        }
        const int token = r / p.group, qh = at.head * p.group + r % p.group;
        const int64_t part = static_cast<int64_t>(slot) * rp.rows + r;
        if (patch) {
          const int sees = keys_seen(token, len_q, at.len_k, p.causal);
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = put_back(y[e], fix, c + e, sees);
        }
        if (ends) {  // this thread's own sums of the stretches before
          const float2 st = prev[((ends - 1) & 1) * 64 + r];
          const float top = fmaxf(all, st.x), f0 = moved(st.x, top, sl2), f1 = moved(all, top, sl2);
          const float* sum = rp.parts + part * p.head_dim + c;
#pragma unroll
          for (int e = 0; e < 8; ++e) y[e] = fmaf(sum[e], f0, y[e] * f1);
          norm = fmaf(st.y, f0, norm * f1);
          all = top;
        }
        const float inv = !whole ? 1.f : (norm == 0.f ? 0.f : 1.f / norm);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] *= inv;
        if (whole) {
          *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (q0 + token) * p.o_ts + qh * p.o_hs + c) =
              make_uint4(pack_out<T>(y[0], y[1]), pack_out<T>(y[2], y[3]), pack_out<T>(y[4], y[5]), pack_out<T>(y[6], y[7]));
          if (c == 0 && p.lse)
            p.lse[static_cast<int64_t>(q0 + token) * p.q_heads + qh] = norm == 0.f ? -INFINITY : fmaf(all, p.scale, logf(norm * kProbUnit<T>));
        } else {
          float4* dst = reinterpret_cast<float4*>(rp.parts + part * p.head_dim + c);
          dst[0] = make_float4(y[0], y[1], y[2], y[3]);
          dst[1] = make_float4(y[4], y[5], y[6], y[7]);
          if (c == 0) {
            if (more) prev[(ends & 1) * 64 + r] = make_float2(all, norm);
            else *reinterpret_cast<float2*>(rp.stats + part * 2) = make_float2(all, norm);
          }
        }
      }
      if (patch) {
        named_bar_sync(1, kRowsCompute);
        for (int i = tid; i < kFixInts; i += kRowsCompute) fix[i] = INT_MAX;
        if (tid == 0) *fixed = 0;
      }
      if (!more) part_first = 0;  // of the next (sequence, head), if this run takes one
      fence_proxy_async_smem();      // these accesses before the stage's next TMA write
      named_bar_sync(1, kRowsCompute);  // and before the next statistics
      fresh = true;
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(empty + u % kStages);
    at.advance(p);
  }
  grid_dep_launch();
}

// Joins the parts of every (sequence, head) that was cut: block c - 1 takes the one that run c heads.
// A thread has 8 columns of a row.
template <typename T>
__global__ void __launch_bounds__(kRowsCompute) attention_rows_join_kernel(const RowsParams rp) {
  grid_dep_launch();
  grid_dep_wait();
  const AttnParams& p = rp.a;
  const int c = blockIdx.x + 1;
  const JoinHead run = rp.runs[c];
  if (run.parts == 0) return;
  const int vecs = p.head_dim / 8;
  for (int i = threadIdx.x; i < run.rows * vecs; i += kRowsCompute) {
    const int r = i / vecs;
    // part k is run c - 1 + k's: the second slot of the first run, the first slot of the others
    auto row_of = [&](int k) { return (static_cast<int64_t>(2 * (c - 1 + k) + (k == 0 ? 1 : 0))) * rp.rows + r; };
    join_row<T>(p, rp.parts, rp.stats, run.parts, row_of, i % vecs * 8, run.q0 + r / p.group, run.head * p.group + r % p.group);
  }
}

}  // namespace aexrt
