// Attention of a few query rows per sequence over the paged cache: one new token, or some drafted ones.
//
// The rows of a sequence that share a key/value head (new tokens x query heads of the head, at most
// 64) form MT tiles of 16 for the warp-level tensor instructions; each cached K and V row is read once from
// memory, which is what bounds the kernel.  Work is a list of units, one per sequence, head and 64 keys, cut into
// equal runs over a fixed grid: any mix of lengths fills the GPU, with one long sequence as with
// many short ones.  A run's loads (cp.async, a ring of stages) go on across the sequences' borders.  A (sequence,
// head) that lies inside one run is finished there; one that is cut leaves each part's
// unnormalised sum with its maximum and normaliser in the workspace, and a second launch joins the
// parts in a fixed order, so results do not depend on timing.
//
// Four warps: MT over the row tiles, 4 / MT over the keys of a stage; each keeps its own running
// maximum and the accumulators of its keys, joined once per (sequence, head) through shared memory.
#pragma once
#include <climits>

#include "attention_math.cuh"

namespace aexrt {

constexpr int kRowsThreads = 128;
constexpr int kRowsKeys = 64;     // keys of a unit
constexpr int kRowsMinUnits = 2;  // units of a run at least: shorter runs cost more in the joining than they save

template <int DP>
constexpr int rows_stages() { return DP == 128 ? 3 : 6; }

template <int DP>
struct RowsSmem {
  static constexpr int kHalf = kRowsKeys * DP * 2, kStage = 2 * kHalf;  // K, V
  static constexpr int kPitch = 36;                                     // floats of a row of the joining buffer
  static constexpr int kJoin = rows_stages<DP>() * kStage;
  static constexpr int kStat = kJoin + 4 * 16 * kPitch * 4;             // m, l of each warp's rows
  static constexpr int kFix = kStat + 4 * 16 * 2 * 4;
  static constexpr int kBytes = kFix + 3 * 128 * 4 + 16;
};

// What a run leaves for the joining: its first unit's place.
struct RowsRun {
  int64_t start, units;  // first unit of the run, units of the whole call
  int seq, head, tile, tiles;  // the first unit's sequence, head, tile, and the tiles of that (sequence, head)
  int runs, pad[3];      // runs of the call
};
static_assert(sizeof(RowsRun) == 48, "16-byte multiple");

struct RowsParams {
  AttnParams a;
  RowsRun* runs;    // [grid]
  float* parts;     // [grid][2][rows][head_dim]: first a run's part of a (sequence, head) begun before it, then of one that goes on behind it
  float* stats;     // [grid][2][rows][2]: maximum (raw score units), normaliser
  int rows;         // max_q * group
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

template <bool kTrans>
__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  if constexpr (kTrans)
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
  else
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}

template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (__is_same(T, __nv_bfloat16))
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
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

// First unit of run c when `units` are cut into `runs`.
__device__ __forceinline__ int64_t run_start(int64_t units, int runs, int c) { return units * c / runs; }

template <typename T, int DP, int MT>
__global__ void __launch_bounds__(kRowsThreads, 2) attention_rows_kernel(const RowsParams rp) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using L = RowsSmem<DP>;
  constexpr int kStages = rows_stages<DP>(), kKeyWarps = 4 / MT, kWarpKeys = kRowsKeys / kKeyWarps;
  constexpr int kPieces = DP / 8;                                       // 16-byte pieces of a padded row
  constexpr int kRowStep = kRowsThreads / kPieces, kRowLoads = kRowsKeys / kRowStep;
  const AttnParams& p = rp.a;
  float* join = reinterpret_cast<float*>(smem + L::kJoin);
  float* stat = reinterpret_cast<float*>(smem + L::kStat);
  int* fix = reinterpret_cast<int*>(smem + L::kFix);
  int* fixed = fix + 3 * 128;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int wr = warp % MT, wk = warp / MT;
  grid_dep_wait();

  // ---- this CTA's run
  for (int i = tid; i < 3 * 128; i += kRowsThreads) fix[i] = INT_MAX;
  if (tid == 0) *fixed = 0;
  int64_t units, mine_start;
  int runs;
  RowsPlace at;
  {
    __shared__ int64_t sums[kRowsThreads / 32];
    __shared__ RowsPlace found;
    int64_t mine = 0;
    for (int s = tid; s < p.num_seqs; s += kRowsThreads) mine += rows_tiles(p, s);
#pragma unroll
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(~0u, mine, o);
    if (lane == 0) sums[warp] = mine;
    __syncthreads();
    units = (sums[0] + sums[1] + sums[2] + sums[3]) * p.kv_heads;
    runs = static_cast<int>(min(static_cast<int64_t>(gridDim.x), (units + kRowsMinUnits - 1) / kRowsMinUnits));
    const int c = blockIdx.x;
    mine_start = c < runs ? run_start(units, runs, c) : units;
    if (c < runs && warp == 0) {  // the sequence that holds unit mine_start
      int64_t before = 0;
      for (int base = 0; base < p.num_seqs; base += 32) {
        const int s = base + lane;
        const int n = s < p.num_seqs ? rows_tiles(p, s) : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int z = __shfl_up_sync(~0u, sum, o);
          if (lane >= o) sum += z;
        }
        const uint32_t past = __ballot_sync(~0u, (before + sum) * p.kv_heads > mine_start);
        if (past) {
          const int src = __ffs(past) - 1;
          if (lane == src) {
            const int64_t off = mine_start - (before + sum - n) * p.kv_heads;
            found.seq = s;
            found.head = static_cast<int>(off / n);
            found.tile = static_cast<int>(off % n);
            found.tiles = n;
            found.len_k = k_len<true>(p, s);
          }
          break;
        }
        before += __shfl_sync(~0u, sum, 31);
      }
    }
    __syncthreads();
    at = found;
    if (tid == 0) {
      RowsRun r = {};
      r.start = mine_start;
      r.units = units;
      r.runs = runs;
      if (c < runs) {
        r.seq = at.seq;
        r.head = at.head;
        r.tile = at.tile;
        r.tiles = at.tiles;
      }
      rp.runs[c] = r;
    }
    if (c >= runs) return;
  }
  const int count = static_cast<int>(run_start(units, runs, blockIdx.x + 1) - mine_start);

  // ---- loads: thread = one 16-byte piece of every kRowStep-th key
  const int piece = tid % kPieces, row0 = tid / kPieces;
  const bool in_row = piece * 8 < p.head_dim;                       // else zeros, up to a whole step of 16
  const bool pad = !in_row && piece < (p.head_dim + 15) / 16 * 2;
  RowsPlace ahead = at;
  auto load = [&](int stage) {
    const int64_t table = static_cast<int64_t>(ahead.seq) * p.table_stride;
    const uint32_t dst = smem_u32(smem) + stage * L::kStage;
    if (in_row || pad) {
#pragma unroll
      for (int i = 0; i < kRowLoads; ++i) {
        const int r = row0 + i * kRowStep, key = ahead.tile * kRowsKeys + r;
        int page = -1;
        if (key < ahead.len_k) {
          page = __ldg(p.block_table + table + (key >> p.page_shift));
          if (page < 0 || page >= p.kv_tokens) {
            page = -1;
            atomicOr(p.status, kAttnBadPage);
          }
        }
        const bool there = in_row && page >= 0;
        const int64_t in_page = key & ((1 << p.page_shift) - 1);
        const int64_t ko = there ? page * p.k_ps + in_page * p.k_ts + ahead.head * p.k_hs + piece * 8 : 0;
        const int64_t vo = there ? page * p.v_ps + in_page * p.v_ts + ahead.head * p.v_hs + piece * 8 : 0;
        const uint32_t to = dst + r * (DP * 2) + ((piece ^ (r & 7)) << 4);
        cp_async16(to, static_cast<const T*>(p.k) + ko, there);
        cp_async16(to + L::kHalf, static_cast<const T*>(p.v) + vo, there);
      }
    }
    ahead.advance(p);
  };
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < count) load(i);
    cp_async_commit();
  }

  const float scale = fmaxf(p.scale, 1e-30f);  // 0 would make NaN of a masked score's -inf
  const float sl2 = scale * 1.4426950408889634f;
  const int steps = (p.head_dim + 15) / 16;
  const int g = lane >> 2, quad = lane & 3;

  uint32_t qf[DP / 16][4];
  float o[DP / 8][4];
  float m[2], l[2];
  int seen[2], common = 0, rows = 0, q0 = 0;
  bool fresh = true;
  int part_first = at.tile;  // first tile of the current (sequence, head) that this run takes

  for (int u = 0; u < count; ++u) {
    if (fresh) {  // a new (sequence, head): its rows of q into registers
      const int len_q = q_len(p, at.seq);
      q0 = q_start(p, at.seq);
      rows = min(len_q, p.max_q) * p.group;
      common = keys_seen(0, len_q, at.len_k, p.causal);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int r = wr * 16 + g + 8 * e, token = r / p.group;
        const bool on = r < rows;
        seen[e] = on ? keys_seen(token, len_q, at.len_k, p.causal) : 0;
        const T* src = static_cast<const T*>(p.q) + (q0 + token) * p.q_ts + (at.head * p.group + r % p.group) * p.q_hs;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const int d = k * 16 + f * 8 + quad * 2;
            qf[k][e + 2 * f] = on && d < p.head_dim ? *reinterpret_cast<const uint32_t*>(src + d) : 0u;
          }
        m[e] = -INFINITY;
        l[e] = 0.f;
      }
#pragma unroll
      for (int n = 0; n < DP / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][e] = 0.f;
      part_first = at.tile;
      fresh = false;
    }
    cp_async_wait<kStages - 2>();
    __syncthreads();
    {
      const int next = u + kStages - 1;
      if (next < count) load(next % kStages);
      cp_async_commit();
    }
    uint8_t* stage = smem + (u % kStages) * L::kStage;
    const uint32_t ks = smem_u32(stage), vs = ks + L::kHalf;
    const int key0 = at.tile * kRowsKeys;
    if (key0 + kRowsKeys > common && common < at.len_k) {
      // P is 0 where a row does not see a key, but 0 * inf and 0 * NaN are not: non-finite values of
      // keys that only some rows see are taken out here and put back into the rows that do
      const int lo = max(0, common - key0), hi = min(kRowsKeys, at.len_k - key0);
      for (int r = lo + row0; r < hi; r += kRowStep)
        if (in_row) {
          uint4* v = reinterpret_cast<uint4*>(stage + L::kHalf + r * (DP * 2) + ((piece ^ (r & 7)) << 4));
          const uint4 x = *v;
          if (non_finite_bits<T>(x.x) | non_finite_bits<T>(x.y) | non_finite_bits<T>(x.z) | non_finite_bits<T>(x.w)) {
            *v = take_non_finite<T>(x, key0 + r, piece * 8, fix);
            *fixed = 1;
          }
        }
      __syncthreads();
    }

    // ---- S = Q K^T for this warp's keys
    float s[kWarpKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
    for (int k = 0; k < DP / 16; ++k) {
      if (k < steps) {
#pragma unroll
        for (int n = 0; n < kWarpKeys / 16; ++n) {
          const int key = wk * kWarpKeys + n * 16 + ((lane >> 4) << 3) + (lane & 7), c = 2 * k + ((lane >> 3) & 1);
          uint32_t b[4];
          ldmatrix4<false>(ks + key * (DP * 2) + ((c ^ (key & 7)) << 4), b);
          mma_16816<T>(s[2 * n], qf[k], b[0], b[1]);
          mma_16816<T>(s[2 * n + 1], qf[k], b[2], b[3]);
        }
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
    const float base[2] = {m[0] == -INFINITY ? 0.f : -m[0] * sl2, m[1] == -INFINITY ? 0.f : -m[1] * sl2};
#pragma unroll
    for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[n][e] = exp2_sfu(fmaf(s[n][e], sl2, base[e >> 1]));
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
          ldmatrix4<true>(vs + key * (DP * 2) + (((2 * n + (lane >> 4)) ^ (key & 7)) << 4), b);
          mma_16816<T>(o[2 * n], a, b[0], b[1]);
          mma_16816<T>(o[2 * n + 1], a, b[2], b[3]);
        }
      }
    }

    // ---- the end of a (sequence, head), or of the run: join the key warps, write
    if (at.tile + 1 == at.tiles || u + 1 == count) {
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
      __syncthreads();
      const bool patch = *fixed != 0;
      // every thread scales its accumulators to its rows' maximum over the key warps
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float all = -INFINITY;
#pragma unroll
        for (int w = 0; w < kKeyWarps; ++w) all = fmaxf(all, stat[((w * MT + wr) * 16 + g + 8 * e) * 2]);
        f[e] = m[e] == -INFINITY ? 0.f : exp2_sfu((m[e] - all) * sl2);
        if (m[e] == all) f[e] = 1.f;  // infinite maxima too
      }
      for (int c0 = 0; c0 < p.head_dim; c0 += 32) {  // 32 columns at a time
#pragma unroll
        for (int n = 0; n < DP / 8; ++n)
          if (n * 8 >= c0 && n * 8 < c0 + 32) {
#pragma unroll
            for (int e = 0; e < 2; ++e)
              *reinterpret_cast<float2*>(join + (warp * 16 + g + 8 * e) * L::kPitch + n * 8 - c0 + quad * 2) =
                  make_float2(o[n][2 * e] * f[e], o[n][2 * e + 1] * f[e]);
          }
        __syncthreads();
        for (int i = tid; i < rows * 4; i += kRowsThreads) {  // 8 columns of one row
          const int r = i >> 2, c = (i & 3) * 8, t = r >> 4;
          if (c0 + c >= p.head_dim) continue;
          float y[8] = {}, all = -INFINITY, norm = 0.f;
#pragma unroll
          for (int w = 0; w < kKeyWarps; ++w) {
            const float* src = join + ((w * MT + t) * 16 + (r & 15)) * L::kPitch + c;
            all = fmaxf(all, stat[((w * MT + t) * 16 + (r & 15)) * 2]);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] += src[e];
          }
#pragma unroll
          for (int w = 0; w < kKeyWarps; ++w) {
            const float* st = stat + ((w * MT + t) * 16 + (r & 15)) * 2;
            norm += st[0] == all ? st[1] : (st[0] == -INFINITY ? 0.f : st[1] * exp2_sfu((st[0] - all) * sl2));
          }
          const int token = r / p.group, qh = at.head * p.group + r % p.group;
          const int sees = keys_seen(token, q_len(p, at.seq), at.len_k, p.causal);
          const float inv = !whole ? 1.f : (norm == 0.f ? 0.f : 1.f / norm);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            y[e] *= inv;
            if (patch) y[e] = put_back(y[e], fix, c0 + c + e, sees);
          }
          if (whole) {
            *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (q0 + token) * p.o_ts + qh * p.o_hs + c0 + c) =
                make_uint4(pack16<T>(y[0], y[1]), pack16<T>(y[2], y[3]), pack16<T>(y[4], y[5]), pack16<T>(y[6], y[7]));
            if (c0 + c == 0 && p.lse)
              p.lse[static_cast<int64_t>(q0 + token) * p.q_heads + qh] = norm == 0.f ? -INFINITY : fmaf(all, scale, logf(norm));
          } else {
            float* dst = rp.parts + (static_cast<int64_t>(slot) * rp.rows + r) * p.head_dim + c0 + c;
            *reinterpret_cast<float4*>(dst) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(dst + 4) = make_float4(y[4], y[5], y[6], y[7]);
            if (c0 + c == 0)
              *reinterpret_cast<float2*>(rp.stats + (static_cast<int64_t>(slot) * rp.rows + r) * 2) = make_float2(all, norm);
          }
        }
        __syncthreads();
      }
      if (patch) {
        for (int i = tid; i < 3 * 128; i += kRowsThreads) fix[i] = INT_MAX;
        if (tid == 0) *fixed = 0;
        __syncthreads();
      }
      fresh = true;
    }
    at.advance(p);
  }
  grid_dep_launch();
}

// Joins the parts of every (sequence, head) that was cut: block c - 1 takes the one that run c goes on
// with, when run c is the first to do so.  Parts are summed in the order of the keys.
template <typename T>
__global__ void __launch_bounds__(kRowsThreads) attention_rows_join_kernel(const RowsParams rp) {
  grid_dep_launch();
  grid_dep_wait();
  const AttnParams& p = rp.a;
  const int c = blockIdx.x + 1;
  const RowsRun run = rp.runs[c];
  if (c >= run.runs || run.tile == 0) return;
  const int64_t first = run.start - run.tile, end = first + run.tiles;
  if (run_start(run.units, run.runs, c - 1) > first) return;
  int parts = 1;  // run c - 1's, then one for each run that starts before the end
  while (c + parts - 1 < run.runs && run_start(run.units, run.runs, c + parts - 1) < end) ++parts;
  const float scale = fmaxf(p.scale, 1e-30f), sl2 = scale * 1.4426950408889634f;
  const int rows = min(q_len(p, run.seq), p.max_q) * p.group, q0 = q_start(p, run.seq), vecs = p.head_dim / 8;
  for (int i = threadIdx.x; i < rows * vecs; i += kRowsThreads) {
    const int r = i / vecs, d = i % vecs * 8;
    auto row_of = [&](int k) { return (static_cast<int64_t>(2 * (c - 1 + k) + (k == 0 ? 1 : 0))) * rp.rows + r; };
    float all = -INFINITY;
    for (int k = 0; k < parts; ++k) all = fmaxf(all, rp.stats[row_of(k) * 2]);
    float y[8] = {}, norm = 0.f;
    for (int k = 0; k < parts; ++k) {
      const float2 st = *reinterpret_cast<const float2*>(rp.stats + row_of(k) * 2);
      const float f = st.x == all ? 1.f : (st.x == -INFINITY ? 0.f : exp2_sfu((st.x - all) * sl2));
      norm = fmaf(st.y, f, norm);
      const float4* src = reinterpret_cast<const float4*>(rp.parts + row_of(k) * p.head_dim + d);
      const float4 a = src[0], b = src[1];
      const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = f == 0.f && !isfinite(x[e]) ? y[e] + x[e] : fmaf(x[e], f, y[e]);
    }
    const float inv = norm == 0.f ? 0.f : 1.f / norm;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= inv;
    const int token = r / p.group, qh = run.head * p.group + r % p.group;
    *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (q0 + token) * p.o_ts + qh * p.o_hs + d) =
        make_uint4(pack16<T>(y[0], y[1]), pack16<T>(y[2], y[3]), pack16<T>(y[4], y[5]), pack16<T>(y[6], y[7]));
    if (d == 0 && p.lse)
      p.lse[static_cast<int64_t>(q0 + token) * p.q_heads + qh] = norm == 0.f ? -INFINITY : fmaf(all, scale, logf(norm));
  }
}

}  // namespace aexrt
