// Attention of many query rows on the tensor cores: packed prompts, and chunks of new tokens over
// the paged cache.
//
// One CTA takes two tiles of 128 query rows of one key/value head (rows: token x the query heads that
// share the head, so grouped heads read each key tile once) and walks the keys that they see in
// tiles of 128.  Per tile and key tile: S = Q K^T into TMEM, the softmax warps turn S into
// probabilities P, which replace S in TMEM as 16-bit pairs, and O += P V with P as the TMEM operand.
// Two row tiles share every K and V tile, so that the tensor core works on one while the softmax
// warps work on the other.  A thread owns a row, so the running maximum m and sum l need no exchange
// between threads.  O in TMEM is in units of a reference maximum that moves only when a row's true
// maximum has passed it by 2^8: P stays below 2^8 (far inside fp16) and the rescaling of O, a
// round trip through registers, is skipped for almost every tile.
//
// Roles: warps 0-3 softmax of tile 0, warps 4-7 of tile 1, warp 8 (one thread) issues the MMAs, warp 9
// loads, warps 10 and 11 only complete the third warpgroup: registers are split by warpgroup, 216 for a softmax thread
// (it holds a whole row of S) and 72 for the others, 2 * 216 + 72 = 3 * 168 as launched.
// TMEM columns: S0 0-127, S1 128-255, O0 256-, O1 384-.
#pragma once
#include <climits>

#include "attention_math.cuh"

namespace aexrt {

constexpr int kTcRows = 128;   // query rows of a tile
constexpr int kTcKeys = 128;   // keys of a tile
constexpr int kTcThreads = 384;

// Slots of the K / V ring (K and V tiles alternate): what 227 KB hold beside the two Q tiles.
template <int DP>
constexpr int tc_slots() { return DP == 128 ? 5 : 8; }

template <int DP>
struct TcSmem {
  static constexpr int kTile = 128 * DP * 2;
  static constexpr int kQ = 0, kRing = 2 * kTile, kBars = kRing + tc_slots<DP>() * kTile;
  // barriers, TMEM base, flags, then the first key with a +inf, -inf or NaN in a value column
  static constexpr int kFix = kBars + 256, kBytes = kFix + 3 * 128 * 4;
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
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

struct TcWork {
  int seq, tile, len_q, rows_q, len_k, q0, k0;  // rows_q: query tokens taken (len_q, at most max_q)
};

// The work item that is number `w` when every sequence has ceil(rows / tokens) of them; false past the end.
template <bool kPaged>
__device__ __forceinline__ bool tc_find(const AttnParams& p, int64_t w, int tokens, TcWork& out) {
  const int lane = threadIdx.x & 31;
  int64_t before = 0;
  for (int base = 0; base < p.num_seqs; base += 32) {
    const int s = base + lane;
    int rows = 0;
    if (s < p.num_seqs) {
      rows = q_len(p, s);
      if (kPaged) rows = min(rows, p.max_q);
    }
    const int n = (rows + tokens - 1) / tokens;
    int sum = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int z = __shfl_up_sync(~0u, sum, o);
      if (lane >= o) sum += z;
    }
    const uint32_t past = __ballot_sync(~0u, before + sum > w);
    if (past) {
      const int src = __ffs(past) - 1;
      out.seq = base + src;
      const int tiles = __shfl_sync(~0u, n, src);
      const int first = __shfl_sync(~0u, sum - n, src);
      out.rows_q = __shfl_sync(~0u, rows, src);
      // the last tiles of a causal sequence see the most keys: they go first
      out.tile = tiles - 1 - static_cast<int>(w - before - first);
      out.len_q = q_len(p, out.seq);
      out.q0 = q_start(p, out.seq);
      out.len_k = k_len<kPaged>(p, out.seq);
      out.k0 = k_start<kPaged>(p, out.seq);
      return true;
    }
    before += __shfl_sync(~0u, sum, 31);
  }
  return false;
}

template <int kRegs>
__device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

template <typename T, bool kPaged, int DP>
__global__ void __launch_bounds__(kTcThreads, 1)
    attention_tc_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ CUtensorMap k_map,
                        const __grid_constant__ CUtensorMap v_map, const AttnParams p) {
  extern __shared__ __align__(1024) uint8_t smem[];
  using L = TcSmem<DP>;
  constexpr int NS = tc_slots<DP>(), kHalves = DP / 64;
  uint64_t* q_full = reinterpret_cast<uint64_t*>(smem + L::kBars);
  uint64_t *kv_full = q_full + 2, *kv_empty = kv_full + NS, *raw = kv_empty + NS, *s_full = raw + 1, *p_full = s_full + 2,
           *o_done = p_full + 2;
  uint64_t* drain = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  int* fixed = reinterpret_cast<int*>(tmem_slot + 1);
  int* fix = reinterpret_cast<int*>(smem + L::kFix);
  static_assert((2 + 2 * tc_slots<DP>() + 8) * 8 + 8 <= 256, "barriers fit");

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  grid_dep_launch();
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(q_full + i, 1);
      mbar_init(s_full + i, 1);
      mbar_init(p_full + i, 128);
      mbar_init(o_done + i, 1);
    }
    for (int i = 0; i < NS; ++i) {
      mbar_init(kv_full + i, 1);
      mbar_init(kv_empty + i, 1);
    }
    mbar_init(raw, 1);
    mbar_init(drain, 1);
    fence_mbar_init();
    *fixed = 0;
  }
  for (int i = threadIdx.x; i < 3 * 128; i += kTcThreads) fix[i] = INT_MAX;
  if (warp == 8) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  grid_dep_wait();
  const int tokens = kTcRows / p.group;  // query tokens of a tile
  const int head = static_cast<int>(blockIdx.x % p.kv_heads);
  TcWork w;
  const bool found = tc_find<kPaged>(p, blockIdx.x / p.kv_heads, 2 * tokens, w);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (found) {
    int first[2], valid[2], keys[2], n[2];  // per row tile: first token, tokens, keys seen by the last, key tiles
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      first[s] = w.tile * 2 * tokens + s * tokens;
      valid[s] = clampi(w.rows_q - first[s], 0, tokens);
      keys[s] = valid[s] ? keys_seen(first[s] + valid[s] - 1, w.len_q, w.len_k, p.causal) : 0;
      n[s] = (keys[s] + kTcKeys - 1) / kTcKeys;
    }
    const int key_end = max(keys[0], keys[1]), nmax = max(n[0], n[1]);
    // keys at and above `common` are seen by some rows of the CTA and not by others
    const int common = min(keys_seen(first[0], w.len_q, w.len_k, p.causal), key_end);

    if (warp >= 8) {
      regs_down<72>();
      if (warp == 9) {
      // ---------------------------------------------------------------- loads
      const uint32_t q_bytes = static_cast<uint32_t>(tokens * p.group * 128 * kHalves);
      auto load_q = [&](int s) {
        if (lane == 0) {
          mbar_arrive_expect_tx(q_full + s, q_bytes);
          for (int h = 0; h < kHalves; ++h)
            tma_load_4d(smem + L::kQ + s * L::kTile + h * 16384, &q_map, q_full + s, h * 64, 0, head, w.q0 + first[s]);
        }
      };
      // one K or V tile; the bytes count whole boxes, what lies outside the tensor arrives as zeros
      auto load_kv = [&](const CUtensorMap* map, uint8_t* dst, uint64_t* bar, int j) {
        if (lane == 0) mbar_arrive_expect_tx(bar, L::kTile);
        __syncwarp();
        if constexpr (kPaged) {
          const int rows = min(1 << p.page_shift, kTcKeys);
          const int key = j * kTcKeys + lane * rows;
          if (lane * rows < kTcKeys) {
            int page = p.kv_tokens;  // outside: zeros
            if (key < key_end) {
              const int id = __ldg(p.block_table + w.seq * p.table_stride + (key >> p.page_shift));
              if (id >= 0 && id < p.kv_tokens) page = id; else atomicOr(p.status, kAttnBadPage);
            }
            for (int h = 0; h < kHalves; ++h)
              tma_load_4d(dst + h * 16384 + lane * rows * 128, map, bar, h * 64, head, key & ((1 << p.page_shift) - 1), page);
          }
        } else if (lane == 0) {
          for (int h = 0; h < kHalves; ++h) tma_load_3d(dst + h * 16384, map, bar, h * 64, head, w.k0 + j * kTcKeys);
        }
        __syncwarp();
      };
      bool ok = true;
      int raw_phase = 0;
      if (nmax) load_q(0);
      for (int i = 0; i < 2 * nmax && ok; ++i) {  // K0 V0 K1 V1 ...
        const int slot = i % NS, j = i >> 1;
        uint8_t* dst = smem + L::kRing + slot * L::kTile;
        ok = mbar_wait_bounded(kv_empty + slot, ((i / NS) & 1) ^ 1, p.status, kAttnTimeout);
        if (!ok) break;
        const int last = key_end - j * kTcKeys, seen = common - j * kTcKeys;  // rows of this tile below them
        const bool clean = (i & 1) && (last < kTcKeys || (seen < kTcKeys && seen < last));
        load_kv((i & 1) ? &v_map : &k_map, dst, clean ? raw : kv_full + slot, j);
        if (i == 0 && n[1]) load_q(1);
        if (clean) {
          // P is 0 where a row does not see a key, but 0 * inf and 0 * NaN are not: rows behind the
          // last key become zeros, and non-finite values of keys that only some rows see are taken
          // out and put back into the outputs of the rows that do
          ok = mbar_wait_bounded(raw, raw_phase & 1, p.status, kAttnTimeout);
          ++raw_phase;
          if (ok) {
            for (int h = 0; h < kHalves; ++h)
              for (int r = max(0, min(seen, last)); r < kTcKeys; r += 4) {
                const int row = r + (lane >> 3);
                if (row < kTcKeys) {
                  // 16-byte piece c of row r lies at piece c ^ (r % 8) (the 128-byte swizzle)
                  uint4* at = reinterpret_cast<uint4*>(dst + h * 16384 + row * 128) + (lane & 7);
                  if (row >= last) {
                    *at = make_uint4(0, 0, 0, 0);
                  } else {
                    const uint4 x = *at;
                    if (non_finite_bits<T>(x.x) | non_finite_bits<T>(x.y) | non_finite_bits<T>(x.z) | non_finite_bits<T>(x.w)) {
                      *at = take_non_finite<T>(x, j * kTcKeys + row, h * 64 + ((lane & 7) ^ (row & 7)) * 8, fix);
                      *fixed = 1;
                    }
                  }
                }
              }
            fence_proxy_async_smem();
          }
          __syncwarp();
          if (ok && lane == 0) mbar_arrive(kv_full + slot);
        }
      }
      if (!ok) {
        // a wait gave up: the loads in flight still have to land before the CTA may leave
        for (int i = 0; i < 2 * (NS + 3); ++i) {
          uint64_t* bar = i < 2 * NS ? kv_full + (i >> 1) : (i < 2 * NS + 4 ? q_full + ((i - 2 * NS) >> 1) : raw);
          mbar_wait_bounded(bar, i & 1, p.status, kAttnTimeout);
        }
      }
      } else if (warp == 8) {
      // ---------------------------------------------------------------- MMA issue
      if (lane == 0 && nmax) {
        const uint32_t id_s = tc_idesc<T>(kTcKeys, false), id_o = tc_idesc<T>((p.head_dim + 15) / 16 * 16, true);
        const int steps = (p.head_dim + 15) / 16;
        const uint32_t q_at = smem_u32(smem + L::kQ), ring = smem_u32(smem + L::kRing);
        auto full = [&](int i) { return mbar_wait_bounded(kv_full + i % NS, (i / NS) & 1, p.status, kAttnTimeout); };
        auto scores = [&](int s, int i) {  // S_s = Q_s K^T, K in ring item i
          const uint32_t a = q_at + s * L::kTile, b = ring + (i % NS) * L::kTile;
          for (int k = 0; k < steps; ++k) {
            const uint32_t off = (k >> 2) * 16384 + (k & 3) * 32;
            tc_mma<true>(tmem + s * 128, desc_sw128(a + off, 16, 1024), desc_sw128(b + off, 16, 1024), id_s, k != 0);
          }
          tc_commit(s_full + s);
        };
        bool ok = mbar_wait_bounded(q_full, 0, p.status, kAttnTimeout) && full(0);
        if (ok) {
          tc_fence_after();
          if (n[0]) scores(0, 0);
          if (n[1]) {
            ok = mbar_wait_bounded(q_full + 1, 0, p.status, kAttnTimeout);
            if (ok) scores(1, 0);
          }
          tc_commit(kv_empty);
        }
        for (int j = 0; j < nmax && ok; ++j) {
          const int iv = 2 * j + 1, ik = 2 * j + 2;
          ok = full(iv) && (j + 1 == nmax || full(ik));
          for (int s = 0; s < 2 && ok; ++s) {
            if (j >= n[s]) continue;
            ok = mbar_wait_bounded(p_full + s, j & 1, p.status, kAttnTimeout);
            if (!ok) break;
            tc_fence_after();
            const uint32_t b = ring + (iv % NS) * L::kTile;
#pragma unroll
            for (int k = 0; k < kTcKeys / 16; ++k)
              tc_mma_ts(tmem + 256 + s * 128, tmem + s * 128 + k * 8, desc_sw128(b + k * 2048, 16384, 1024), id_o, (j | k) != 0);
            tc_commit(o_done + s);
            if (j + 1 < n[s]) scores(s, ik);
          }
          if (ok) {
            tc_commit(kv_empty + iv % NS);
            if (j + 1 < nmax) tc_commit(kv_empty + ik % NS);
          }
        }
        if (!ok) {  // a wait gave up: the products in flight end before TMEM is freed
          tc_commit(drain);
          mbar_wait_bounded(drain, 0, p.status, kAttnTimeout);
        }
      }
      __syncwarp();
      }
    } else {
      // ---------------------------------------------------------------- softmax: one row per thread
      regs_up<216>();
      const int s = warp >> 2, row = threadIdx.x & 127;
      const int token = first[s] + row / p.group;
      const bool mine = row < tokens * p.group && row / p.group < valid[s];
      const int seen = mine ? keys_seen(token, w.len_q, w.len_k, p.causal) : 0;
      const int all_see = valid[s] ? keys_seen(first[s], w.len_q, w.len_k, p.causal) : 0;
      const uint32_t lanes = tmem + (static_cast<uint32_t>(warp & 3) << 21);  // this warp's 32 TMEM lanes
      const uint32_t s_at = lanes + s * 128, o_at = lanes + 256 + s * 128;
      const float scale = fmaxf(p.scale, 1e-30f);  // 0 would make NaN of a masked score's -inf
      const float sl2 = scale * 1.4426950408889634f;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int j = 0; j < n[s]; ++j) {
        ok = mbar_wait_bounded(s_full + s, j & 1, p.status, kAttnTimeout);
        ok = __all_sync(~0u, ok);
        if (!ok) break;
        tc_fence_after();
        uint32_t x[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(s_at + c * 32, *reinterpret_cast<uint32_t(*)[32]>(x + c * 32));
        tmem_ld_wait();
        if ((j + 1) * kTcKeys > all_see) {
          const int lim = seen - j * kTcKeys;
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (c >= lim) x[c] = 0xff800000u;
        }
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 128; c += 4)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = fmaxf(mx[e], __uint_as_float(x[c + e]));
        const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
        const bool move = (top - m) * sl2 > kLazyLog2;  // from -inf too
        if (__any_sync(~0u, move)) {
          const float old = m;
          if (move) m = top;
          const float f = move ? exp2_sfu((old - m) * sl2) : 1.f;
          l *= f;
          if (__any_sync(~0u, move && old != -INFINITY)) {
            ok = mbar_wait_bounded(o_done + s, (j - 1) & 1, p.status, kAttnTimeout);
            ok = __all_sync(~0u, ok);
            if (!ok) break;
            tc_fence_after();
            uint32_t o[32];
            for (int c = 0; c < DP; c += 32) {
              tmem_ld_32x32(o_at + c, o);
              tmem_ld_wait();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
              tmem_st_32x32(o_at + c, o);
            }
            tmem_st_wait();
          }
        }
        const float base = m == -INFINITY ? 0.f : -m * sl2;
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
        tmem_st_32x32(s_at, x);
        tmem_st_32x32(s_at + 32, x + 32);
        float a, b;
        f2_unpack(f2_add(sum[0], sum[1]), a, b);
        l += a + b;
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(p_full + s);
      }
      if (ok && n[s]) ok = mbar_wait_bounded(o_done + s, (n[s] - 1) & 1, p.status, kAttnTimeout);
      ok = __all_sync(~0u, ok);
      if (ok && valid[s]) {
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t tok = w.q0 + token;
        const int qh = head * p.group + row % p.group;
        T* dst = static_cast<T*>(p.out) + tok * p.o_ts + qh * p.o_hs;
        const bool patch = *reinterpret_cast<volatile int*>(fixed) != 0;
        for (int c = 0; c < p.head_dim; c += 32) {
          uint32_t o[32];
          if (n[s]) {
            tmem_ld_32x32(o_at + c, o);
            tmem_ld_wait();
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
          if (mine) {
#pragma unroll
            for (int v = 0; v < 4; ++v) {
              if (c + 8 * v >= p.head_dim) break;
              uint32_t y[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const int i = 8 * v + 2 * e;
                float a = __uint_as_float(o[i]) * inv, b = __uint_as_float(o[i + 1]) * inv;
                if (seen == 0) a = b = 0.f;
                if (patch) {
                  a = put_back(a, fix, c + i, seen);
                  b = put_back(b, fix, c + i + 1, seen);
                }
                y[e] = pack16<T>(a, b);
              }
              *reinterpret_cast<uint4*>(dst + c + 8 * v) = make_uint4(y[0], y[1], y[2], y[3]);
            }
          }
        }
        if (mine && p.lse) p.lse[tok * p.q_heads + qh] = l == 0.f ? -INFINITY : fmaf(m, scale, logf(l));
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace aexrt
