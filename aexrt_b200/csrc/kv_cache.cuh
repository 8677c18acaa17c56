// The paged cache's side of attention: the tables of a step from request lengths, and the write of
// new rows to their slots.
#pragma once
#include <cstdint>

#include "ptx.cuh"

namespace aexrt {

constexpr int kTablesThreads = 1024;
constexpr int kTablesMaxSeqs = 16384;
constexpr int kTablesMaxCtas = 8;

struct TablesParams {
  const int32_t *ctx, *add, *free_pages, *state_in;
  int32_t *table, *state_out, *cu_q, *kv_lens, *slots;
  int num_seqs, page_shift, columns, free_capacity, slot_capacity;
  int64_t table_stride;
};

// Exclusive sums over the block of one 64-bit value per thread; returns the total in `total`.
__device__ __forceinline__ int64_t block_exclusive_sum(int64_t x, int64_t& total) {
  __shared__ int64_t part[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int64_t y = x;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t z = __shfl_up_sync(~0u, y, o);
    if (lane >= o) y += z;
  }
  __syncthreads();
  if (lane == 31) part[warp] = y;
  __syncthreads();
  int64_t before = 0;
  total = 0;
  for (int i = 0; i < static_cast<int>(blockDim.x >> 5); ++i) {
    if (i < warp) before += part[i];
    total += part[i];
  }
  return before + y - x;
}

// Entries of sums[0 .. n] (not decreasing, sums[0] = 0) at or below x, less one: the request that
// item x of the concatenation belongs to.
__device__ __forceinline__ int find_request(const int32_t* sums, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (sums[mid] <= x) lo = mid; else hi = mid;
  }
  return lo;
}

// Every CTA sums all requests' new tokens and new pages into its own shared
// memory (a few KB, read from L2 by each), then fills its share of the slots, of the new table
// columns and of the per-request outputs.  A slot in a new page takes the page from the free stack
// directly, by the page's rank in the order of taking, so no CTA waits for another's table writes;
// the cluster barrier between the reads of lengths and state and all writes is what lets kv_lens
// and the state be updated in place.  Latency-bound: a few dependent rounds of loads and one barrier
// (256 requests of one token: 5.8 us; 65536 new tokens, on 64 blocks: 10 us, a binary search per slot).
__global__ void __launch_bounds__(kTablesThreads) page_tables_kernel(const TablesParams p) {
  extern __shared__ int32_t sums[];  // new tokens [n + 1], new pages [n + 1], context [n]
  grid_dep_launch();
  grid_dep_wait();
  const int n = p.num_seqs;
  int32_t *cu = sums, *taken = sums + n + 1, *ctx = sums + 2 * (n + 1);
  constexpr int64_t kMax = INT32_MAX;
  const int64_t ps = 1ll << p.page_shift;
  int64_t tokens_before = 0, pages_before = 0;
  for (int base = 0; base < n; base += kTablesThreads) {
    const int i = base + threadIdx.x;
    int64_t c = 0, a = 0, pages = 0;
    if (i < n) {
      c = max(0, __ldcg(p.ctx + i));
      a = max(0, __ldcg(p.add + i));
      a = min(a, kMax - c);
      const int64_t have = min((c + ps - 1) >> p.page_shift, static_cast<int64_t>(p.columns));
      pages = min((c + a + ps - 1) >> p.page_shift, static_cast<int64_t>(p.columns)) - have;
    }
    int64_t all_tokens, all_pages;
    const int64_t t0 = tokens_before + block_exclusive_sum(a, all_tokens);
    const int64_t g0 = pages_before + block_exclusive_sum(pages, all_pages);
    if (i < n) {
      ctx[i] = static_cast<int32_t>(c);
      cu[i] = static_cast<int32_t>(min(t0, kMax));
      taken[i] = static_cast<int32_t>(min(g0, kMax));
      if (i == n - 1) {
        cu[n] = static_cast<int32_t>(min(t0 + a, kMax));
        taken[n] = static_cast<int32_t>(min(g0 + pages, kMax));
      }
    }
    tokens_before += all_tokens;
    pages_before += all_pages;
  }
  const int top = min(max(0, __ldcg(p.state_in)), p.free_capacity);
  if (n == 0 && threadIdx.x == 0) cu[0] = taken[0] = 0;
  __syncthreads();
  // in place, the CTAs are one cluster: every one has read ctx and the state, outputs may take their place
  // (alone, each is a cluster of its own)
  cluster_sync_all();
  const int at = blockIdx.x * kTablesThreads + threadIdx.x, step = gridDim.x * kTablesThreads;
  for (int i = at; i <= n; i += step) {
    p.cu_q[i] = cu[i];
    if (i < n) p.kv_lens[i] = ctx[i] + (cu[i + 1] - cu[i]);
  }
  const int all = taken[n];
  if (at == 0) {
    p.state_out[0] = max(0, top - all);
    p.state_out[1] = max(0, all - top);
  }
  for (int64_t next = at; next < all; next += step) {  // `all` may be 2^31 - 1: a step past it needs 64 bits
    const int g = static_cast<int>(next);
    const int s = find_request(taken, n, g);
    const int col = static_cast<int>((ctx[s] + ps - 1) >> p.page_shift) + (g - taken[s]);
    p.table[s * p.table_stride + col] = g < top ? __ldg(p.free_pages + top - 1 - g) : -1;
  }
  for (int t = at; t < p.slot_capacity; t += step) {
    int slot = -1;
    if (t < cu[n]) {
      const int s = find_request(cu, n, t);
      const int pos = ctx[s] + (t - cu[s]);
      const int col = pos >> p.page_shift, fresh = col - static_cast<int>((ctx[s] + ps - 1) >> p.page_shift);
      int page = -1;
      if (col < p.columns) {
        if (fresh < 0) {
          page = p.table[s * p.table_stride + col];
        } else {
          const int g = taken[s] + fresh;
          if (g < top) page = __ldg(p.free_pages + top - 1 - g);
        }
      }
      const int64_t there = page * ps + (pos & (ps - 1));
      if (page >= 0 && there <= kMax) slot = static_cast<int>(there);
    }
    p.slots[t] = slot;
  }
}

struct AppendParams {
  const uint4 *k, *v;
  uint4 *k_cache, *v_cache;
  const int32_t* slots;
  int tokens, kv_heads, row_vecs, page_shift, num_slots;  // row_vecs: 16-byte pieces of a head's row
  int64_t k_ts, k_hs, v_ts, v_hs, kc_ps, kc_ts, kc_hs, vc_ps, vc_ts, vc_hs;  // in 16-byte pieces
};

// One thread copies one 16-byte piece of k and the same piece of v: HBM-bound, 32768 rows of 8 heads of 128 in
// 45 us (5.96 TB/s); 64 rows in 2 us.
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendParams p) {
  grid_dep_launch();
  grid_dep_wait();
  const int per_token = p.kv_heads * p.row_vecs;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int t = static_cast<int>(i / per_token), u = static_cast<int>(i % per_token);
  if (t >= p.tokens) return;
  const int slot = __ldg(p.slots + t);
  if (slot < 0 || slot >= p.num_slots) return;
  const int h = u / p.row_vecs, c = u % p.row_vecs;
  const int64_t page = slot >> p.page_shift, r = slot & ((1 << p.page_shift) - 1);
  const uint4 a = p.k[t * p.k_ts + h * p.k_hs + c];
  const uint4 b = p.v[t * p.v_ts + h * p.v_hs + c];
  p.k_cache[page * p.kc_ps + r * p.kc_ts + h * p.kc_hs + c] = a;
  p.v_cache[page * p.vc_ps + r * p.vc_ts + h * p.vc_hs + c] = b;
}

}  // namespace aexrt
