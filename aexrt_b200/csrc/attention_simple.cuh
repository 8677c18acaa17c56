// Attention one query row at a time: a warp holds one row of one query head (four of its elements
// per lane), walks the keys it sees and keeps the running maximum m, the sum l and the weighted sum
// of v.  Right for every size; it reads k and v once per row, so its time goes to L1 / L2 traffic
// and to the five shuffles of each key's dot product.
#pragma once
#include "attention_common.cuh"

namespace aexrt {

template <typename T, bool kPaged>
__global__ void __launch_bounds__(128) attention_row_kernel(const AttnParams p) {
  grid_dep_launch();
  grid_dep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const int token = static_cast<int>(row / p.q_heads), head = static_cast<int>(row % p.q_heads);
  if (token >= p.q_tokens) return;
  int s = 0;  // the sequence whose rows hold token
  while (s < p.num_seqs && !(q_start(p, s) <= token && token < q_start(p, s + 1))) ++s;
  if (s == p.num_seqs) return;
  const int i = token - q_start(p, s);
  if (kPaged && i >= p.max_q) return;
  const int len_k = k_len<kPaged>(p, s), k0 = k_start<kPaged>(p, s);
  const int seen = keys_seen(i, q_len(p, s), len_k, p.causal);
  const int d0 = lane * 4, kvh = head / p.group;
  const bool on = d0 < p.head_dim;
  float q[4] = {}, acc[4] = {}, m = -INFINITY, l = 0.f;
  if (on)
    for (int e = 0; e < 4; ++e) q[e] = to_f32(static_cast<const T*>(p.q)[token * p.q_ts + head * p.q_hs + d0 + e]);
  for (int j = 0; j < seen; ++j) {
    int64_t ko, vo;
    bool there = true;
    if constexpr (kPaged) {
      const int page = __ldg(p.block_table + s * p.table_stride + (j >> p.page_shift));
      const int r = j & ((1 << p.page_shift) - 1);
      there = page >= 0 && page < p.kv_tokens;
      if (!there && lane == 0) atomicOr(p.status, kAttnBadPage);
      ko = page * p.k_ps + r * p.k_ts;
      vo = page * p.v_ps + r * p.v_ts;
    } else {
      ko = static_cast<int64_t>(k0 + j) * p.k_ts;
      vo = static_cast<int64_t>(k0 + j) * p.v_ts;
    }
    float x = 0.f;
    if (on && there)
      for (int e = 0; e < 4; ++e) x = fmaf(q[e], to_f32(static_cast<const T*>(p.k)[ko + kvh * p.k_hs + d0 + e]), x);
    for (int o = 16; o; o >>= 1) x += __shfl_xor_sync(~0u, x, o);
    x *= p.scale;
    const float m2 = fmaxf(m, x);
    const float old = m2 == -INFINITY ? 1.f : __expf(m - m2), w = m2 == -INFINITY ? 0.f : __expf(x - m2);
    l = l * old + w;
    m = m2;
    if (on)
      for (int e = 0; e < 4; ++e)
        acc[e] = acc[e] * old + (there ? w * to_f32(static_cast<const T*>(p.v)[vo + kvh * p.v_hs + d0 + e]) : 0.f);
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (on)
    for (int e = 0; e < 4; ++e)
      static_cast<T*>(p.out)[token * p.o_ts + head * p.o_hs + d0 + e] = from_f32<T>(seen ? acc[e] * inv : 0.f);
  if (lane == 0 && p.lse) p.lse[static_cast<int64_t>(token) * p.q_heads + head] = m + logf(l);
}

}  // namespace aexrt
