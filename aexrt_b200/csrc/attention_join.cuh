// Joining the parts of a row whose keys were split over several blocks.
#pragma once
#include "attention_math.cuh"

namespace aexrt {

// What a block leaves about rows that a second launch joins: their parts (0: nothing to join), the query
// tokens or rows, the first query token, the key/value head.
struct JoinHead {
  int parts, rows, q0, head;
};

// Columns d .. d + 7 of one output row (query token `token`, query head `qh`) from `parts` unnormalised sums with
// their maxima (raw score units) and normalisers; part k is row row_of(k) of `sums` and `stats`.  Summed in the order
// of the keys, four parts' loads at a time.
template <typename T, typename RowOf>
__device__ __forceinline__ void join_row(const AttnParams& p, const float* sums, const float* stats, int parts, RowOf row_of, int d,
                                         int token, int qh) {
  const float sl2 = p.scale * 1.4426950408889634f;
  float y[8] = {}, all = -INFINITY, norm = 0.f;
  for (int k0 = 0; k0 < parts; k0 += 4) {
    float2 st[4];
    float4 a[4], b[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t row = row_of(min(k0 + k, parts - 1));
      st[k] = *reinterpret_cast<const float2*>(stats + row * 2);
      const float4* src = reinterpret_cast<const float4*>(sums + row * p.head_dim + d);
      a[k] = src[0];
      b[k] = src[1];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (k0 + k >= parts) break;
      if (st[k].x > all) {  // a new maximum: what is summed so far shrinks
        const float f = all == -INFINITY ? 0.f : exp2_sfu((all - st[k].x) * sl2);
        norm *= f;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = f == 0.f && !isfinite(y[e]) ? y[e] : y[e] * f;
        all = st[k].x;
      }
      const float f = st[k].x == all ? 1.f : (st[k].x == -INFINITY ? 0.f : exp2_sfu((st[k].x - all) * sl2));
      norm = fmaf(st[k].y, f, norm);
      const float x[8] = {a[k].x, a[k].y, a[k].z, a[k].w, b[k].x, b[k].y, b[k].z, b[k].w};
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = f == 0.f && !isfinite(x[e]) ? y[e] + x[e] : fmaf(x[e], f, y[e]);
    }
  }
  const float inv = norm == 0.f ? 0.f : 1.f / norm;
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] *= inv;
  *reinterpret_cast<uint4*>(static_cast<T*>(p.out) + token * p.o_ts + qh * p.o_hs + d) =
      make_uint4(pack_out<T>(y[0], y[1]), pack_out<T>(y[2], y[3]), pack_out<T>(y[4], y[5]), pack_out<T>(y[6], y[7]));
  if (d == 0 && p.lse)
    p.lse[static_cast<int64_t>(token) * p.q_heads + qh] = norm == 0.f ? -INFINITY : fmaf(all, p.scale, logf(norm * kProbUnit<T>));
}

}  // namespace aexrt
