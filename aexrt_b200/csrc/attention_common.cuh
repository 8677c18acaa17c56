// What the attention kernels share: the call's parameters, where a sequence's rows and keys lie, and
// the conversions of the two 16-bit types.  Lengths come from device memory; they are cut to the
// extents that the host passed, so that no index derived from them leaves a tensor.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstdint>

#include "ptx.cuh"

namespace aexrt {

// Bits of the attention status word (AEXRT_B200_ATTENTION_*).
enum : uint32_t { kAttnBadPage = 1u << 0, kAttnTimeout = 1u << 1 };

// What a scale of 0 is replaced by, fp32's smallest number: 0 would make NaN of a masked score's -inf.  The largest score
// becomes 2^-21, as much as rounding its exponential may take.
constexpr float kMinScale = 1.401298464e-45f;

struct AttnParams {
  const void *q, *k, *v;  // k, v: packed rows or the paged caches
  void* out;
  float* lse;                 // [q_tokens][q_heads] or null
  const int32_t* cu_q;        // [num_seqs + 1]
  const int32_t* cu_k;        // packed: [num_seqs + 1]
  const int32_t* kv_lens;     // paged: [num_seqs]
  const int32_t* block_table; // paged
  uint32_t* status;
  int64_t q_ts, q_hs, o_ts, o_hs;  // token and head strides, elements
  int64_t k_ts, k_hs, k_ps, v_ts, v_hs, v_ps;
  int num_seqs, q_tokens, max_q, q_heads, kv_heads, group, head_dim;
  int kv_tokens;  // packed: rows of k, v; paged: pages
  int page_shift, table_columns;
  int no_page;  // paged: a page number outside the tensor maps (they have one page at least), whose rows load as zeros
  int64_t table_stride;
  int causal;
  float scale;  // of the scores, in natural units: kMinScale to 1e38, so that scale * log2 e is neither 0 nor infinite
};

__device__ __forceinline__ int clampi(int x, int lo, int hi) { return x < lo ? lo : (x > hi ? hi : x); }

// First query row and query rows of sequence s (0 rows for offsets that go back).
__device__ __forceinline__ int q_start(const AttnParams& p, int s) { return clampi(__ldg(p.cu_q + s), 0, p.q_tokens); }
__device__ __forceinline__ int q_len(const AttnParams& p, int s) { return max(0, q_start(p, s + 1) - q_start(p, s)); }

template <bool kPaged>
__device__ __forceinline__ int k_start(const AttnParams& p, int s) {
  return kPaged ? 0 : clampi(__ldg(p.cu_k + s), 0, p.kv_tokens);
}
template <bool kPaged>
__device__ __forceinline__ int k_len(const AttnParams& p, int s) {
  if constexpr (kPaged) {
    const int64_t room = static_cast<int64_t>(p.table_columns) << p.page_shift;
    const int n = max(0, __ldg(p.kv_lens + s));
    return n < room ? n : static_cast<int>(room);
  } else {
    return max(0, clampi(__ldg(p.cu_k + s + 1), 0, p.kv_tokens) - k_start<kPaged>(p, s));
  }
}

// Keys that query token i of a sequence sees: keys 0 .. keys_seen - 1.
__device__ __forceinline__ int keys_seen(int i, int len_q, int len_k, int causal) {
  return causal ? clampi(i + 1 + len_k - len_q, 0, len_k) : len_k;
}

template <typename T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

}  // namespace aexrt
