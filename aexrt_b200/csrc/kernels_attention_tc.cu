// The tensor-core attention kernel's instances: type x packed, paged or paged with split items x padded head size.
#include "attention_tc.cuh"
#include "kernels_attention.cuh"

namespace aexrt {

template <typename T, bool kPaged, bool kSplit>
static TcKernel pick(int head_dim) {
  const auto join = attention_tc_join_kernel<T>;
  if (head_dim <= 64) return TcKernel{attention_tc_kernel<T, kPaged, 64, kSplit>, join, TcSmem<64>::kBytes};
  return TcKernel{attention_tc_kernel<T, kPaged, 128, kSplit>, join, TcSmem<128>::kBytes};
}

template <typename T>
static TcKernel pick(bool paged, bool split, int head_dim) {
  return paged ? (split ? pick<T, true, true>(head_dim) : pick<T, true, false>(head_dim)) : pick<T, false, false>(head_dim);
}

TcKernel attention_tc_for(bool bf16, bool paged, bool split, int head_dim) {
  return bf16 ? pick<__nv_bfloat16>(paged, split, head_dim) : pick<__half>(paged, split, head_dim);
}

}  // namespace aexrt
