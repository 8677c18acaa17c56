// The tensor-core attention kernel's instances: type x packed or paged x padded head size.
#include "attention_tc.cuh"
#include "kernels_attention.cuh"

namespace aexrt {

template <typename T, bool kPaged>
static TcKernel pick(int head_dim) {
  if (head_dim <= 64) return TcKernel{attention_tc_kernel<T, kPaged, 64>, TcSmem<64>::kBytes};
  return TcKernel{attention_tc_kernel<T, kPaged, 128>, TcSmem<128>::kBytes};
}

TcKernel attention_tc_for(bool bf16, bool paged, int head_dim) {
  if (bf16) return paged ? pick<__nv_bfloat16, true>(head_dim) : pick<__nv_bfloat16, false>(head_dim);
  return paged ? pick<__half, true>(head_dim) : pick<__half, false>(head_dim);
}

}  // namespace aexrt
