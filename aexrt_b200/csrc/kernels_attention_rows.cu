// The few-rows attention kernel's instances: type x padded head size x tiles of 16 rows.
#include "attention_rows.cuh"
#include "kernels_attention.cuh"

namespace aexrt {

template <typename T, int DP>
static RowsKernel pick(int rows) {
  const auto join = attention_rows_join_kernel<T>;
  constexpr int smem = RowsSmem<DP>::kBytes;
  if (rows <= 16) return RowsKernel{attention_rows_kernel<T, DP, 1>, join, smem};
  if (rows <= 32) return RowsKernel{attention_rows_kernel<T, DP, 2>, join, smem};
  return RowsKernel{attention_rows_kernel<T, DP, 4>, join, smem};
}

RowsKernel attention_rows_for(bool bf16, int head_dim, int rows) {
  if (bf16) return head_dim <= 64 ? pick<__nv_bfloat16, 64>(rows) : pick<__nv_bfloat16, 128>(rows);
  return head_dim <= 64 ? pick<__half, 64>(rows) : pick<__half, 128>(rows);
}

}  // namespace aexrt
